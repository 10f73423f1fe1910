"""CPU tests of what the expert calls do at their edges: scratch and stream captures."""
from test_abi_cpu import run_host_test


def test_scratch_does_not_grow_inside_a_capture(tmp_path):
    """tests/cpp/kept_scratch_test.cpp: growing, with fakes for the runtime calls."""
    run_host_test(tmp_path, "kept_scratch_test")
