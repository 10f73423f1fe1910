"""CPU tests of what the expert calls do at their edges: scratch and stream captures, look-ups that fail, grids and items."""
from test_abi_cpu import run_host_test


def test_scratch_does_not_grow_inside_a_capture(tmp_path):
    """tests/cpp/kept_scratch_test.cpp: growing, with fakes for the runtime calls."""
    run_host_test(tmp_path, "kept_scratch_test")


def test_a_failed_look_up_is_made_again(tmp_path):
    """tests/cpp/look_up_test.cpp: the driver's function that describes tiles to the copy engine is remembered once it is found."""
    run_host_test(tmp_path, "look_up_test")


def test_balance_grids_cover_the_largest_batches(tmp_path):
    """tests/cpp/balance_blocks_test.cpp: tokens of up to 2^32 - 1."""
    run_host_test(tmp_path, "balance_blocks_test")


def test_quantisation_items_fit_the_rows(tmp_path):
    """tests/cpp/quantize_steps_test.cpp: short rows and small calls are cut finer."""
    run_host_test(tmp_path, "quantize_steps_test")
