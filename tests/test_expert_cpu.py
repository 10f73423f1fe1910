"""CPU tests of the expert products, the combine and the balance loss: arguments that are refused, and the plain forms that
perf/operators.py compares the kernels with, on small cases against the definitions in 64 bits."""
import importlib.util
from pathlib import Path

import pytest
import torch

from test_abi_cpu import run_host_test

ROOT = Path(__file__).resolve().parent.parent


def test_arguments_are_checked_before_any_launch(tmp_path):
    """tests/cpp/expert_checks_test.cpp: every refusal of the argument checks, without a GPU."""
    run_host_test(tmp_path, "expert_checks_test")


def test_entry_points_refuse_a_null_handle(pkg):
    library = pkg.library()
    assert library.moe_quantize_rows(None, None, None, 0, 1, 1, 1, 0, None, 0, None, None) == 1
    assert library.moe_expert_product(None, None, None, None, 1, 16, None, None, 1, 1, None, None, 0, 1) == 1
    assert library.moe_combine_routes(None, None, None, 0, 1, 1, None, None, None, 1, 1, 1, None, None) == 1
    assert library.moe_expert_check(None, None, None) == 1
    assert library.moe_balance_loss(None, None, None, 1, None, None, None, None, 1.0, None, None, None) == 1
    assert library.moe_balance_loss_backward(None, None, None, 1, None, None, 1.0, None, None, None) == 1


@pytest.fixture()
def operators():
    spec = importlib.util.spec_from_file_location("perf_operators_cpu", ROOT / "perf" / "operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.DEVICE = "cpu"
    return module


SMALL = [
    dict(kind="quantize", tokens=9, top_k=3, columns=136, dtype="bf16", gate=False),
    dict(kind="quantize", tokens=5, top_k=2, columns=264, dtype="f32", gate=True),
    dict(kind="product", tokens=7, top_k=2, experts=8, columns=144, outputs=130, out="f32"),
    dict(kind="product", tokens=7, top_k=1, experts=1, columns=256, outputs=65, out="bf16"),
    dict(kind="combine", tokens=11, top_k=3, columns=37, dtype="bf16", base=True),
    dict(kind="balance", tokens=23, experts=12, top_k=3, score="softmax", mask=True),
    dict(kind="balance", tokens=23, experts=12, top_k=3, score="sigmoid", mask=False),
    dict(kind="balance", tokens=23, experts=12, top_k=3, score="sqrtsoftplus", mask=True),
    dict(kind="layer", tokens=8, top_k=2, experts=4, columns=400, inner=336),
]


@pytest.mark.parametrize("case", SMALL, ids=lambda c: f"{c['kind']}-{c['tokens']}")
def test_plain_forms_agree_with_the_definitions(operators, case):
    """Relative error in the 2-norm.  An fp32 result is off by its last rounding (2^-24) and by sums of at most 256 terms (each
    addition 2^-24 of a partial sum that is at most sqrt(256) times the result in these random sums: 2^-12); bf16 results
    round by 2^-9 at most on average over a binade, e4m3 by 2^-4."""
    state = operators.prepare(case, 3)
    got, want = operators.run(state), operators.exact(case, 3)
    got = got if isinstance(got, dict) else dict(out=got)
    want = want if isinstance(want, dict) else dict(out=want)
    for name, value in want.items():
        if value is None:
            continue
        off = float((got[name].double() - value).norm() / value.norm())
        bound = {torch.float32: 2.0 ** -12, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}[got[name].dtype]
        assert off <= bound, (name, off)


def test_plain_balance_gradient_against_differences(operators):
    """Central differences of the loss in 64 bits along random directions: the third derivative of the normalised scores is of
    order one, so a step of 1e-3 leaves 1e-6 of the gradient; the fp32 result adds 2^-24."""
    for score in ("softmax", "sigmoid", "sqrtsoftplus"):
        case = dict(kind="balance", tokens=19, experts=10, top_k=3, score=score, mask=True)
        state = operators.prepare(case, 5)
        gradient = operators.run(state)["gradient"].double()

        def loss(logits):
            kept = state["mask"]
            p, _ = operators._probabilities(logits, score)
            counts = torch.bincount(state["plan"]["expert"][kept[state["plan"]["route_token"].long()]], minlength=10).double()
            return state["loss_gradient"].double()[0] * state["coefficient"] * (counts * 10 / (3 * kept.sum()) * p[kept].mean(dim=0)).sum()

        generator = torch.Generator().manual_seed(1)
        for _ in range(4):
            direction = torch.randn(state["logits"].shape, generator=generator).double()
            step = 1e-3
            slope = (loss(state["logits"].double() + step * direction) - loss(state["logits"].double() - step * direction)) / (2 * step)
            scale = float((gradient.abs() * direction.abs()).sum())
            assert abs(float((gradient * direction).sum() - slope)) <= 1e-5 * scale
