"""Edges of the expert calls on the GPU: scratch and stream captures.  Helpers and the rule for tolerances: tests/test_expert_gpu.py."""
import pytest

from test_expert_gpu import U, combine_reference, plan_of, randn

pytestmark = pytest.mark.gpu


def assert_combined(torch, out, rows, plan, tokens, top_k):
    want, size = combine_reference(torch, rows, plan, tokens, None)
    assert bool(((out.double() - want).abs() <= (top_k + 1) * U * size + U * want.abs()).all())


@pytest.mark.parametrize("mode", ["relaxed", "thread_local", "global"])
def test_combine_refuses_to_grow_inside_a_capture(pkg, torch_cuda, mode):
    """The call is refused in every mode, the capture goes on, and calls behind it find cleared scratch."""
    torch = torch_cuda
    tokens, top_k, columns = 700, 3, 40
    plan, rows = plan_of(torch, 5, tokens, 12, top_k), randn(torch, 6, tokens * top_k, columns)
    arguments = rows, plan["token"], plan["rank"], plan["weight"], tokens, top_k
    out, captured, copy = (torch.zeros((tokens, columns), device="cuda") for _ in range(3))
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode=mode):
            copy.copy_(rows[:tokens])
            with pytest.raises(pkg.MoeError, match="inside a stream capture"):
                handle.combine_routes(*arguments, out=captured)
        with torch.cuda.stream(side):   # before the first replay
            handle.combine_routes(*arguments, out=out)
            graph.replay()
        side.synchronize()
        assert_combined(torch, out, rows, plan, tokens, top_k)
        assert torch.equal(copy, rows[:tokens]) and bool((captured == 0).all())
        again = torch.cuda.CUDAGraph()
        with torch.cuda.graph(again, stream=side, capture_error_mode=mode):     # the scratch is there now
            handle.combine_routes(*arguments, out=captured)
        with torch.cuda.stream(side):
            again.replay()
            again.replay()
        side.synchronize()
        assert torch.equal(captured, out) and handle.expert_check() == 0
    finally:
        handle.close()


def test_balance_refuses_to_grow_inside_a_capture(pkg, torch_cuda):
    torch = torch_cuda
    plan, logits = plan_of(torch, 5, 300, 12, 2), randn(torch, 6, 300, 12)
    place = pkg.BalanceLoss(torch.zeros(1, device="cuda"), torch.zeros(13, dtype=torch.int32, device="cuda"), torch.zeros(12, device="cuda"))
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            place.loss.add_(1)
            with pytest.raises(pkg.MoeError, match="inside a stream capture"):
                handle.balance_loss(logits, plan["offsets"], plan["token"], 2, out=place)
        want = handle.balance_loss(logits, plan["offsets"], plan["token"], 2)
        torch.cuda.synchronize()
        again = torch.cuda.CUDAGraph()
        with torch.cuda.graph(again, stream=side):
            handle.balance_loss(logits, plan["offsets"], plan["token"], 2, out=place)
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(place.loss, want.loss) and torch.equal(place.expert_probability, want.expert_probability)
    finally:
        handle.close()
