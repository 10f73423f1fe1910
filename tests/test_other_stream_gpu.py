"""Calls on a stream that is not the current one: their results are made there.  On the current stream their memory could be filled
behind the kernels that write it, or be handed out while they write."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def randn(torch, seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def tensors_of(torch, result):
    if torch.is_tensor(result):
        return [result]
    if isinstance(result, dict):
        result = result.values()
    elif not isinstance(result, (tuple, list)):
        result = vars(result).values()
    return [t for part in result for t in (tensors_of(torch, part) if part is not None and not isinstance(part, int) else [])]


def calls(pkg, torch, handle):
    """Every method that makes device results, by name: a call on a stream."""
    rows, vocab, tokens, experts, top_k, columns = 4096, 2048, 70000, 16, 4, 64
    logits = randn(torch, 1, rows, vocab)
    params = np.zeros(rows, dtype=pkg.ROW_PARAMS_DTYPE)
    params["temperature"], params["top_k"], params["top_p"] = 0.7, 8, 0.9
    params["row_id"] = np.arange(rows)
    scores = randn(torch, 2, tokens, experts)
    plan = handle.router_dispatch(scores, top_k)
    hidden = randn(torch, 3, tokens, columns)
    values, scales = handle.quantize_rows(hidden, route_token=plan.route_token)
    weights = (randn(torch, 4, experts, 128, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    weight_scales = torch.ones((experts, 1, 1), device="cuda")
    routed = handle.expert_product(values, scales, weights, weight_scales, expert_offsets=plan.expert_offsets)
    balance = handle.balance_loss(scores, plan.expert_offsets, plan.route_token, top_k)
    candidates = handle.local_candidates(logits, 0, 64)
    proposed = torch.zeros((256, 2), dtype=torch.int32, device="cuda")
    target, draft = logits[:768].view(256, 3, vocab), logits[768:1280].view(256, 2, vocab)
    return {
        "sample_batch": lambda stream: handle.sample_batch(logits, params, topk_stride=128, stream=stream),
        "sample_batch_kept": lambda stream: handle.sample_batch(logits, params, kept_stride=128, stream=stream),
        "speculative_verify": lambda stream: handle.speculative_verify(target[0], draft[0], proposed[0], params[:1], stream=stream, sync=False),
        "speculative_verify_batch": lambda stream: handle.speculative_verify_batch(target, draft, proposed, params[:256], stream=stream, sync=False),
        "local_candidates": lambda stream: handle.local_candidates(logits, 0, 64, stream=stream),
        "merge_candidates": lambda stream: handle.merge_candidates(candidates[None], params, 64, topk_stride=128, stream=stream),
        "router_dispatch": lambda stream: handle.router_dispatch(scores, top_k, stream=stream),
        "regroup_gather": lambda stream: handle.regroup_gather(hidden, plan.route_token, stream=stream),
        "indexer_topk": lambda stream: handle.indexer_topk(logits, 200, with_scores=True, stream=stream),
        "quantize_rows": lambda stream: handle.quantize_rows(hidden, route_token=plan.route_token, stream=stream),
        "expert_product": lambda stream: handle.expert_product(values, scales, weights, weight_scales, expert_offsets=plan.expert_offsets, stream=stream),
        "combine_routes": lambda stream: handle.combine_routes(routed, plan.route_token, plan.route_rank, plan.route_weight, tokens, top_k, stream=stream),
        "balance_loss": lambda stream: handle.balance_loss(scores, plan.expert_offsets, plan.route_token, top_k, stream=stream),
        "balance_loss_backward": lambda stream: handle.balance_loss_backward(scores, balance.expert_tokens, top_k, stream=stream),
    }


NAMES = ["sample_batch", "sample_batch_kept", "speculative_verify", "speculative_verify_batch", "local_candidates", "merge_candidates", "router_dispatch", "regroup_gather",
         "indexer_topk", "quantize_rows", "expert_product", "combine_routes", "balance_loss", "balance_loss_backward"]


@pytest.fixture(scope="module")
def all_calls(pkg, torch_cuda):
    handle = pkg.Sampler(max_rows=4096, max_vocab=2048)
    yield calls(pkg, torch_cuda, handle)
    torch_cuda.cuda.synchronize()
    handle.close()


@pytest.mark.parametrize("name", NAMES)
def test_results_belong_to_the_stream_of_the_call(all_calls, torch_cuda, name):
    """Dropped results are not handed out on the current stream, and are what a call on the current stream returns."""
    torch = torch_cuda
    want = [t.clone() for t in tensors_of(torch, all_calls[name](None))]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    for handle_of in (side, torch.cuda.default_stream()):
        with torch.cuda.stream(torch.cuda.Stream() if handle_of is not side else torch.cuda.default_stream()):
            got = tensors_of(torch, all_calls[name](handle_of.cuda_stream))
            torch.cuda.synchronize()
            assert len(got) == len(want)
            for a, b in zip(got, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            held = {t.data_ptr(): t.numel() * t.element_size() for t in got if t.numel()}
            del got, a, b
            again = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2) for size in held.values()]
            assert not {t.data_ptr() for t in again} & set(held)
            del again


def test_a_refusal_is_not_cleared_by_earlier_work_of_the_current_stream(pkg, torch_cuda):
    """The status of a refused dispatch, which is made as a zero, with the current stream busy meanwhile."""
    torch = torch_cuda
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        logits = randn(torch, 1, 300, 16)
        logits[4, 3] = float("inf")
        side = torch.cuda.Stream()
        handle.router_dispatch(logits, 2)
        torch.cuda.synchronize()
        torch.cuda._sleep(50_000_000)       # some 30 ms
        plan = handle.router_dispatch(logits, 2, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert int(plan.status) == 101      # "router logits must be finite"
    finally:
        handle.close()
