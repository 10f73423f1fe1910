"""Edges of the expert calls on the GPU: scratch and stream captures, extreme values, waits that run out, offsets beyond 32 bits.
Helpers and the rule for tolerances: tests/test_expert_gpu.py."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

import test_expert_gpu
from test_expert_gpu import U, assert_product, blocks_of, combine_reference, plan_of, product_reference, randn, score_code

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


def test_a_captured_dispatch_outlives_larger_ones(pkg, torch_cuda):
    """The scratch that a graph was captured with stays when a later call needs more."""
    torch = torch_cuda
    handle = pkg.Sampler(max_rows=1, max_vocab=64)

    def fields(plan):
        return [t.clone() for t in (plan.expert_offsets, plan.route_token, plan.route_rank, plan.route_weight, plan.status)]

    try:
        small, large = randn(torch, 1, 300, 16), randn(torch, 2, 40000, 200)
        side = torch.cuda.Stream()
        want, plan = handle.router_dispatch(small, 2), handle.router_dispatch(small, 2)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            handle.router_dispatch(small, 2, out=plan)
            with pytest.raises(pkg.MoeError, match="inside a stream capture"):
                handle.router_dispatch(large, 4)
        first = None
        for _ in range(3):
            for t in (plan.expert_offsets, plan.route_token, plan.route_rank, plan.route_weight):
                t.zero_()
            plan.status.fill_(-1)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                other = handle.router_dispatch(large, 4)
                graph.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(fields(plan), fields(want)))
            assert first is None or all(torch.equal(a, b) for a, b in zip(fields(other), first))
            first = fields(other)
    finally:
        handle.close()


def often_routed(torch, source_rows, columns):
    """Rows that are quantised once and copied: 4.5 routes a row, 2^25 values and more."""
    routes = source_rows * 9 // 2
    source = randn(torch, 7, source_rows, columns).bfloat16()
    index = torch.randint(source_rows, (routes,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").int()
    blocks = (columns + 127) // 128
    out = (torch.zeros((routes, columns), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((blocks, routes), device="cuda"))
    return source, index, out


def test_quantize_scratch_is_bounded(pkg, sampler, torch_cuda):
    """Whatever calls a handle has seen, it holds 48 MiB for rows that are quantised once (allocations come in 2 MiB)."""
    torch = torch_cuda
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        calls = [often_routed(torch, rows, 4096) for rows in (2500, 6200, 6500, 11500)]
        for source, index, out in calls:    # another handle: what the kernels themselves need is on the device then
            sampler.quantize_rows(source, route_token=index, out=out)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        for source, index, out in calls:
            handle.quantize_rows(source, route_token=index, out=out)
        torch.cuda.synchronize()
        assert before - torch.cuda.mem_get_info()[0] <= 50 << 20
    finally:
        handle.close()


def test_quantize_captured_before_any_scratch(pkg, torch_cuda):
    """Captured as the handle's first call: the bits of the call that quantises each row once."""
    torch = torch_cuda
    source, index, out = often_routed(torch, 2500, 4096)
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            handle.quantize_rows(source, route_token=index, out=out)
        graph.replay()
        torch.cuda.synchronize()
        values, scales = handle.quantize_rows(source, route_token=index)
        assert torch.equal(values.view(torch.uint8), out[0].view(torch.uint8)) and torch.equal(scales, out[1])
    finally:
        handle.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,columns", [(1300, 4096), (4200, 4096), (4200, 4087), (9000, 2000), (30000, 640)])
def test_quantize_wide_and_narrow_items(sampler, pkg, torch_cuda, dtype, gated, rows, columns):
    """Calls that take the wide items, by type, gate and alignment, and long calls of short rows, which do not."""
    test_expert_gpu.test_quantize_large_calls_are_their_parts(sampler, pkg, torch_cuda, dtype, gated, rows, columns)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,columns", [(64, 300), (1500, 4096)])
def test_quantize_gate_far_below_zero(sampler, pkg, torch_cuda, dtype, rows, columns):
    """Gates whose exp(-gate) is beyond fp32 and ups that bring the product back: h = gate * e * up * e with e = exp(gate / 2), two
    units in the last place (4 U) each, and three products: 11 U.  The scale adds its division, a value e4m3's half step and both."""
    torch = torch_cuda
    x = torch.empty((rows, 2 * columns), device="cuda")
    x[:, :columns] = -88.75 - 14 * torch.rand((rows, columns), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    x[:, columns:] = 1e30 * randn(torch, 4, rows, columns)
    x = x.to(getattr(torch, dtype))
    values, scales = sampler.quantize_rows(x, activation=pkg.ACTIVATION_SILU_GATE)
    gate, up = x.double()[:, :columns], x.double()[:, columns:]
    h = gate * torch.sigmoid(gate) * up
    padded = torch.nn.functional.pad(h, (0, -columns % 128)).view(rows, -1, 128)
    want = (padded.abs().amax(dim=2) / 448).t()
    assert bool((want > 1e-30).all()) and bool(((scales.double() - want).abs() <= 13 * U * want).all())
    wide = scales.double().t().repeat_interleave(128, dim=1)[:, :columns]
    off = (values.double() * wide - h).abs()
    assert bool((off <= (2.0 ** -4 + 32 * U) * h.abs().clamp_min(2.0 ** -6 * wide)).all())


def test_quantize_gate_of_infinities(sampler, pkg, torch_cuda):
    """NaN where the formula has none, and only there: -inf / inf, and 0 times an infinity."""
    torch = torch_cuda
    inf = float("inf")
    gate = torch.tensor([-inf, -300.0, -89.0, 0.0, 5.0, inf, 5.0, float("nan")], device="cuda")
    up = torch.tensor([1.0, 1.0, 1.0, inf, 2.0, 0.0, 0.0, 1.0], device="cuda")
    values, scales = sampler.quantize_rows(torch.cat([gate, up])[None], activation=pkg.ACTIVATION_SILU_GATE)
    decoded = values.float()[0] * scales[0]
    assert torch.isnan(decoded).tolist() == [True, False, False, True, False, True, False, True]
    assert decoded[[1, 2, 6]].abs().max() == 0    # far below the block's largest, or zero
    assert abs(float(decoded[4]) - 10 / (1 + 2.718281828459045 ** -5)) <= 2.0 ** -4 * 10


@pytest.mark.parametrize("score", ["sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("experts", [24, 256, 1000, 1500])
@pytest.mark.parametrize("lowest", [float("-inf"), -3.4028234663852886e38])
def test_balance_of_tokens_masked_for_every_expert(sampler, pkg, torch_cuda, score, experts, lowest):
    """Scores that are zeros: the token counts with probabilities 0 and has gradient 0.  One expert left: gradient 0 for the others."""
    torch = torch_cuda
    tokens, code = 20, score_code(pkg, score)
    logits = 1.5 * randn(torch, 31, tokens, experts)
    plan = plan_of(torch, 8, tokens, experts, 3)
    logits[4] = lowest
    logits[9, 1:] = lowest
    out = sampler.balance_loss(logits, plan["offsets"], plan["token"], 3, score_function=code)
    rest = logits.clone()
    rest[4] = 0
    mask = torch.ones(tokens, dtype=torch.bool, device="cuda")
    mask[4] = False
    without = sampler.balance_loss(rest, plan["offsets"], plan["token"], 3, score_function=code, token_mask=mask)
    want = without.expert_probability.double() * (tokens - 1) / tokens
    # the same sums in another order over at most 20 tokens, and a division each
    assert bool(((out.expert_probability.double() - want).abs() <= 24 * U * want).all()) and int(out.expert_tokens[-1]) == tokens
    gradient = sampler.balance_loss_backward(logits, out.expert_tokens, 3, score_function=code)
    assert bool((gradient[4] == 0).all()) and bool(torch.isfinite(gradient).all())
    assert bool((gradient[9, 1:] == 0).all())


def test_waits_run_out(torch_cuda):
    """tests/cuda/waits.cu: a wait for what never comes ends, marks the CTA, and ends the waits of the other warps."""
    source = Path(__file__).resolve().parent / "cuda" / "waits.cu"
    target = source.with_name("libtest_waits.so")
    csrc = source.parent.parent.parent / "ncnn-moe-runtime_b200" / "csrc"
    inputs = [source, csrc / "moe_tensor.cuh", csrc / "moe_common.cuh"]
    if not target.exists() or any(path.stat().st_mtime > target.stat().st_mtime for path in inputs):
        nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
        subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-o", str(target), str(source)], check=True)
    results, microseconds = (ctypes.c_int * 7)(), ctypes.c_float()
    library = ctypes.CDLL(str(target))
    assert library.test_waits(ctypes.c_uint32(1000), results, ctypes.byref(microseconds)) == 0
    assert list(results) == [0, 1, 0, 0, 1, 1, 1]
    assert microseconds.value < 1e5     # two times 1000 looks of 4 us, and the 64000 looks cut short after a millisecond


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("source_rows,routes,columns", [(50, 173, 40), (50, 173, 264), (300, 1100, 4096), (1000, 33000, 1040), (1000, 33000, 1032)])
def test_quantize_gates_routed_rows(sampler, pkg, torch_cuda, dtype, source_rows, routes, columns):
    """Gate and route in one call, route by route and with rows quantised once: the bits of the gated rows, gathered."""
    torch = torch_cuda
    source = (2 * randn(torch, 7, source_rows, 2 * columns)).to(getattr(torch, dtype))
    index = torch.randint(source_rows, (routes,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").int()
    rows, row_scales = sampler.quantize_rows(source, activation=pkg.ACTIVATION_SILU_GATE)
    values, scales = sampler.quantize_rows(source, route_token=index, activation=pkg.ACTIVATION_SILU_GATE)
    want, want_scales = rows.view(torch.uint8)[index.long()], row_scales[:, index.long()]
    assert torch.equal(values.view(torch.uint8), want) and torch.equal(scales, want_scales)
    assert sampler.expert_check() == 0
    index[[5, routes - 1]] = torch.tensor([source_rows, -1], dtype=torch.int32, device="cuda")
    values, scales = sampler.quantize_rows(source, route_token=index, activation=pkg.ACTIVATION_SILU_GATE)
    assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE
    want[[5, routes - 1]] = 0
    want_scales[:, [5, routes - 1]] = 0
    assert torch.equal(values.view(torch.uint8), want) and torch.equal(scales, want_scales)


# experts, rows of all, outputs, columns: which kernel, and what has more than 2^32 bytes or values
BEYOND = [pytest.param(70, 70 * 20, 8192, 8208, id="tiles of 32 rows, weights"), pytest.param(70, 70 * 33, 128, 480000, id="tiles of 64 rows, weights"),
          pytest.param(70, 70 * 40, 8192, 8208, id="many rows, weights"), pytest.param(4096, 65536, 16, 65552, id="tiles of 16 rows, values and weights"),
          pytest.param(1, 530000, 16, 8208, id="many rows, values"), pytest.param(4096, 65536, 65600, 16, id="tiles of 16 rows, outputs"),
          pytest.param(1, (1 << 22) + 200, 1040, 16, id="many rows, outputs in whole lines"), pytest.param(1, (1 << 22) + 200, 1039, 16, id="many rows, outputs anywhere")]


@pytest.mark.parametrize("experts,rows,outputs,columns", BEYOND)
def test_products_beyond_32_bits(sampler, torch_cuda, experts, rows, outputs, columns):
    """The last rows, of the last expert; all others are zeros."""
    torch = torch_cuda
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    last = 16 if experts == 4096 else 40
    values = torch.zeros((rows, columns), dtype=torch.float8_e4m3fn, device="cuda")
    values[-last:] = (randn(torch, 3, last, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    weights = torch.zeros((experts, outputs, columns), dtype=torch.float8_e4m3fn, device="cuda")
    weights[-1] = (randn(torch, 2, outputs, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.ones((blocks_of(columns), rows), device="cuda")
    weight_scales = torch.ones((experts, blocks_of(outputs), blocks_of(columns)), device="cuda")
    scales[:, -last:] = torch.rand((blocks_of(columns), last), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") + 0.1
    if experts == 4096:
        offsets = 16 * torch.arange(experts + 1, dtype=torch.int32, device="cuda")
    else:   # the first expert and the last one
        offsets = torch.full((experts + 1,), rows - last, dtype=torch.int32, device="cuda")
        offsets[0], offsets[-1] = 0, rows
    out = torch.full((rows, outputs), -7.0, dtype=torch.bfloat16, device="cuda")
    sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets if experts > 1 else None, out=out)
    one = torch.tensor([0, last], dtype=torch.int32, device="cuda")
    reference = product_reference(torch, values[-last:], scales[:, -last:].contiguous(), weights[-1:], weight_scales[-1:], one)
    assert_product(torch, out[-last:], reference, columns)
    for first in range(0, rows - last, 1 << 18):
        assert not bool(out[first:min(first + (1 << 18), rows - last)].any())
    assert sampler.expert_check() == 0
    del values, weights, out, reference
    torch.cuda.empty_cache()
