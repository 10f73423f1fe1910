"""Expert products, combine and balance loss on the GPU, each against a plain implementation in 64 bits.

Tolerances are worst cases of the roundings: a value rounded to bf16 is off by at most 2^-8 of itself, to fp32 by 2^-24, to e4m3
by 2^-4 (half of 2^-9 below e4m3's smallest normal 2^-6); a sum of m terms kept in fp32 by (m - 1) * 2^-24 of the sum of their
magnitudes, twice that where an adder truncates."""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def rounding(torch, dtype):
    return {torch.float32: U, torch.bfloat16: 2.0 ** -8}[dtype]


def blocks_of(columns):
    return (columns + 127) // 128


def randn(torch, seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def plan_of(torch, seed, tokens, experts, top_k, skew=1.0):
    """Route arrays in the order of a dispatch plan: experts ascending, inside an expert tokens ascending."""
    taste = randn(torch, seed, tokens, experts) + skew * randn(torch, seed + 1, experts)
    best = taste.topk(top_k, dim=1)
    weight = torch.softmax(best.values, dim=1).reshape(-1)
    order = best.indices.reshape(-1).sort(stable=True)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(order.values, minlength=experts).cumsum(0)
    return dict(offsets=offsets, expert=order.values, token=(order.indices // top_k).int(), rank=(order.indices % top_k).int(), weight=weight[order.indices])


# ---- quantisation ---------------------------------------------------------------------


def quantize_reference(torch, x):
    """Scales and values of fp32 rows on the CPU, where a division is a division: [blocks, rows], [rows, columns] as floats."""
    x = x.float().cpu()
    rows, columns = x.shape
    padded = torch.nn.functional.pad(x, (0, blocks_of(columns) * 128 - columns)).view(rows, -1, 128)
    scales = padded.abs().amax(dim=2) / torch.tensor(448.0)
    quotient = torch.where(scales[..., None] > 0, padded / scales[..., None], padded)
    values = quotient.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return values.reshape(rows, -1)[:, :columns], scales.t()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 1024), (7, 1032), (4, 2880), (33, 4096), (2, 8200), (301, 264)])
def test_quantize_is_exact(sampler, torch_cuda, dtype, rows, columns):
    torch = torch_cuda
    x = (randn(torch, rows, rows, columns) * torch.logspace(-3, 3, rows, device="cuda")[:, None]).to(getattr(torch, dtype))
    x[0, : columns // 2] *= 64
    values, scales = sampler.quantize_rows(x)
    want_values, want_scales = quantize_reference(torch, x)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(values.float().cpu(), want_values)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("columns", [40, 256, 1000, 4096])
def test_quantize_gathers(sampler, torch_cuda, dtype, columns):
    torch = torch_cuda
    x = randn(torch, 5, 50, columns).to(getattr(torch, dtype))
    index = torch.randint(50, (173,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").int()
    values, scales = sampler.quantize_rows(x, route_token=index)
    want_values, want_scales = quantize_reference(torch, x[index.long()])
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(values.float().cpu(), want_values)
    assert sampler.expert_check() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("source_rows,routes,columns", [(1000, 33000, 1040), (2000, 16400, 2064), (7, 18000, 1872), (4200, 16799, 2064),
                                                         (1000, 33000, 1032)])
def test_quantize_gathers_rows_that_are_routed_often(sampler, pkg, torch_cuda, dtype, source_rows, routes, columns):
    """Four routes a row on average, and 2^25 values: the rows are quantised once and copied (below that, or with columns that are no
    multiple of 16, they are not)."""
    torch = torch_cuda
    x = (randn(torch, 5, source_rows, columns + 8) * 3).to(getattr(torch, dtype))[:, :columns]
    index = torch.randint(source_rows, (routes,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").int()
    values, scales = sampler.quantize_rows(x, route_token=index)
    want_values, want_scales = quantize_reference(torch, x[index.long()])
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(values.float().cpu(), want_values)
    assert sampler.expert_check() == 0
    index[[5, routes - 1]] = torch.tensor([source_rows, -1], dtype=torch.int32, device="cuda")
    spoiled = sampler.quantize_rows(x, route_token=index)
    assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE
    values.view(torch.uint8)[[5, routes - 1]] = 0
    scales[:, [5, routes - 1]] = 0
    assert torch.equal(spoiled[0].view(torch.uint8), values.view(torch.uint8)) and torch.equal(spoiled[1], scales)


def test_quantize_strides_alignments_and_sentinels(sampler, torch_cuda):
    """Rows inside a wider matrix, starts that no vector load takes, and nothing written outside the outputs."""
    torch = torch_cuda
    for dtype in (torch.float32, torch.bfloat16):
        wide = randn(torch, 2, 20, 900).to(dtype)
        for first, columns in ((0, 512), (8, 256), (1, 256), (3, 131), (4, 8)):
            part = wide[:, first:first + columns]
            values_store = torch.full((20 * columns + 64,), 0x55, dtype=torch.uint8, device="cuda")
            scales_store = torch.full((blocks_of(columns) * 20 + 8,), 7.0, device="cuda")
            out = (values_store[: 20 * columns].view(torch.float8_e4m3fn).view(20, columns), scales_store[:-8].view(-1, 20))
            sampler.quantize_rows(part, out=out)
            want_values, want_scales = quantize_reference(torch, part)
            assert torch.equal(out[1].cpu(), want_scales) and torch.equal(out[0].float().cpu(), want_values)
            assert bool((values_store[20 * columns:] == 0x55).all()) and bool((scales_store[-8:] == 7.0).all())


def test_quantize_special_values(sampler, torch_cuda):
    torch = torch_cuda
    x = randn(torch, 3, 8, 256)
    x[0] = 0                                    # zeros: scale 0
    x[1, 5] = float("nan")                      # a NaN stays in its place
    x[2, 200] = float("inf")                    # an infinity takes its block
    x[3] *= 1e-43                               # denormal block whose scale is denormal or zero
    x[4] *= 1e30
    x[5] *= 1e-30
    x[6] = 448.0
    x[7, :128] = torch.finfo(torch.float32).max
    values, scales = sampler.quantize_rows(x)
    values, scales = values.float().cpu(), scales.cpu()
    decoded = values * scales.t().repeat_interleave(128, dim=1)
    assert bool((decoded[0] == 0).all()) and bool((scales[:, 0] == 0).all())
    assert torch.isnan(decoded[1]).nonzero()[:, 0].tolist() == [5]
    assert bool(torch.isnan(decoded[2, 128:]).all()) and bool(torch.isfinite(decoded[2, :128]).all())
    for row in (3, 4, 5, 6):
        want_values, want_scales = quantize_reference(torch, x[row:row + 1])
        assert torch.equal(values[row], want_values[0]) and torch.equal(scales[:, row], want_scales[:, 0])
    assert bool((values[7, :128] == 448).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,columns", [(5000, 1032), (4300, 999), (1100, 4104), (34000, 130)])
def test_quantize_large_calls_are_their_parts(sampler, pkg, torch_cuda, dtype, gated, rows, columns):
    """Small and large calls divide the work differently and must agree bit for bit, special values included; ungated rows also
    with the plain formula."""
    torch = torch_cuda
    activation = pkg.ACTIVATION_SILU_GATE if gated else pkg.ACTIVATION_NONE
    x = randn(torch, 4, rows, columns * (2 if gated else 1)).to(getattr(torch, dtype))
    x[7] = 0
    x[9, 3] = float("nan")
    x[rows - 2, -1] = float("inf")
    x[11] *= 1e-38
    x[12] *= 1e30
    x[13, : columns // 2] = 448.0
    values, scales = sampler.quantize_rows(x, activation=activation)
    for first in range(0, rows, 100):
        part, part_scales = sampler.quantize_rows(x[first:first + 100], activation=activation)
        assert torch.equal(part.view(torch.uint8), values[first:first + 100].view(torch.uint8))
        assert torch.equal(part_scales, scales[:, first:first + 100])
    if not gated:
        plain = [row for row in range(rows) if row not in (9, rows - 2)]
        want_values, want_scales = quantize_reference(torch, x[plain])
        assert torch.equal(scales.cpu()[:, plain], want_scales) and torch.equal(values.float().cpu()[plain], want_values)


def test_quantize_refuses_to_follow_a_bad_route(sampler, pkg, torch_cuda):
    torch = torch_cuda
    x = randn(torch, 3, 4, 300)
    index = torch.tensor([0, 4, 3, -1], dtype=torch.int32, device="cuda")
    values, scales = sampler.quantize_rows(x, route_token=index)
    assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE and sampler.expert_check() == 0
    want_values, want_scales = quantize_reference(torch, x[[0, 3]])
    assert torch.equal(values.float().cpu()[[0, 2]], want_values) and torch.equal(scales.cpu()[:, [0, 2]], want_scales)
    assert bool((values.float()[[1, 3]] == 0).all()) and bool((scales[:, [1, 3]] == 0).all())
    values, scales = sampler.quantize_rows(x, route_token=index[:0])
    assert values.shape == (0, 300) and scales.shape == (3, 0)
    values, scales = sampler.quantize_rows(x[:0])
    assert values.shape == (0, 300)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,columns", [(1, 8), (5, 130), (128, 2880), (9, 1023)])
def test_quantize_gate(sampler, pkg, torch_cuda, dtype, rows, columns):
    """h = gate / (1 + exp(-gate)) * up: exp 2 roundings, the sum, the division and the product one each, 5 in all.  The scale is
    off by that and its own division's; a value by e4m3's half step and by both."""
    torch = torch_cuda
    x = (2 * randn(torch, columns, rows, 2 * columns)).to(getattr(torch, dtype))
    values, scales = sampler.quantize_rows(x, activation=pkg.ACTIVATION_SILU_GATE)
    gate, up = x.double()[:, :columns], x.double()[:, columns:]
    h = gate * torch.sigmoid(gate) * up
    padded = torch.nn.functional.pad(h, (0, blocks_of(columns) * 128 - columns)).view(rows, -1, 128)
    want = (padded.abs().amax(dim=2) / 448).t()
    assert bool(((scales.double() - want).abs() <= 7 * U * want).all())
    wide = scales.double().t().repeat_interleave(128, dim=1)[:, :columns]
    off = (values.double() * wide - h).abs()
    assert bool((off <= (2.0 ** -4 + 16 * U) * h.abs().clamp_min(2.0 ** -6 * wide)).all())


# ---- products -------------------------------------------------------------------------


def product_inputs(torch, seed, rows, columns, experts, outputs):
    values = (randn(torch, seed, rows, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    weights = (randn(torch, seed + 1, experts, outputs, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.rand((blocks_of(columns), rows), generator=torch.Generator(device="cuda").manual_seed(seed + 2), device="cuda") + 0.1
    weight_scales = torch.rand((experts, blocks_of(outputs), blocks_of(columns)), generator=torch.Generator(device="cuda").manual_seed(seed + 3), device="cuda") + 0.1
    return values, scales, weights, weight_scales


def product_reference(torch, values, scales, weights, weight_scales, offsets):
    """The sums in 64 bits and the sums of the magnitudes, expert by expert; NaN in rows of no expert."""
    rows, columns = values.shape
    experts, outputs, _ = weights.shape
    total = torch.full((rows, outputs), float("nan"), dtype=torch.float64, device="cuda")
    size = total.clone()
    bounds = [0, rows] if offsets is None else offsets.tolist()
    for e in range(experts):
        begin, end = bounds[e], bounds[e + 1]
        x = values[begin:end].double() * scales[:, begin:end].double().t().repeat_interleave(128, dim=1)[:, :columns]
        w = weights[e].double() * weight_scales[e].double().repeat_interleave(128, dim=0)[:outputs].repeat_interleave(128, dim=1)[:, :columns]
        total[begin:end] = x @ w.t()
        size[begin:end] = x.abs() @ w.abs().t()
    return total, size


def assert_product(torch, out, reference, columns):
    """A block's sum has 128 terms, then come its scales' product, the multiplication and the sum over the blocks."""
    total, size = reference
    bound = (2 * 128 + 2 + blocks_of(columns)) * U * size + rounding(torch, out.dtype) * total.abs()
    assert bool(((out.double() - total).abs() <= bound).all()), float(((out.double() - total).abs() / bound).max())


DENSE = [(1, 16, 1), (1, 128, 128), (2, 144, 129), (15, 272, 100), (16, 256, 256), (17, 2880, 64), (64, 512, 300), (65, 400, 127), (127, 1024, 384), (129, 896, 200),
         (200, 4096, 136), (257, 384, 1), (300, 640, 513), (1000, 256, 260), (1025, 1040, 640)]


@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,columns,outputs", DENSE)
def test_dense_product(sampler, torch_cuda, rows, columns, outputs, out_dtype):
    torch = torch_cuda
    inputs = product_inputs(torch, rows, rows, columns, 1, outputs)
    out = sampler.expert_product(*inputs, out_dtype=getattr(torch, out_dtype))
    assert_product(torch, out, product_reference(torch, *inputs, None), columns)
    assert torch.equal(out, sampler.expert_product(*inputs, out_dtype=getattr(torch, out_dtype)))
    assert sampler.expert_check() == 0


GROUPED = [(1, 8, 8, 256, 128), (3, 64, 4, 144, 200), (32, 128, 4, 2880, 320), (40, 16, 2, 512, 1000), (257, 8, 2, 384, 130), (130, 300, 3, 272, 72), (700, 4, 1, 1040, 264),
           (2048, 32, 4, 256, 256)]
# several tiles of 128 rows a CTA, with one to four blocks of columns and 16 to 128 columns in the last
GROUPED += [(4000, 4, 2, columns, 1300) for columns in (16, 128, 144, 256, 336, 512)] + [(3001, 3, 2, 384, 1000)]
# several tiles of 16, 32 and 64 rows a CTA
GROUPED += [(300, 80, 3, columns, 520) for columns in (32, 256, 384)] + [(600, 60, 3, 272, 520), (700, 40, 3, 144, 129), (700, 40, 3, 640, 700)]


@pytest.mark.parametrize("tokens,experts,top_k,columns,outputs", GROUPED)
def test_grouped_product(sampler, torch_cuda, tokens, experts, top_k, columns, outputs):
    torch = torch_cuda
    plan = plan_of(torch, tokens, tokens, experts, top_k)
    inputs = product_inputs(torch, tokens, tokens * top_k, columns, experts, outputs)
    reference = product_reference(torch, *inputs, plan["offsets"])
    for dtype in (torch.bfloat16, torch.float32):
        out = sampler.expert_product(*inputs, expert_offsets=plan["offsets"], out_dtype=dtype)
        assert_product(torch, out, reference, columns)
    assert sampler.expert_check() == 0


def test_product_leaves_other_rows_alone(sampler, torch_cuda):
    """Rows before the first expert's and behind the last one's, columns behind the outputs, and a plan without rows."""
    torch = torch_cuda
    for rows, cuts in ((90, [3, 3, 20, 21, 60]), (300, [17, 150, 150, 151, 299]), (64, [0, 0, 0, 0, 0]), (64, [64, 64, 64, 64, 64])):
        inputs = product_inputs(torch, rows, rows, 272, 4, 130)
        offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
        store = torch.full((rows, 140), -7.0, dtype=torch.bfloat16, device="cuda")
        out = sampler.expert_product(*inputs, expert_offsets=offsets, out=store[:, :130])
        begin, end = cuts[0], cuts[-1]
        total, size = product_reference(torch, *inputs, offsets)
        if end > begin:
            assert_product(torch, out[begin:end], (total[begin:end], size[begin:end]), 272)
        assert bool((store[:begin] == -7).all()) and bool((store[end:] == -7).all()) and bool((store[:, 130:] == -7).all())
    assert sampler.expert_check() == 0


def test_product_does_not_follow_bad_offsets(sampler, pkg, torch_cuda):
    torch = torch_cuda
    inputs = product_inputs(torch, 4, 40, 256, 3, 140)
    for cuts in ([0, 20, 10, 40], [0, 10, 20, 41], [0, -1, 20, 40], [50, 50, 50, 50]):
        out = torch.full((40, 140), 5.0, device="cuda")
        sampler.expert_product(*inputs, expert_offsets=torch.tensor(cuts, dtype=torch.int32, device="cuda"), out=out)
        assert bool((out == 5).all())
        assert sampler.expert_check() == pkg.EXPERT_FLAG_OFFSETS
    assert sampler.expert_check() == 0


def test_product_non_finite_rows_stay_in_their_rows(sampler, torch_cuda):
    """NaN values, infinite scales and rows of neighbouring experts in the same tile of the activations."""
    torch = torch_cuda
    values, scales, weights, weight_scales = product_inputs(torch, 9, 70, 256, 3, 140)
    offsets = torch.tensor([0, 21, 22, 70], dtype=torch.int32, device="cuda")
    clean = sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets)
    values.view(torch.uint8)[21, 3] = 0x7F
    scales[1, 40] = float("inf")
    out = sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[[21, 40]] = True
    assert torch.equal(out[~bad], clean[~bad])
    assert bool(torch.isnan(out[21]).all()) and not bool(torch.isfinite(out[40]).any())


def test_product_strides_and_one_expert_of_many(sampler, torch_cuda):
    torch = torch_cuda
    rows, experts = 333, 40
    inputs = product_inputs(torch, 2, rows, 384, experts, 264)
    cuts = [0] * 17 + [rows] * (experts + 1 - 17)      # expert 16 has every row
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    store = torch.zeros((rows, 300), device="cuda")
    out = sampler.expert_product(*inputs, expert_offsets=offsets, out=store[:, 5:269])
    assert_product(torch, out, product_reference(torch, *inputs, offsets), 384)
    assert bool((store[:, :5] == 0).all()) and bool((store[:, 269:] == 0).all())


@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("outputs,width,first", [(4096, 4096, 0), (4096, 4112, 16), (4104, 4128, 8), (4112, 4120, 0), (4112, 4112, 0), (4101, 4200, 32), (4096, 4097, 1), (4100, 4104, 4),
                                                 (4240, 4256, 0)])
def test_product_of_many_rows_into_any_place(sampler, torch_cuda, outputs, width, first, out_dtype):
    """Tiles of 128 rows, filled and partly filled, into outputs of every alignment; nothing else is written."""
    torch = torch_cuda
    rows, cuts = 1500, [3, 700, 701, 1490]
    inputs = product_inputs(torch, 5, rows, 144, 3, outputs)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    store = torch.full((rows, width), -7.0, dtype=getattr(torch, out_dtype), device="cuda")
    out = sampler.expert_product(*inputs, expert_offsets=offsets, out=store[:, first:first + outputs])
    total, size = product_reference(torch, *inputs, offsets)
    assert_product(torch, out[3:1490], (total[3:1490], size[3:1490]), 144)
    assert bool((store[:3] == -7).all()) and bool((store[1490:] == -7).all()) and bool((store[:, :first] == -7).all()) and bool((store[:, first + outputs:] == -7).all())


@pytest.mark.parametrize("rows_each,outputs", [(1, 130), (40, 200), (40, 201), (66, 129)])
def test_product_of_the_most_experts(sampler, pkg, torch_cuda, rows_each, outputs):
    torch = torch_cuda
    experts = pkg.EXPERT_MAX_EXPERTS
    inputs = product_inputs(torch, 6, rows_each * experts, 32, experts, outputs)
    offsets = rows_each * torch.arange(experts + 1, dtype=torch.int32, device="cuda")
    out = sampler.expert_product(*inputs, expert_offsets=offsets, out_dtype=torch.float32)
    values, scales, weights, weight_scales = inputs
    for e in (0, 1, 77, experts - 2, experts - 1):
        mine = slice(e * rows_each, (e + 1) * rows_each)
        part = (values[mine], scales[:, mine].contiguous(), weights[e:e + 1], weight_scales[e:e + 1])
        assert_product(torch, out[mine], product_reference(torch, *part, None), 32)
    assert sampler.expert_check() == 0


def test_product_refusals(sampler, pkg, torch_cuda):
    torch = torch_cuda
    values, scales, weights, weight_scales = product_inputs(torch, 2, 8, 256, 2, 64)
    offsets = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(pkg.MoeError, match="expert_offsets may only be null"):
        sampler.expert_product(values, scales, weights, weight_scales)
    narrow = product_inputs(torch, 2, 8, 136, 2, 64)
    with pytest.raises(pkg.MoeError, match="multiple of 16"):
        sampler.expert_product(*narrow, expert_offsets=offsets)
    with pytest.raises(ValueError):
        sampler.expert_product(values, scales.t(), weights, weight_scales, expert_offsets=offsets)
    with pytest.raises(TypeError):
        sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets.long())
    with pytest.raises(TypeError):
        sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        sampler.expert_product(values.cpu(), scales, weights, weight_scales, expert_offsets=offsets)
    store = torch.zeros(8 * 256 + 16, dtype=torch.uint8, device="cuda")
    with pytest.raises(pkg.MoeError, match="16-byte aligned"):
        sampler.expert_product(store[8:8 + 8 * 256].view(torch.float8_e4m3fn).view(8, 256), scales, weights, weight_scales, expert_offsets=offsets)
    assert sampler.expert_product(values[:0], scales[:, :0].contiguous(), weights, weight_scales, expert_offsets=offsets).shape == (0, 64)


# ---- combine --------------------------------------------------------------------------


def combine_reference(torch, rows, plan, tokens, base):
    out = torch.zeros((tokens, rows.shape[1]), dtype=torch.float64, device="cuda") if base is None else base.double()
    weighted = rows.double() * plan["weight"].double()[:, None]
    size = out.abs().index_add(0, plan["token"].long(), weighted.abs())
    return out.index_add(0, plan["token"].long(), weighted), size


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens,top_k,columns", [(1, 1, 1), (1, 8, 4096), (32, 4, 2880), (33, 6, 131), (200, 8, 72), (1500, 3, 264), (4, 40, 257), (700, 2, 1030), (3, 1, 8), (70, 100, 40), (2100, 1, 9),
                                                  (600, 8, 512)])
def test_combine(sampler, torch_cuda, dtype, tokens, top_k, columns):
    """A multiplication per route and a sum of top_k + 1 terms."""
    torch = torch_cuda
    plan = plan_of(torch, tokens, tokens, max(top_k, 12), top_k)
    rows = randn(torch, columns, tokens * top_k, columns).to(getattr(torch, dtype))
    for base in (None, randn(torch, 77, tokens, columns).to(rows.dtype)):
        want, size = combine_reference(torch, rows, plan, tokens, base)
        out = sampler.combine_routes(rows, plan["token"], plan["rank"], plan["weight"], tokens, top_k, base=base)
        bound = (top_k + 1) * U * size + rounding(torch, rows.dtype) * want.abs()
        assert bool(((out.double() - want).abs() <= bound).all())
        if base is not None:    # in place
            again = sampler.combine_routes(rows, plan["token"], plan["rank"], plan["weight"], tokens, top_k, base=base, out=base)
            assert again is base and torch.equal(again, out)
    assert sampler.expert_check() == 0


@pytest.mark.parametrize("routes_kept,tokens", [(150, 60), (0, 5), (2500, 900)])
def test_combine_partial_plans_and_strides(sampler, torch_cuda, routes_kept, tokens):
    """Routes that were dropped contribute nothing, whatever an earlier call left behind; rows inside a wider matrix."""
    torch = torch_cuda
    plan = plan_of(torch, 8, tokens, 16, 4)
    wide = randn(torch, 1, tokens * 4, 200)
    full = sampler.combine_routes(wide[:, 3:100], plan["token"], plan["rank"], plan["weight"], tokens, 4)
    want, size = combine_reference(torch, wide[:, 3:100], plan, tokens, None)
    assert bool(((full.double() - want).abs() <= 5 * U * size + U * want.abs()).all())
    kept = torch.randperm(tokens * 4, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")[:routes_kept]
    part = {name: plan[name][kept].contiguous() for name in ("token", "rank", "weight")}
    out = sampler.combine_routes(wide[kept], part["token"], part["rank"], part["weight"], tokens, 4)
    want, size = combine_reference(torch, wide[kept], part, tokens, None)
    assert bool(((out.double() - want).abs() <= 5 * U * size + U * want.abs()).all())


@pytest.mark.parametrize("tokens", [5, 129, 4000])
@pytest.mark.parametrize("top_k", [0, 4])
def test_combine_without_routes(sampler, torch_cuda, tokens, top_k):
    """A step whose routes were all dropped: every token gets its base, or zeros."""
    torch = torch_cuda
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rows, weight, base = torch.empty((0, 72), device="cuda"), torch.empty(0, device="cuda"), randn(torch, 3, tokens, 72)
    assert bool((sampler.combine_routes(rows, none, none, weight, tokens, top_k) == 0).all())
    assert torch.equal(sampler.combine_routes(rows, none, none, weight, tokens, top_k, base=base), base)


@pytest.mark.parametrize("tokens", [4, 3000])
def test_combine_bad_and_repeated_routes(sampler, pkg, torch_cuda, tokens):
    torch = torch_cuda
    rows = randn(torch, 1, 6, 50)
    token = torch.tensor([0, 1, tokens, 1, -1, 3], dtype=torch.int32, device="cuda")
    rank = torch.tensor([0, 0, 0, 0, 1, 2], dtype=torch.int32, device="cuda")     # (1, 0) twice, rank 2 of top 2
    weight = torch.tensor([0.5, 2.0, 1.0, 3.0, 1.0, 1.0], device="cuda")
    out = sampler.combine_routes(rows, token, rank, weight, tokens, 2)
    assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE and sampler.expert_check() == 0
    want = torch.zeros((tokens, 50), device="cuda")
    want[0], want[1] = 0.5 * rows[0], 3.0 * rows[3]
    assert torch.equal(out, want)


# ---- balance --------------------------------------------------------------------------

SCORES = ["softmax", "sigmoid", "sqrtsoftplus"]


def score_code(pkg, name):
    return {"softmax": pkg.ROUTER_SOFTMAX, "sigmoid": pkg.ROUTER_SIGMOID, "sqrtsoftplus": pkg.ROUTER_SQRT_SOFTPLUS}[name]


def probabilities(torch, logits, score):
    if score == "softmax":
        return torch.softmax(logits, dim=1)
    # not torch.sigmoid: its derivative s (1 - s) is zero from x = 37 on in 64 bits
    s = 1 / (1 + torch.exp(-logits)) if score == "sigmoid" else torch.nn.functional.softplus(logits, threshold=700.0).sqrt()
    return s / s.sum(dim=1, keepdim=True)


def balance_reference(torch, logits, plan, top_k, score, mask, coefficient, scale):
    """Counts, probabilities, loss, gradient by autograd in 64 bits, and the size of the gradient's two terms."""
    tokens, experts = logits.shape
    x = logits.double().requires_grad_()
    kept = torch.ones(tokens, dtype=torch.bool, device="cuda") if mask is None else mask.bool()
    n = int(kept.sum())
    counts = torch.bincount(plan["expert"][kept[plan["token"].long()]], minlength=experts)
    p = probabilities(torch, x, score)
    mean = p[kept].sum(dim=0) / n
    loss = coefficient * (counts.double() * experts / (top_k * n) * mean).sum()
    gradient, = torch.autograd.grad(loss * scale, x)
    g = (coefficient * scale / (top_k * n * n) * (experts * counts.double() - counts.sum())).abs()
    with torch.no_grad():
        if score == "softmax":
            slope = p
        else:
            s = torch.sigmoid(x)
            q = s if score == "sigmoid" else torch.nn.functional.softplus(x, threshold=700.0).sqrt()
            slope = (s * torch.sigmoid(-x) if score == "sigmoid" else s / (2 * q)) / q.sum(dim=1, keepdim=True)
        size = slope.abs() * (g + (p * g).sum(dim=1, keepdim=True))
    return counts, n, mean.detach(), float(loss.detach()), gradient, size


BALANCE = [(1, 1, 1), (1, 4, 2), (5, 7, 3), (61, 128, 4), (64, 32, 1), (100, 60, 8), (333, 160, 6), (70, 257, 5), (2000, 256, 8), (40, 1000, 4), (9, 1500, 16), (3, 4096, 8), (4097, 8, 2)]


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("tokens,experts,top_k", BALANCE)
def test_balance(sampler, pkg, torch_cuda, tokens, experts, top_k, score):
    """A score has at most 8 roundings, a token's sum `experts`, the division one: that is a probability's relative error; the sum
    over the tokens (all terms positive) adds `tokens`.  The loss adds a sum over the experts."""
    torch = torch_cuda
    logits = 1.5 * randn(torch, tokens, tokens, experts) + randn(torch, 3, experts)
    if tokens > 4:
        logits[2] *= 20          # saturated scores
        logits[3] = 0.25         # all equal
    plan = plan_of(torch, 8, tokens, experts, top_k)
    scale = torch.tensor([1.75], device="cuda")
    masks = [None]
    if tokens > 1:
        masks.append(torch.rand(tokens, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") < 0.7)
        masks[1][0] = True
    for mask in masks:
        counts, n, mean, loss, gradient, size = balance_reference(torch, logits, plan, top_k, score, mask, 0.01, 1.75)
        out = sampler.balance_loss(logits, plan["offsets"], plan["token"], top_k, score_function=score_code(pkg, score), token_mask=mask, coefficient=0.01)
        assert torch.equal(out.expert_tokens[:-1].long(), counts) and int(out.expert_tokens[-1]) == n
        rel = (experts + tokens + 16) * U
        assert bool(((out.expert_probability.double() - mean).abs() <= rel * mean + 1e-40).all())
        assert abs(float(out.loss) - loss) <= (rel + (experts + 8) * U) * abs(loss)
        got = sampler.balance_loss_backward(logits, out.expert_tokens, top_k, score_function=score_code(pkg, score), token_mask=mask, coefficient=0.01, loss_gradient=scale)
        bound = (2 * experts + 32) * U * size + 1e-40
        assert bool(((got.double() - gradient).abs() <= bound).all()), float(((got.double() - gradient).abs() / bound).max())
        if mask is not None:
            assert bool((got[~mask] == 0).all())
        again = sampler.balance_loss(logits, plan["offsets"], plan["token"], top_k, score_function=score_code(pkg, score), token_mask=mask, coefficient=0.01)
        assert torch.equal(out.loss, again.loss) and torch.equal(out.expert_probability, again.expert_probability)
    assert sampler.expert_check() == 0


@pytest.mark.parametrize("score", SCORES)
def test_balance_gradient_against_differences(sampler, pkg, torch_cuda, score):
    """Central differences of the loss in 64 bits, step 1e-3: what they leave of the third derivative is below 1e-5 of the sum of
    magnitudes, the fp32 gradient's own error far below that."""
    torch = torch_cuda
    logits, top_k = 1.2 * randn(torch, 6, 40, 24), 3
    plan = plan_of(torch, 8, 40, 24, top_k)
    out = sampler.balance_loss(logits, plan["offsets"], plan["token"], top_k, score_function=score_code(pkg, score), coefficient=1.0)
    gradient = sampler.balance_loss_backward(logits, out.expert_tokens, top_k, score_function=score_code(pkg, score), coefficient=1.0).double()
    share = out.expert_tokens[:-1].double() * 24 / (top_k * 40)
    for seed in range(3):
        direction = randn(torch, 50 + seed, 40, 24).double()
        ends = [(share * probabilities(torch, logits.double() + step * direction, score).mean(dim=0)).sum() for step in (1e-3, -1e-3)]
        slope = (ends[0] - ends[1]) / 2e-3
        assert abs(float((gradient * direction).sum() - slope)) <= 1e-5 * float((gradient.abs() * direction.abs()).sum())


def test_balance_without_tokens_and_with_dead_rows(sampler, pkg, torch_cuda):
    torch = torch_cuda
    plan = plan_of(torch, 8, 30, 16, 2)
    logits = randn(torch, 2, 30, 16)
    nobody = torch.zeros(30, dtype=torch.uint8, device="cuda")
    for score in SCORES:
        out = sampler.balance_loss(logits, plan["offsets"], plan["token"], 2, score_function=score_code(pkg, score), token_mask=nobody)
        assert float(out.loss) == 0 and bool((out.expert_tokens == 0).all()) and bool((out.expert_probability == 0).all())
        gradient = sampler.balance_loss_backward(logits, out.expert_tokens, 2, score_function=score_code(pkg, score), token_mask=nobody)
        assert bool((gradient == 0).all())
    # masked rows are not looked at
    spoiled = logits.clone()
    spoiled[4] = float("nan")
    spoiled[7] = float("inf")
    mask = torch.ones(30, dtype=torch.bool, device="cuda")
    mask[[4, 7]] = False
    for score in SCORES:
        code = score_code(pkg, score)
        clean, dirty = (sampler.balance_loss(x, plan["offsets"], plan["token"], 2, score_function=code, token_mask=mask) for x in (logits, spoiled))
        assert torch.equal(clean.loss, dirty.loss) and torch.equal(clean.expert_probability, dirty.expert_probability)
        got = sampler.balance_loss_backward(spoiled, dirty.expert_tokens, 2, score_function=code, token_mask=mask)
        assert bool(torch.isfinite(got).all()) and bool((got[~mask] == 0).all())
    # scores that all underflow count as zeros
    logits[5] = -300.0
    for score in ("sigmoid", "sqrtsoftplus"):
        code = score_code(pkg, score)
        out = sampler.balance_loss(logits, plan["offsets"], plan["token"], 2, score_function=code)
        kept = torch.ones(30, dtype=torch.bool, device="cuda")
        kept[5] = False
        mean = probabilities(torch, logits.double(), score)[kept].sum(dim=0) / 30
        assert bool(((out.expert_probability.double() - mean).abs() <= 80 * U * mean).all())
        gradient = sampler.balance_loss_backward(logits, out.expert_tokens, 2, score_function=code)
        assert bool((gradient[5] == 0).all()) and bool(torch.isfinite(gradient).all())


@pytest.mark.parametrize("score,tops", [("sigmoid", (-42.0, -80.0, -89.0, -95.0, -102.0)), ("sqrtsoftplus", (-84.0, -160.0, -176.0, -190.0, -204.0))])
@pytest.mark.parametrize("experts", [24, 256, 1000, 1500])
def test_balance_of_tiny_scores(sampler, pkg, torch_cuda, score, tops, experts):
    """Tokens whose scores are tiny or subnormal for every expert, down to where the largest is about to become zero.  Bounds as in
    test_balance, and 256 units more: the rounding of x - peak (at most 2^-24 of 256) is a score's relative error."""
    torch = torch_cuda
    logits = 1.5 * randn(torch, 21, 40, experts)
    for row, top in enumerate(tops):
        logits[row] += top - logits[row].max()
        logits[row + 8] = top       # all equal
    logits[20, 1:] = tops[1]        # one expert far above the others
    plan = plan_of(torch, 8, 40, experts, 3)
    counts, n, mean, loss, gradient, size = balance_reference(torch, logits, plan, 3, score, None, 0.01, 1.0)
    out = sampler.balance_loss(logits, plan["offsets"], plan["token"], 3, score_function=score_code(pkg, score), coefficient=0.01)
    rel = (experts + 40 + 16 + 256) * U
    assert bool(((out.expert_probability.double() - mean).abs() <= rel * mean + 1e-40).all())
    assert abs(float(out.loss) - loss) <= (rel + (experts + 8) * U) * abs(loss)
    got = sampler.balance_loss_backward(logits, out.expert_tokens, 3, score_function=score_code(pkg, score), coefficient=0.01)
    bound = (2 * experts + 32 + 512) * U * size + 1e-40
    assert bool(((got.double() - gradient).abs() <= bound).all()), float(((got.double() - gradient).abs() / bound).max())


def test_balance_does_not_follow_bad_plans(sampler, pkg, torch_cuda):
    torch = torch_cuda
    logits = randn(torch, 2, 30, 8)
    plan = plan_of(torch, 8, 30, 8, 2)
    for cuts in ([0, 9, 8, 10, 20, 30, 40, 50, 60], [0, 1, 2, 3, 4, 5, 6, 7, 61], [0, -1, 2, 3, 4, 5, 6, 7, 60]):
        out = sampler.balance_loss(logits, torch.tensor(cuts, dtype=torch.int32, device="cuda"), plan["token"], 2)
        assert sampler.expert_check() == pkg.EXPERT_FLAG_OFFSETS
        assert bool((out.expert_tokens[:-1] == 0).all()) and int(out.expert_tokens[-1]) == 30 and float(out.loss) == 0
    token = plan["token"].clone()
    token[0] = 30
    out = sampler.balance_loss(logits, plan["offsets"], token, 2)
    assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE and int(out.expert_tokens[:-1].sum()) == 59
    with pytest.raises(pkg.MoeError, match="score_function"):
        sampler.balance_loss(logits, plan["offsets"], plan["token"], 2, score_function=5)
    with pytest.raises(pkg.MoeError, match="finite"):
        sampler.balance_loss(logits, plan["offsets"], plan["token"], 2, coefficient=float("inf"))
    with pytest.raises(ValueError):
        sampler.balance_loss(logits, plan["offsets"], plan["token"], 3)


# ---- together -------------------------------------------------------------------------


def expert_layer(sampler, pkg, state, buffers):
    """Dispatch, first product, gate, second product, combine: what a host does per layer."""
    plan = sampler.router_dispatch(state["logits"], state["top_k"], out=buffers["plan"])
    sampler.quantize_rows(state["hidden"], route_token=plan.route_token, out=buffers["in"])
    sampler.expert_product(*buffers["in"], *state["first"], expert_offsets=plan.expert_offsets, out=buffers["inner"])
    sampler.quantize_rows(buffers["inner"], activation=pkg.ACTIVATION_SILU_GATE, out=buffers["gated"])
    sampler.expert_product(*buffers["gated"], *state["second"], expert_offsets=plan.expert_offsets, out=buffers["rows"])
    sampler.combine_routes(buffers["rows"], plan.route_token, plan.route_rank, plan.route_weight, state["hidden"].shape[0], state["top_k"],
                           base=state["hidden"], out=buffers["out"])
    return plan


def layer_state(torch, pkg, tokens, experts, top_k, columns, inner):
    _, _, w1, s1 = product_inputs(torch, 21, 1, columns, experts, 2 * inner)
    _, _, w2, s2 = product_inputs(torch, 22, 1, inner, experts, columns)
    state = dict(hidden=randn(torch, 1, tokens, columns).bfloat16(), logits=randn(torch, 2, tokens, experts), top_k=top_k,
                 first=(w1, s1 / (70 * columns ** 0.5)), second=(w2, s2 / (70 * inner ** 0.5)))
    routes = tokens * top_k
    empty = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")
    buffers = dict(plan=pkg.DispatchPlan(empty(experts + 1, dtype=torch.int32), empty(routes, dtype=torch.int32), empty(routes, dtype=torch.int32),
                                         empty(routes, dtype=torch.float32), torch.zeros(1, dtype=torch.int32, device="cuda")),
                   **{"in": (empty(routes, columns, dtype=torch.float8_e4m3fn), empty(blocks_of(columns), routes, dtype=torch.float32))},
                   inner=empty(routes, 2 * inner, dtype=torch.bfloat16), gated=(empty(routes, inner, dtype=torch.float8_e4m3fn), empty(blocks_of(inner), routes, dtype=torch.float32)),
                   rows=empty(routes, columns, dtype=torch.bfloat16), out=empty(tokens, columns, dtype=torch.bfloat16))
    return state, buffers


def assert_layer(torch, state, buffers, plan):
    """Every step against 64 bits on what the step before it really wrote."""
    tokens = state["hidden"].shape[0]
    routes = dict(offsets=plan.expert_offsets, token=plan.route_token, weight=plan.route_weight)
    values, scales = quantize_reference(torch, state["hidden"][plan.route_token.long()])
    assert torch.equal(buffers["in"][0].float().cpu(), values) and torch.equal(buffers["in"][1].cpu(), scales)
    assert_product(torch, buffers["inner"], product_reference(torch, *buffers["in"], *state["first"], plan.expert_offsets), values.shape[1])
    columns = buffers["gated"][0].shape[1]
    gate, up = buffers["inner"].double()[:, :columns], buffers["inner"].double()[:, columns:]
    h = gate * torch.sigmoid(gate) * up
    wide = buffers["gated"][1].double().t().repeat_interleave(128, dim=1)[:, :columns]
    assert bool(((buffers["gated"][0].double() * wide - h).abs() <= (2.0 ** -4 + 16 * U) * h.abs().clamp_min(2.0 ** -6 * wide)).all())
    assert_product(torch, buffers["rows"], product_reference(torch, *buffers["gated"], *state["second"], plan.expert_offsets), columns)
    want, size = combine_reference(torch, buffers["rows"], routes, tokens, state["hidden"])
    assert bool(((buffers["out"].double() - want).abs() <= (state["top_k"] + 1) * U * size + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("tokens,experts,top_k,columns,inner", [(1, 16, 4, 256, 144), (32, 64, 4, 720, 336), (300, 8, 2, 512, 256)])
def test_expert_layer(sampler, pkg, torch_cuda, tokens, experts, top_k, columns, inner):
    torch = torch_cuda
    state, buffers = layer_state(torch, pkg, tokens, experts, top_k, columns, inner)
    plan = expert_layer(sampler, pkg, state, buffers)
    assert_layer(torch, state, buffers, plan)
    assert sampler.expert_check() == 0


def test_expert_layer_in_a_graph(pkg, torch_cuda):
    """Captured once, replayed on new inputs, on a stream of its own; eager calls of the same handle in between."""
    torch = torch_cuda
    state, buffers = layer_state(torch, pkg, 24, 16, 2, 272, 160)
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            expert_layer(handle, pkg, state, buffers)       # scratch is allocated before the capture
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan = expert_layer(handle, pkg, state, buffers)
        for seed in range(4):
            with torch.cuda.stream(side):
                state["hidden"].copy_(randn(torch, 100 + seed, 24, 272))
                state["logits"].copy_(randn(torch, 200 + seed, 24, 16))
                graph.replay()
            side.synchronize()
            assert_layer(torch, state, buffers, plan)
            got = buffers["out"].clone()
            with torch.cuda.stream(side):
                expert_layer(handle, pkg, state, buffers)
            side.synchronize()
            assert torch.equal(got, buffers["out"])
        assert handle.expert_check() == 0
    finally:
        handle.close()


def test_captured_graphs_outlive_larger_calls(pkg, torch_cuda):
    """Scratch that a graph was captured with stays when a later call needs more; the larger call and the graph do not disturb each other."""
    torch = torch_cuda
    handle = pkg.Sampler(max_rows=1, max_vocab=64)
    try:
        def inputs(tokens, experts, seed):
            plan = plan_of(torch, seed, tokens, experts, 8)
            return plan, randn(torch, seed, tokens * 8, 48), randn(torch, seed + 1, tokens, 2048), randn(torch, seed + 2, tokens, experts)

        def run(plan, rows, source, logits, out):
            tokens = source.shape[0]
            handle.combine_routes(rows, plan["token"], plan["rank"], plan["weight"], tokens, 8, out=out["sum"])
            handle.quantize_rows(source, route_token=plan["token"], out=out["quantized"])
            handle.balance_loss(logits, plan["offsets"], plan["token"], 8, out=out["balance"])

        def outputs(tokens, experts):
            return dict(sum=torch.zeros((tokens, 48), device="cuda"),
                        quantized=(torch.zeros((tokens * 8, 2048), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((16, tokens * 8), device="cuda")),
                        balance=pkg.BalanceLoss(torch.zeros(1, device="cuda"), torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.zeros(experts, device="cuda")))

        small, large = inputs(2100, 16, 1), inputs(4000, 200, 2)
        out, want, other = outputs(2100, 16), outputs(2100, 16), outputs(4000, 200)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*small, want)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(*small, out)
        first = None
        for _ in range(3):
            with torch.cuda.stream(side):
                graph.replay()
                run(*large, other)
            side.synchronize()
            assert torch.equal(out["sum"], want["sum"])
            assert torch.equal(out["quantized"][0].view(torch.uint8), want["quantized"][0].view(torch.uint8)) and torch.equal(out["quantized"][1], want["quantized"][1])
            assert torch.equal(out["balance"].loss, want["balance"].loss) and torch.equal(out["balance"].expert_tokens, want["balance"].expert_tokens)
            now = (other["sum"].clone(), other["quantized"][0].view(torch.uint8).clone(), other["balance"].loss.clone())
            assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
            first = now
            out["sum"].zero_()
            other["sum"].zero_()
            torch.cuda.synchronize()
        assert handle.expert_check() == 0
    finally:
        handle.close()


def test_layer_behind_a_refused_dispatch(sampler, pkg, torch_cuda):
    """Plan arrays that no dispatch has filled: every call stays inside its buffers, and the check says that something was wrong."""
    torch = torch_cuda
    generator = torch.Generator(device="cuda").manual_seed(9)
    tokens, experts, top_k, columns, outputs = 300, 8, 4, 256, 384
    routes = tokens * top_k
    x = randn(torch, 1, tokens, columns)
    weights = (randn(torch, 2, experts, outputs, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    weight_scales = torch.ones((experts, blocks_of(outputs), blocks_of(columns)), device="cuda")
    for low, high in ((-2 ** 31, 2 ** 31 - 1), (0, 2 * tokens), (0, 2 * routes)):
        offsets, token, rank = (torch.randint(low, high, (n,), generator=generator, device="cuda").int() for n in (experts + 1, routes, routes))
        store = torch.full((routes + 16, outputs), -7.0, device="cuda")
        total_store = torch.full((tokens + 16, outputs), -7.0, device="cuda")
        values, scales = sampler.quantize_rows(x, route_token=token)
        sampler.expert_product(values, scales, weights, weight_scales, expert_offsets=offsets, out=store[8:-8])
        sampler.combine_routes(store[8:-8], token, rank, torch.ones(routes, device="cuda"), tokens, top_k, out=total_store[8:-8])
        out = sampler.balance_loss(randn(torch, 3, tokens, experts), offsets, token, top_k)
        assert sampler.expert_check() == pkg.EXPERT_FLAG_TOKEN_RANGE | pkg.EXPERT_FLAG_OFFSETS
        assert int(out.expert_tokens[:-1].sum()) == 0
        for part in (store[:8], store[-8:], total_store[:8], total_store[-8:], store[8:-8]):
            assert bool((part == -7).all())    # the product did not follow such offsets


def test_two_handles_on_two_streams(pkg, torch_cuda):
    torch = torch_cuda
    handles = [pkg.Sampler(max_rows=1, max_vocab=64) for _ in range(2)]
    try:
        states = [layer_state(torch, pkg, tokens, 16, 4, 512, 256) for tokens in (48, 200)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        plans = [None, None]
        for _ in range(10):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    plans[i] = expert_layer(handles[i], pkg, *states[i])
        torch.cuda.synchronize()
        for i in range(2):
            assert_layer(torch, *states[i], plans[i])
            assert handles[i].expert_check() == 0
    finally:
        for handle in handles:
            handle.close()


def test_offsets_beyond_32_bits(sampler, torch_cuda):
    """The last rows of arrays that hold more than 2^32 values or bytes."""
    torch = torch_cuda
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    rows, columns = 530000, 8208
    source = torch.zeros((rows, columns), dtype=torch.bfloat16, device="cuda")
    source[-3:] = randn(torch, 1, 3, columns).bfloat16()
    values, scales = sampler.quantize_rows(source)
    want_values, want_scales = quantize_reference(torch, source[-3:])
    assert torch.equal(values[-3:].float().cpu(), want_values) and torch.equal(scales[:, -3:].cpu(), want_scales)
    assert bool((scales[:, :-3] == 0).all())
    # combine: the routed rows of the last tokens
    tokens = 4
    token = torch.full((rows,), tokens, dtype=torch.int32, device="cuda")     # out of range: left out
    token[-3:] = torch.tensor([3, 0, 3], dtype=torch.int32, device="cuda")
    rank = torch.zeros(rows, dtype=torch.int32, device="cuda")
    rank[-1] = 1
    weight = torch.full((rows,), 0.5, device="cuda")
    out = sampler.combine_routes(source, token, rank, weight, tokens, 2)
    sampler.expert_check()
    want = torch.zeros((tokens, columns), device="cuda")
    want[3], want[0] = 0.5 * source[-3].float() + 0.5 * source[-1].float(), 0.5 * source[-2].float()
    assert bool(((out.float() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * U * source.float()[-3:].abs().sum(dim=0)).all())
    del source, values, scales, token, rank, weight
    # weights of more than 2^32 bytes
    experts, outputs, columns = 70, 8192, 8208
    weights = torch.zeros((experts, outputs, columns), dtype=torch.float8_e4m3fn, device="cuda")
    weights[-1] = (randn(torch, 2, outputs, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    weight_scales = torch.ones((experts, 64, 65), device="cuda")
    for count in (2, 90):
        x = (randn(torch, 3, count, columns) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        x_scales = torch.ones((65, count), device="cuda")
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        offsets[-1] = count
        out = sampler.expert_product(x, x_scales, weights, weight_scales, expert_offsets=offsets, out_dtype=torch.float32)
        one = torch.tensor([0, count], dtype=torch.int32, device="cuda")
        assert_product(torch, out, product_reference(torch, x, x_scales, weights[-1:], weight_scales[-1:], one), columns)
    del weights
    torch.cuda.empty_cache()


def test_calls_follow_a_producer_that_lets_them_start_early(sampler, pkg, torch_cuda, test_kernels):
    """Inputs that the kernel before writes after it has let its successors start (see tests/test_launch_order.py)."""
    from test_launch_order import produce_late
    torch = torch_cuda
    rows, columns, outputs = 40, 512, 256
    source = randn(torch, 1, rows, columns)
    late = torch.zeros_like(source)
    want = sampler.quantize_rows(source)
    produce_late(test_kernels, torch, source, late)
    got = sampler.quantize_rows(late)
    assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got[1], want[1])
    values, scales, weights, weight_scales = product_inputs(torch, 3, rows, columns, 1, outputs)
    expected = sampler.expert_product(values, scales, weights, weight_scales)
    for name, tensor in (("values", values), ("scales", scales), ("weights", weights), ("weight_scales", weight_scales)):
        inputs = dict(values=values, scales=scales, weights=weights, weight_scales=weight_scales)
        inputs[name] = torch.zeros_like(tensor.view(torch.uint8)).view(tensor.dtype)
        torch.cuda.synchronize()
        produce_late(test_kernels, torch, tensor, inputs[name])
        assert torch.equal(sampler.expert_product(**inputs), expected), name
    plan = plan_of(torch, 4, 10, 8, 4)
    full = sampler.combine_routes(source, plan["token"], plan["rank"], plan["weight"], 10, 4)
    late.zero_()
    produce_late(test_kernels, torch, source, late)
    assert torch.equal(sampler.combine_routes(late, plan["token"], plan["rank"], plan["weight"], 10, 4), full)
    logits = randn(torch, 5, 10, 8)
    expected = sampler.balance_loss(logits, plan["offsets"], plan["token"], 4)
    gradient = sampler.balance_loss_backward(logits, expected.expert_tokens, 4)
    late = torch.zeros_like(logits)
    torch.cuda.synchronize()
    produce_late(test_kernels, torch, logits, late)
    assert torch.equal(sampler.balance_loss(late, plan["offsets"], plan["token"], 4).loss, expected.loss)
    late.zero_()
    torch.cuda.synchronize()
    produce_late(test_kernels, torch, logits, late)
    assert torch.equal(sampler.balance_loss_backward(late, expected.expert_tokens, 4), gradient)
