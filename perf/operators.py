"""The operators around the experts' products, each in a plain form and as a call of the library.

After the router has grouped the routes of a step by expert, a mixture-of-experts layer quantises the
rows of the routed tokens, multiplies each expert's rows with its weights, brings the results back to
the tokens, and watches (or trains) how evenly the experts are used:

  quantize   rows to e4m3 with one fp32 scale per block of 128 columns, gathered by route or gated (SiLU) on the way
  product    the experts' products in e4m3, fp32 scales per 1 x 128 block of a row and 128 x 128 block of a weight
  combine    the weighted sum of a token's routed rows, onto a base
  balance    tokens per expert, mean router probabilities, the balance loss and its gradient with respect to the logits
  layer      all of them but the last, as one expert layer of a decode step

Shapes are those of the benchmark's router workloads (4096 tokens x 256 experts x top 8 x 4096 columns, 32 tokens x
128 experts x top 4 x 2880 columns) and generic ones between one token and a long batch.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 128        # columns that share a scale
E4M3_MAX = 448.0   # largest finite e4m3 value
E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # Prefill: the rows of 4096 tokens, gathered once per route and quantised for the experts' first product.
        dict(name="quantize_gather_prefill", kind="quantize", tokens=4096, top_k=8, columns=4096, dtype="bf16", gate=False),
        # Decode: gate and up halves of the first product become the quantised input of the second; 2880 ends in half a block.
        dict(name="quantize_gate_decode", kind="quantize", tokens=32, top_k=4, columns=2880, dtype="f32", gate=True),
        # One Session decoding alone: eight experts with one row each, all weight traffic.
        dict(name="product_1_token", kind="product", tokens=1, top_k=8, experts=256, columns=4096, outputs=4096, out="bf16"),
        # A decode step of 32 Sessions: most experts are hit by a row or two.
        dict(name="product_decode", kind="product", tokens=32, top_k=4, experts=128, columns=2880, outputs=5760, out="bf16"),
        # Prefill: about 128 rows an expert, every expert's weights read once.
        dict(name="product_prefill", kind="product", tokens=4096, top_k=8, experts=256, columns=4096, outputs=4096, out="bf16"),
        # A dense product (a shared expert) over a chunk of tokens that no tile divides, fp32 out.
        dict(name="product_dense", kind="product", tokens=4099, top_k=1, experts=1, columns=4096, outputs=2880, out="f32"),
        # Prefill: eight routed rows a token, summed onto the shared expert's output.
        dict(name="combine_prefill", kind="combine", tokens=4096, top_k=8, columns=4096, dtype="bf16", base=True),
        # Decode: four routed rows a token, fp32.
        dict(name="combine_decode", kind="combine", tokens=32, top_k=4, columns=2880, dtype="f32", base=False),
        # Balance figures of one small batch.
        dict(name="balance_small", kind="balance", tokens=61, experts=128, top_k=4, score="softmax", mask=False),
        # A long padded batch: one token in nine is padding.
        dict(name="balance_long", kind="balance", tokens=65536, experts=256, top_k=8, score="sigmoid", mask=True),
        # The whole expert layer of a decode step.
        dict(name="layer_decode", kind="layer", tokens=32, top_k=4, experts=128, columns=2880, inner=2880),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    kind = rng.choice(["quantize", "product", "product", "product", "combine", "balance", "layer"])
    if kind == "quantize":
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), top_k=rng.randint(1, 8), columns=8 * _log_int(rng, 8, 512), dtype=rng.choice(["f32", "bf16"]), gate=rng.random() < 0.5)
    if kind == "product":
        experts, top_k = rng.choice([(1, 1), (8, 2), (32, 4), (64, 6), (128, 4), (160, 6), (256, 8)])
        tokens, columns, outputs = _log_int(rng, 1, 4096), 16 * _log_int(rng, 8, 256), _log_int(rng, 100, 4096)
        return dict(kind=kind, tokens=tokens, top_k=top_k, experts=experts, columns=columns, outputs=outputs, out=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "combine":
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), top_k=rng.randint(1, 8), columns=_log_int(rng, 64, 4096), dtype=rng.choice(["f32", "bf16"]), base=rng.random() < 0.5)
    if kind == "balance":
        return dict(kind=kind, tokens=_log_int(rng, 1, 65536), experts=rng.choice([8, 32, 60, 128, 160, 256]), top_k=rng.randint(1, 8),
                    score=rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]), mask=rng.random() < 0.5)
    return dict(kind=kind, tokens=_log_int(rng, 1, 64), top_k=rng.choice([2, 4]), experts=rng.choice([16, 32, 64, 128]), columns=16 * rng.randint(16, 180), inner=16 * rng.randint(16, 180))


# ---- inputs ---------------------------------------------------------------------------------------------


def _activations(generator, rows, columns):
    """Normal rows with a few channels that are eight times as large, as hidden states have them."""
    x = torch.randn((rows, columns), generator=generator, device=DEVICE)
    loud = torch.rand(columns, generator=generator, device=DEVICE) < 1 / 64
    return torch.where(loud, 8 * x, x)


def _blocks(columns):
    return (columns + BLOCK - 1) // BLOCK


def _weights(generator, experts, outputs, columns):
    """e4m3 weights [experts, outputs, columns] of standard deviation 1 / sqrt(columns), and their block scales."""
    values = torch.empty((experts, outputs, columns), dtype=E4M3, device=DEVICE)
    chunk = max(1, (1 << 28) // (outputs * columns))
    for first in range(0, experts, chunk):
        part = values[first:first + chunk]
        part.copy_(torch.randn(part.shape, generator=generator, device=DEVICE, dtype=torch.bfloat16).mul_(100).clamp_(-E4M3_MAX, E4M3_MAX))
    spread = torch.rand((experts, _blocks(outputs), _blocks(columns)), generator=generator, device=DEVICE)
    return values, (0.6 + 0.8 * spread) / (100 * math.sqrt(columns))


def _routing(generator, tokens, experts, top_k):
    """A plan in expert order as router_dispatch gives it: offsets, token, rank, weight.  Some experts are more popular."""
    taste = torch.randn((tokens, experts), generator=generator, device=DEVICE) + 0.5 * torch.randn(experts, generator=generator, device=DEVICE)
    best = taste.topk(top_k, dim=1)
    weight = torch.softmax(best.values, dim=1).reshape(-1)
    order = best.indices.reshape(-1).sort(stable=True)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEVICE)
    offsets[1:] = torch.bincount(order.values, minlength=experts).cumsum(0)
    route = order.indices
    return dict(expert_offsets=offsets, route_token=(route // top_k).to(torch.int32), route_rank=(route % top_k).to(torch.int32),
                route_weight=weight[route].contiguous(), expert=order.values)


def _packing(plan, experts):
    """The plain product's view of a plan: the experts that have rows, each row's place in its expert's batch, the largest batch."""
    counts = plan["expert_offsets"].diff()
    active = counts.nonzero()[:, 0]
    rank_of = torch.zeros(experts, dtype=torch.int64, device=DEVICE)
    rank_of[active] = torch.arange(active.numel(), device=DEVICE)
    place = torch.arange(plan["expert"].numel(), device=DEVICE) - plan["expert_offsets"][plan["expert"]]
    return dict(active=active, batch=rank_of[plan["expert"]], place=place, most=int(counts.max()))


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, tokens, top_k = case["kind"], case["tokens"], case["top_k"]
    state = dict(case=case)
    if kind == "quantize":
        dtype = TYPES[case["dtype"]]
        if case["gate"]:
            state["source"] = torch.randn((tokens * top_k, 2 * case["columns"]), generator=generator, device=DEVICE).mul_(2).to(dtype)
        else:
            state["source"] = _activations(generator, tokens, case["columns"]).to(dtype)
            state["plan"] = _routing(generator, tokens, max(64, top_k), top_k)
    elif kind == "product":
        experts = case["experts"]
        state["plan"] = _routing(generator, tokens, experts, top_k)
        state["packing"] = _packing(state["plan"], experts)
        values, scales = plain_quantize(_activations(generator, tokens, case["columns"]))
        state["values"] = values.view(torch.uint8)[state["plan"]["route_token"]].view(E4M3)
        state["scales"] = scales[:, state["plan"]["route_token"]].contiguous()
        state["weights"], state["weight_scales"] = _weights(generator, experts, case["outputs"], case["columns"])
    elif kind == "combine":
        dtype = TYPES[case["dtype"]]
        state["plan"] = _routing(generator, tokens, max(64, top_k), top_k)
        state["rows"] = torch.randn((tokens * top_k, case["columns"]), generator=generator, device=DEVICE).to(dtype)
        state["base"] = torch.randn((tokens, case["columns"]), generator=generator, device=DEVICE).to(dtype) if case["base"] else None
    elif kind == "balance":
        state["logits"] = torch.randn((tokens, case["experts"]), generator=generator, device=DEVICE) * 1.5 + 0.7 * torch.randn(case["experts"], generator=generator, device=DEVICE)
        state["mask"] = torch.rand(tokens, generator=generator, device=DEVICE) >= 1 / 9 if case["mask"] else None
        best = state["logits"].topk(top_k, dim=1).indices.reshape(-1).sort(stable=True)
        offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device=DEVICE)
        offsets[1:] = torch.bincount(best.values, minlength=case["experts"]).cumsum(0)
        state["plan"] = dict(expert_offsets=offsets, route_token=(best.indices // top_k).to(torch.int32), expert=best.values)
        state["coefficient"] = 0.01
        state["loss_gradient"] = torch.rand(1, generator=generator, device=DEVICE) + 0.5
    else:
        experts, columns, inner = case["experts"], case["columns"], case["inner"]
        state["plan"] = _routing(generator, tokens, experts, top_k)
        state["packing"] = _packing(state["plan"], experts)
        state["hidden"] = _activations(generator, tokens, columns).bfloat16()
        state["first"] = _weights(generator, experts, 2 * inner, columns)
        state["second"] = _weights(generator, experts, columns, inner)
    return state


# ---- plain forms ----------------------------------------------------------------------------------------


def _by_block(x):
    """[rows, columns] as [rows, blocks, 128], zeros behind the last column."""
    rows, columns = x.shape
    return torch.nn.functional.pad(x, (0, _blocks(columns) * BLOCK - columns)).view(rows, -1, BLOCK)


def plain_quantize(source, route_token=None, gate=False):
    x = source.float()
    if route_token is not None:
        x = x[route_token]
    if gate:
        half = x.shape[1] // 2
        x = x[:, :half] / (1 + torch.exp(-x[:, :half])) * x[:, half:]
    blocks = _by_block(x)
    # a tensor divides (one rounding, which decides ties below); a plain number would be multiplied by its reciprocal
    scales = blocks.abs().amax(dim=2) / torch.full((), E4M3_MAX, device=DEVICE)
    values = torch.where(scales[:, :, None] > 0, blocks / scales[:, :, None], 0.0).clamp(-E4M3_MAX, E4M3_MAX)
    return values.reshape(x.shape[0], -1)[:, :x.shape[1]].to(E4M3), scales.t().contiguous()


def _wide(scales, rows, columns, down):
    """Block scales spread over the values they belong to."""
    return scales.repeat_interleave(down, dim=-2)[..., :rows, :].repeat_interleave(BLOCK, dim=-1)[..., :columns]


def plain_product(values, scales, weights, weight_scales, packing, dtype):
    rows, columns = values.shape
    active, batch, place, most = packing["active"], packing["batch"], packing["place"], packing["most"]
    x = torch.zeros((active.numel(), most, columns), device=DEVICE)
    x[batch, place] = values.float() * _wide(scales.t(), rows, columns, 1)
    w = weights.view(torch.uint8)[active].view(E4M3).float()
    w *= _wide(weight_scales[active], w.shape[1], columns, BLOCK)
    return torch.bmm(x, w.transpose(1, 2))[batch, place].to(dtype)


def plain_combine(rows, plan, tokens, top_k, base):
    by_rank = torch.empty((tokens, top_k, rows.shape[1]), device=DEVICE)
    by_rank[plan["route_token"], plan["route_rank"]] = rows.float() * plan["route_weight"][:, None]
    total = by_rank.sum(dim=1)
    return (total if base is None else base.float() + total).to(rows.dtype)


def _probabilities(logits, score):
    """Router scores that sum to one over the experts, and the derivative of each score before that (None: softmax)."""
    if score == "softmax":
        e = torch.exp(logits - logits.amax(dim=1, keepdim=True))
        return e / e.sum(dim=1, keepdim=True), None
    if score == "sigmoid":
        s = 1 / (1 + torch.exp(-logits))
        slope = s * (1 - s)
    else:
        s = torch.sqrt(torch.log1p(torch.exp(-logits.abs())) + logits.clamp_min(0))
        slope = 1 / (1 + torch.exp(-logits)) / (2 * s)
    total = s.sum(dim=1, keepdim=True)
    return s / total, slope / total


def plain_balance(logits, plan, top_k, score, mask, coefficient, loss_gradient):
    tokens, experts = logits.shape
    kept = torch.ones(tokens, dtype=torch.bool, device=DEVICE) if mask is None else mask
    counted = kept.sum()
    most = counted.clamp_min(1)   # a batch of padding alone has the loss zero
    counts = torch.zeros(experts, dtype=torch.int64, device=DEVICE).index_add_(0, plan["expert"], kept[plan["route_token"]].long())
    p, slope = _probabilities(logits.double(), score)   # the gradient is a difference of nearly equal sums
    p = torch.where(kept[:, None], p, 0.0)
    probability = p.sum(dim=0) / most
    share = counts.double() * experts / (top_k * most)
    loss = coefficient * (share * probability).sum()
    g = loss_gradient.double() * coefficient * share / most
    gradient = (g - (p * g).sum(dim=1, keepdim=True)) * (p if slope is None else torch.where(kept[:, None], slope, 0.0))
    return dict(loss=loss.float().reshape(1), tokens=torch.cat([counts, counted[None]]).to(torch.int32), probability=probability.float(),
                gradient=torch.where(kept[:, None], gradient, 0.0).float())


# ---- one pass -------------------------------------------------------------------------------------------

_handle = None


def _library():
    """The package and the handle that a program keeps for its stream."""
    global _handle
    from __graft_entry__ import load_package
    package = load_package()
    if _handle is None:
        _handle = package.Sampler(max_rows=1, max_vocab=1024)
    return package, _handle


def run(state):
    case = state["case"]
    kind, plan = case["kind"], state.get("plan")
    if own:
        package, handle = _library()
        if kind == "quantize":
            if case["gate"]:
                values, scales = handle.quantize_rows(state["source"], activation=package.ACTIVATION_SILU_GATE)
            else:
                values, scales = handle.quantize_rows(state["source"], route_token=plan["route_token"])
            return dict(values=values, scales=scales)
        if kind == "product":
            return handle.expert_product(state["values"], state["scales"], state["weights"], state["weight_scales"],
                                         expert_offsets=plan["expert_offsets"] if case["experts"] > 1 else None, out_dtype=TYPES[case["out"]])
        if kind == "combine":
            return handle.combine_routes(state["rows"], plan["route_token"], plan["route_rank"], plan["route_weight"], case["tokens"], case["top_k"], base=state["base"])
        if kind == "balance":
            score = {"softmax": package.ROUTER_SOFTMAX, "sigmoid": package.ROUTER_SIGMOID, "sqrtsoftplus": package.ROUTER_SQRT_SOFTPLUS}[case["score"]]
            out = handle.balance_loss(state["logits"], plan["expert_offsets"], plan["route_token"], case["top_k"], score_function=score,
                                      token_mask=state["mask"], coefficient=state["coefficient"])
            gradient = handle.balance_loss_backward(state["logits"], out.expert_tokens, case["top_k"], score_function=score, token_mask=state["mask"],
                                                    coefficient=state["coefficient"], loss_gradient=state["loss_gradient"])
            return dict(loss=out.loss, tokens=out.expert_tokens, probability=out.expert_probability, gradient=gradient)
        values, scales = handle.quantize_rows(state["hidden"], route_token=plan["route_token"])
        inner = handle.expert_product(values, scales, *state["first"], expert_offsets=plan["expert_offsets"])
        values, scales = handle.quantize_rows(inner, activation=package.ACTIVATION_SILU_GATE)
        rows = handle.expert_product(values, scales, *state["second"], expert_offsets=plan["expert_offsets"])
        return handle.combine_routes(rows, plan["route_token"], plan["route_rank"], plan["route_weight"], case["tokens"], case["top_k"], base=state["hidden"])
    if kind == "quantize":
        values, scales = plain_quantize(state["source"], plan["route_token"] if plan else None, case["gate"])
        return dict(values=values, scales=scales)
    if kind == "product":
        return plain_product(state["values"], state["scales"], state["weights"], state["weight_scales"], state["packing"], TYPES[case["out"]])
    if kind == "combine":
        return plain_combine(state["rows"], plan, case["tokens"], case["top_k"], state["base"])
    if kind == "balance":
        return plain_balance(state["logits"], plan, case["top_k"], case["score"], state["mask"], state["coefficient"], state["loss_gradient"])
    values, scales = plain_quantize(state["hidden"], plan["route_token"])
    inner = plain_product(values, scales, *state["first"], state["packing"], torch.bfloat16)
    values, scales = plain_quantize(inner, gate=True)
    rows = plain_product(values, scales, *state["second"], state["packing"], torch.bfloat16)
    return plain_combine(rows, plan, case["tokens"], case["top_k"], state["hidden"])


def _product_work(rows, active, columns, outputs, element):
    read = active * (outputs * columns + 4 * _blocks(outputs) * _blocks(columns)) + rows * (columns + 4 * _blocks(columns))
    return read + rows * outputs * element, 2 * rows * outputs * columns


def work(case):
    kind, tokens, top_k = case["kind"], case["tokens"], case["top_k"]
    rows, columns = tokens * top_k, case.get("columns", 0)
    if kind == "quantize":
        element = 4 if case["dtype"] == "f32" else 2
        read = rows * 2 * columns * element if case["gate"] else tokens * columns * element + 4 * rows
        return dict(bytes=read + rows * columns + 4 * rows * _blocks(columns), flops=rows * columns * (8 if case["gate"] else 3))
    if kind in ("product", "layer"):
        experts = case["experts"]
        active = experts * (1 - (1 - top_k / experts) ** tokens)   # experts that get a row, on average
        if kind == "product":
            moved, flops = _product_work(rows, active, columns, case["outputs"], 4 if case["out"] == "f32" else 2)
            return dict(bytes=moved, flops=flops)
        inner = case["inner"]
        first, second = _product_work(rows, active, columns, 2 * inner, 0), _product_work(rows, active, inner, columns, 0)
        weights = first[0] + second[0] - rows * (columns + 4 * _blocks(columns) + inner + 4 * _blocks(inner))
        return dict(bytes=weights + 4 * tokens * columns + 12 * rows, flops=first[1] + second[1])
    if kind == "combine":
        element = 4 if case["dtype"] == "f32" else 2
        return dict(bytes=(rows + tokens * (2 if case["base"] else 1)) * columns * element + 12 * rows, flops=2 * rows * columns)
    # the logits are read once; the gradient is written once
    return dict(bytes=tokens * case["experts"] * 8 + 4 * rows + (tokens if case["mask"] else 0), flops=tokens * case["experts"] * 16)


# ---- in 64 bits, from the definitions -------------------------------------------------------------------


def _nearest(x, digits, lowest):
    """x rounded to `digits` binary digits, ties to even, digits fixed below 2^lowest."""
    exponent = torch.frexp(x).exponent - 1
    step = torch.ldexp(torch.ones_like(x), exponent.clamp_min(lowest) - (digits - 1))
    return torch.round(x / step) * step


def _exact_quantize(x):
    """Scales and unrounded values in their units, one block of columns after the other."""
    scales, values = [], []
    for first in range(0, x.shape[1], BLOCK):
        part = x[:, first:first + BLOCK]
        scale = part.abs().max(dim=1).values / 448
        scales.append(scale)
        values.append(part / torch.where(scale > 0, scale, 1.0)[:, None])
    return torch.cat(values, dim=1), torch.stack(scales)


def _stored_quantize(x):
    """The values and scales that are stored: a scale is an fp32 number, and a value divided by it one before it becomes e4m3.  That
    decides ties, which are common among bf16 rows (448 x / maximum is often a short fraction)."""
    scales = _exact_quantize(x)[1].float().double()
    column = torch.arange(x.shape[1], device=DEVICE) // BLOCK
    wide = scales[column].t()
    units = (x / torch.where(wide > 0, wide, 1.0)).float().double()
    return _nearest(units.clamp(-448, 448), 4, -6), scales


def _exact_gate(x):
    half = x.shape[1] // 2
    return x[:, :half] * torch.special.expit(x[:, :half]) * x[:, half:]


def _exact_product(values, scales, weights, weight_scales, offsets):
    """Expert by expert: the scaled rows times the scaled weights."""
    out = torch.empty((values.shape[0], weights.shape[1]), dtype=torch.float64, device=DEVICE)
    column = torch.arange(values.shape[1], device=DEVICE) // BLOCK
    row = torch.arange(weights.shape[1], device=DEVICE) // BLOCK
    bounds = offsets.tolist()
    for expert in range(len(bounds) - 1):
        begin, end = bounds[expert], bounds[expert + 1]
        if begin < end:
            x = values[begin:end].double() * scales[:, begin:end].double()[column].t()
            w = weights[expert].double() * weight_scales[expert].double()[row][:, column]
            out[begin:end] = x @ w.t()
    return out


def _exact_combine(rows, plan, tokens, base):
    out = torch.zeros((tokens, rows.shape[1]), dtype=torch.float64, device=DEVICE) if base is None else base.double()
    return out.index_add(0, plan["route_token"].long(), rows.double() * plan["route_weight"].double()[:, None])


def exact(case, seed):
    state = prepare(case, seed)
    kind, plan = case["kind"], state.get("plan")
    if kind == "quantize":
        x = state["source"].double()
        values, scales = _exact_quantize(_exact_gate(x) if case["gate"] else x[plan["route_token"].long()])
        return dict(values=values, scales=scales)
    if kind == "product":
        return _exact_product(state["values"], state["scales"], state["weights"], state["weight_scales"], plan["expert_offsets"])
    if kind == "combine":
        return _exact_combine(state["rows"], plan, case["tokens"], state["base"])
    if kind == "balance":
        logits = state["logits"].double().requires_grad_()
        kept = torch.ones(case["tokens"], device=DEVICE, dtype=torch.bool) if state["mask"] is None else state["mask"]
        counted = int(kept.sum())
        valid = plan["expert"][kept[plan["route_token"].long()]]
        counts = torch.bincount(valid, minlength=case["experts"])
        if counted == 0:
            return None
        if case["score"] == "softmax":
            p = torch.softmax(logits, dim=1)
        else:
            s = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.nn.functional.softplus(logits).sqrt()
            p = s / s.sum(dim=1, keepdim=True)
        probability = p[kept].mean(dim=0)
        loss = state["coefficient"] * (counts.double() / (case["top_k"] * counted) * case["experts"] * probability).sum()
        gradient, = torch.autograd.grad(loss * state["loss_gradient"].double()[0], logits)
        return dict(loss=loss.detach().reshape(1), tokens=None, probability=probability.detach(), gradient=gradient)
    # what an operator hands to the next one is rounded to its type there too
    half = lambda x: _nearest(x, 8, -126)
    values, scales = _stored_quantize(state["hidden"].double()[plan["route_token"].long()])
    inner = half(_exact_product(values, scales, *state["first"], plan["expert_offsets"]))
    values, scales = _stored_quantize(_exact_gate(inner))
    rows = half(_exact_product(values, scales, *state["second"], plan["expert_offsets"]))
    return _exact_combine(rows, plan, case["tokens"], state["hidden"])
