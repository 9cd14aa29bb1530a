"""Workloads of the operators around the fused MoE layer: the residual addition with RMS norm in front of it (e4m3 output
for the layer, or differentiable), tokens sorted by expert and back with their gradient, and the weights of the selected
experts with their gradient.

With ``own`` false a pass is computed in elementary torch operations in 32 bits, rounded once at the end; with ``own`` true by
the framework's operators.  Plain values of a case:

  op       "norm_fp8"    residual addition, RMS norm, e4m3 rows and one scale per token per 128 columns
           "norm_train"  residual addition, RMS norm, and its backward pass
           "tokens"      sort by expert, gather, combine with weights; `train` adds both backward passes
           "weights"     weights of the selected experts, and their backward pass
  tokens   batch size, `width` columns of a row, `dtype` of the rows
  stream   type of the residual stream ("" = there is none yet: the first norm of a model)
  normed   the normalised rows are wanted in `dtype` too (what the router reads)
  experts  local experts, `offset` = global id of the first; every token selects 8 of 256
  align    rows of an expert's segment are padded to a multiple of this
  room     capacity in rows of the sorted batch, as a multiple of what a uniform router would need (0 = room for any routing)
  skew     a few hot experts take most of the tokens
  padded   trailing tokens of the batch that select no expert
"""
import math

import torch

own = False

HIDDEN = 7168
INTER = 2048
EXPERTS = 256
GROUPS = 8
TOP_GROUPS = 4
TOP_K = 8
QBLOCK = 128
EPS = 1e-6
SCALE = 2.5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "": 0}


def _norm(name, op, tokens, dtype="bf16", stream="bf16", width=HIDDEN, normed=False):
    return {"name": name, "op": op, "tokens": tokens, "width": width, "dtype": dtype, "stream": stream, "normed": normed}


def _tokens(name, tokens, experts, train, dtype="bf16", width=HIDDEN, offset=0, align=1, room=0.0, skew=False, padded=0):
    return {"name": name, "op": "tokens", "tokens": tokens, "experts": experts, "train": train, "dtype": dtype,
            "width": width, "offset": offset, "align": align, "room": room, "skew": skew, "padded": padded}


def listed():
    return [
        # one sequence being decoded: launches and latency
        _norm("norm_fp8_1", "norm_fp8", 1, normed=True),
        # a decode batch at the first layer: nothing to add yet
        _norm("norm_fp8_80_first", "norm_fp8", 80, stream="", normed=True),
        # a long prefill: bound by the bytes of the residual stream
        _norm("norm_fp8_16384", "norm_fp8", 16384),
        # a short ragged training batch whose residual stream is kept in float32
        _norm("norm_train_333_f32", "norm_train", 333, stream="f32"),
        # a training batch
        _norm("norm_train_8192", "norm_train", 8192),
        # serving: a handful of sequences on one shard's experts
        _tokens("tokens_serve_7", 7, 32, False),
        # serving: a prompt on a shard with hot experts, segments padded for 128-row tiles, capacity for twice the mean load
        _tokens("tokens_serve_1500_shard", 1500, 64, False, offset=64, align=128, room=2.0, skew=True),
        # training in float32 on narrow rows, every expert local, a batch whose tail is padding
        _tokens("tokens_train_1001_f32", 1001, EXPERTS, True, dtype="f32", width=INTER, padded=37),
        # training: every expert local
        _tokens("tokens_train_8192", 8192, EXPERTS, True),
        # the router of a small training batch
        {"name": "weights_64", "op": "weights", "tokens": 64, "padded": 0},
        # the router of a large one
        {"name": "weights_16384", "op": "weights", "tokens": 16384, "padded": 100},
    ]


def draw(rng):
    """A case of the same ranges: one token to long batches (log-uniform), widths of 512 to 8192 columns, each type, a shard of
    8 .. 256 experts anywhere in the model, padded segments and capacities."""
    op = rng.choice(["norm_fp8", "norm_train", "tokens", "tokens", "weights"])
    if op == "weights":
        tokens = int(round(2.0 ** rng.uniform(0.0, 14.0)))
        return {"op": op, "tokens": tokens, "padded": rng.choice([0, tokens // 7])}
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    width = rng.choice([HIDDEN, HIDDEN, QBLOCK * int(round(2.0 ** rng.uniform(2.0, 6.0)))])
    if op != "tokens":
        tokens = int(round(2.0 ** rng.uniform(0.0, 14.0 if op == "norm_fp8" else 13.0)))
        stream = rng.choice([dtype, "f32", ""])
        return {"op": op, "tokens": tokens, "width": width, "dtype": dtype, "stream": stream, "normed": rng.random() < 0.5}
    tokens = int(round(2.0 ** rng.uniform(0.0, 11.0 if dtype == "f32" else 12.0)))
    experts = rng.choice([8, 32, 64, 256])
    room = 0.0 if experts == EXPERTS else rng.choice([0.0, 1.25, 2.0])
    return {"op": op, "tokens": tokens, "experts": experts, "train": rng.random() < 0.6, "dtype": dtype, "width": width,
            "offset": rng.randint(0, EXPERTS - experts), "align": rng.choice([1, 16, 128]), "room": room,
            "skew": rng.random() < 0.5, "padded": rng.choice([0, 0, tokens // 5])}


def _select(tokens, skew, padded, gen):
    """Router logits and the ids of the eight experts of every token, group-limited as the layer selects them; -1 for the
    padding of a batch."""
    logits = torch.randn((tokens, EXPERTS), generator=gen, device=gen.device)
    if skew:
        logits = logits + 1.5 * torch.randn(EXPERTS, generator=gen, device=gen.device)
    score = torch.sigmoid(logits)
    by_group = score.view(-1, GROUPS, EXPERTS // GROUPS)
    keep = by_group.topk(2, dim=2).values.sum(dim=2).topk(TOP_GROUPS, dim=1).indices
    mask = torch.zeros(by_group.shape[:2], device=gen.device).scatter_(1, keep, 1.0)
    masked = torch.where(mask.unsqueeze(2) > 0, by_group, -1.0).view(-1, EXPERTS)
    idx = masked.topk(TOP_K, dim=1).indices.to(torch.int32)
    idx[tokens - padded:] = -1
    return logits, idx


def _capacity(case):
    """Rows of the sorted batch: what any routing fits into, or `room` times the mean load, a multiple of `align`."""
    pairs, align = case["tokens"] * TOP_K, case["align"]
    if case["room"] > 0:
        return max(1, math.ceil(case["room"] * pairs * case["experts"] / EXPERTS / align)) * align
    return pairs if align == 1 else (pairs // align + min(case["experts"], pairs)) * align


def prepare(case, seed):
    """Activations N(0, 1) with a few large channels, norm weights around 1, gradients N(0, 1).  What a training step
    differentiates requires a gradient."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens, op = case["tokens"], case["op"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if op == "weights":
        logits, idx = _select(tokens, False, case["padded"], gen)
        return {"op": op, "logits": logits.requires_grad_(), "idx": idx, "grad": normal(tokens, TOP_K)}
    dtype, width = DTYPES[case["dtype"]], case["width"]
    if op == "tokens":
        logits, idx = _select(tokens, case["skew"], case["padded"], gen)
        weights = torch.rand((tokens, TOP_K), generator=gen, device="cuda") * (SCALE / 4)
        rows = _capacity(case)
        state = {"op": op, "train": case["train"], "idx": idx, "experts": case["experts"], "offset": case["offset"],
                 "align": case["align"], "rows": rows, "weights": weights, "x": normal(tokens, width, dtype=dtype),
                 "h": normal(rows, width, dtype=dtype)}
        if case["train"]:
            for name in ("x", "h", "weights"):
                state[name].requires_grad_()
            state["grad_xs"] = normal(rows, width, dtype=dtype)
            state["grad_y"] = normal(tokens, width, dtype=dtype)
        return state
    channels = 1.0 + 9.0 * (torch.rand(width, generator=gen, device="cuda") < 0.01)
    state = {"op": op, "normed": case["normed"], "x": (normal(tokens, width) * channels).to(dtype), "residual": None,
             "weight": (1.0 + 0.1 * normal(width)).to(dtype)}
    if case["stream"]:
        state["residual"] = (3.0 * normal(tokens, width) * channels).to(DTYPES[case["stream"]])
    if op == "norm_train":
        state["grad_y"] = normal(tokens, width, dtype=dtype)
        if case["stream"]:
            state["grad_r"] = normal(tokens, width, dtype=DTYPES[case["stream"]])
        for name in ("x", "residual", "weight"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


def _plain_norm(state):
    """The residual stream after the addition (rounded to its type: that is what the next layer reads), in 32 bits again, the
    reciprocal root of its mean square, and the normalised rows."""
    x, residual, weight = state["x"], state["residual"], state["weight"]
    r = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    h = r.float()
    rstd = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
    return r, h, rstd, h * rstd * weight.float()


def _plain_norm_fp8(state):
    r, h, rstd, y = _plain_norm(state)
    blocks = y.view(y.shape[0], -1, QBLOCK)
    scale = (blocks.abs().amax(dim=2) * (1.0 / 448.0)).clamp_min(1e-12)
    q = (blocks * (1.0 / scale).unsqueeze(2)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view_as(y)
    out = {"q": q, "scale": scale.t().contiguous(), "stream": r}
    if state["normed"]:
        out["normed"] = y.to(state["x"].dtype)
    return out


def _plain_norm_train(state):
    x, residual, weight = state["x"], state["residual"], state["weight"]
    r, h, rstd, y = _plain_norm(state)
    out = {"y": y.to(x.dtype), "stream": r}
    grad_y = state["grad_y"].float()
    g = grad_y * weight.float()
    grad = rstd * (g - h * (rstd.square() * (g * h).mean(dim=1, keepdim=True)))
    if residual is not None:
        grad = grad + state["grad_r"].float()
        out["grad_residual"] = grad.to(residual.dtype)
    out["grad_x"] = grad.to(x.dtype)
    out["grad_weight"] = (grad_y * h * rstd).sum(dim=0).to(weight.dtype)
    return out


def _plain_sort(idx, experts, offset, align, rows):
    """Stable by expert in the order of the flat (token, k) list: pair (t, k) goes behind the earlier pairs of its expert."""
    flat = idx.flatten().long() - offset
    local = (flat >= 0) & (flat < experts)
    chosen = (flat.unsqueeze(1) == torch.arange(experts, device=flat.device)).to(torch.int32)
    counts = chosen.sum(dim=0)
    segments = (counts + align - 1) // align * align
    offsets = torch.cat([segments.new_zeros(1), segments.cumsum(dim=0)])
    key = flat.clamp(0, experts - 1)
    rank = chosen.cumsum(dim=0).gather(1, key.unsqueeze(1)).squeeze(1) - 1
    place = offsets[key] + rank
    kept = local & (place < rows)
    scatter_map = torch.where(kept, place, -1).to(torch.int32).view_as(idx)
    pairs = torch.full((rows + 1,), -1, dtype=torch.int32, device=flat.device)
    pairs[torch.where(kept, place, rows)] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    row_pairs = pairs[:rows].clone()
    return {"counts": counts.to(torch.int32), "offsets": offsets.clamp(max=rows).to(torch.int32), "row_pairs": row_pairs,
            "scatter_map": scatter_map}


def _plain_tokens(state):
    x, h, weights, idx = state["x"], state["h"], state["weights"], state["idx"]
    out = _plain_sort(idx, state["experts"], state["offset"], state["align"], state["rows"])
    used = (out["row_pairs"] >= 0).unsqueeze(1)
    pair = out["row_pairs"].clamp(min=0).long()
    token = pair // TOP_K
    row = out["scatter_map"].clamp(min=0).long()
    has = (out["scatter_map"] >= 0).unsqueeze(2)
    out["xs"] = torch.where(used, x[token], 0.0).to(x.dtype)
    rows_of = torch.where(has, h[row], 0.0).float()
    out["y"] = (rows_of * weights.unsqueeze(2)).sum(dim=1).to(h.dtype)
    if state["train"]:
        grad_y = state["grad_y"].float()
        out["grad_h"] = torch.where(used, weights.flatten()[pair].unsqueeze(1) * grad_y[token], 0.0).to(h.dtype)
        out["grad_weights"] = (rows_of * grad_y.unsqueeze(1)).sum(dim=2)
        out["grad_x"] = torch.where(has, state["grad_xs"][row], 0.0).float().sum(dim=1).to(x.dtype)
    return out


def _plain_weights(state):
    logits, idx, grad = state["logits"], state["idx"], state["grad"]
    has = (idx >= 0).float()
    key = idx.clamp(min=0).long()
    chosen = logits.gather(1, key)
    s = torch.sigmoid(chosen) * has
    total = s.sum(dim=1, keepdim=True) + 1e-20
    weights = s / total * SCALE
    inner = SCALE / total * (grad - (grad * s).sum(dim=1, keepdim=True) / total)
    grad_logits = torch.zeros_like(logits).scatter_add_(1, key, inner * s * torch.sigmoid(-chosen))
    return {"weights": weights, "grad_logits": grad_logits}


def _own_norm_fp8(state):
    from fused_moe_b200 import norm
    got = norm.add_rms_norm_quantize(state["x"], state["residual"], state["weight"], EPS, with_normed=state["normed"])
    return dict(zip(("q", "scale", "stream", "normed"), got))


def _own_norm_train(state):
    from fused_moe_b200 import norm
    x, residual, weight = state["x"], state["residual"], state["weight"]
    y, r = norm.add_rms_norm(x, residual, weight, EPS)
    if residual is None:
        grad_x, grad_weight = torch.autograd.grad(y, (x, weight), state["grad_y"])
        return {"y": y, "stream": x, "grad_x": grad_x, "grad_weight": grad_weight}
    grads = torch.autograd.grad((y, r), (x, residual, weight), (state["grad_y"], state["grad_r"]))
    return {"y": y, "stream": r, "grad_x": grads[0], "grad_residual": grads[1], "grad_weight": grads[2]}


def _own_tokens(state):
    from fused_moe_b200 import tokens
    x, h, weights = state["x"], state["h"], state["weights"]
    plan = tokens.sort_tokens(state["idx"], state["experts"], state["offset"], align=state["align"], rows=state["rows"])
    xs = tokens.gather_tokens(x, plan)
    y = tokens.combine_tokens(h, weights, plan)
    out = {"counts": plan.counts, "offsets": plan.offsets, "row_pairs": plan.row_pairs, "scatter_map": plan.scatter_map,
           "xs": xs, "y": y}
    if state["train"]:
        grads = torch.autograd.grad((xs, y), (x, h, weights), (state["grad_xs"], state["grad_y"]))
        out["grad_x"], out["grad_h"], out["grad_weights"] = grads
    return out


def _own_weights(state):
    from fused_moe_b200 import tokens
    weights = tokens.route_weights(state["logits"], state["idx"], SCALE)
    return {"weights": weights, "grad_logits": torch.autograd.grad(weights, state["logits"], state["grad"])[0]}


def run(state):
    op = state["op"]
    if own:
        return {"norm_fp8": _own_norm_fp8, "norm_train": _own_norm_train, "tokens": _own_tokens,
                "weights": _own_weights}[op](state)
    with torch.no_grad():
        return {"norm_fp8": _plain_norm_fp8, "norm_train": _plain_norm_train, "tokens": _plain_tokens,
                "weights": _plain_weights}[op](state)


def _exact_norm(case, state):
    x, residual, weight = (v if v is None else v.detach() for v in (state["x"], state["residual"], state["weight"]))
    x64, w64 = x.double(), weight.double()
    stream = x64 if residual is None else x64 + residual.double()
    r = stream.to(x.dtype if residual is None else residual.dtype).double()
    root = torch.sqrt((r * r).sum(dim=1) / r.shape[1] + EPS)
    unit = r / root[:, None]
    y = unit * w64
    if case["op"] == "norm_fp8":
        largest = y.abs().view(y.shape[0], y.shape[1] // QBLOCK, QBLOCK).max(dim=2).values
        scale = torch.maximum(largest / 448.0, torch.full_like(largest, 1e-12))
        out = {"q": y / scale.repeat_interleave(QBLOCK, dim=1), "scale": scale.T.contiguous(), "stream": stream}
        if case["normed"]:
            out["normed"] = y
        return out
    grad_y = state["grad_y"].double()
    up = grad_y * w64
    grad = (up - unit * torch.einsum("th,th->t", up, unit)[:, None] / r.shape[1]) / root[:, None]
    out = {"y": y, "stream": stream, "grad_weight": torch.einsum("th,th->h", grad_y, unit)}
    if residual is not None:
        grad = grad + state["grad_r"].double()
        out["grad_residual"] = grad
    out["grad_x"] = grad
    return out


def _exact_tokens(case, state):
    x, h, weights = (state[n].detach().double() for n in ("x", "h", "weights"))
    idx, experts, rows, align = state["idx"], state["experts"], state["rows"], state["align"]
    expert = idx.flatten().long() - state["offset"]
    expert = torch.where((expert < 0) | (expert >= experts), experts, expert)
    order = torch.sort(expert, stable=True).indices
    counts = torch.bincount(expert, minlength=experts + 1)[:experts]
    starts, at = [0], 0
    for c in counts.tolist():
        at += -(-c // align) * align
        starts.append(at)
    row_pairs = torch.full((rows,), -1, dtype=torch.int64, device=x.device)
    done = 0
    for e, c in enumerate(counts.tolist()):
        n = max(0, min(c, rows - starts[e]))
        row_pairs[starts[e]:starts[e] + n] = order[done:done + n]
        done += c
    row = (row_pairs >= 0).nonzero().squeeze(1)
    pair = row_pairs[row]
    token, w = pair // TOP_K, weights.flatten()[pair]
    scatter_map = torch.full((idx.numel(),), -1, dtype=torch.int64, device=x.device)
    scatter_map[pair] = row
    xs, y = torch.zeros_like(h), torch.zeros_like(x)
    xs[row] = x[token]
    y.index_add_(0, token, h[row] * w[:, None])
    out = {"counts": counts, "offsets": torch.tensor([min(s, rows) for s in starts], device=x.device),
           "row_pairs": row_pairs, "scatter_map": scatter_map.view(idx.shape), "xs": xs, "y": y}
    if case["train"]:
        grad_y = state["grad_y"].double()[token]
        out["grad_h"], out["grad_x"] = torch.zeros_like(h), torch.zeros_like(x)
        out["grad_h"][row] = grad_y * w[:, None]
        out["grad_weights"] = torch.zeros(idx.numel(), dtype=torch.float64, device=x.device)
        out["grad_weights"][pair] = (grad_y * h[row]).sum(dim=1)
        out["grad_weights"] = out["grad_weights"].view(idx.shape)
        out["grad_x"].index_add_(0, token, state["grad_xs"].double()[row])
    return out


def _exact_weights(state):
    logits, idx, grad = state["logits"].detach().double(), state["idx"].long(), state["grad"].double()
    mask = torch.zeros_like(logits)
    token = torch.arange(idx.shape[0], device=idx.device)[:, None].expand_as(idx)
    real = idx >= 0
    mask[token[real], idx[real]] = 1.0
    up = torch.zeros_like(logits)
    up[token[real], idx[real]] = grad[real]
    s = mask / (1.0 + torch.exp(-logits))
    total = s.sum(dim=1, keepdim=True) + 1e-20
    share = s / total
    grad_logits = SCALE * share * (1.0 - s) * mask * (up - (up * share).sum(dim=1, keepdim=True))
    weights = torch.zeros_like(grad)
    weights[real] = SCALE * share[token[real], idx[real]]
    return {"weights": weights, "grad_logits": grad_logits}


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "weights":
        return _exact_weights(state)
    return _exact_tokens(case, state) if case["op"] == "tokens" else _exact_norm(case, state)


def work(case):
    """Every input read once and every output written once.  A shard reads the rows of the tokens that it has a pair of, and
    the rows of its segments; the rows behind them are written as zeros."""
    tokens, op = case["tokens"], case["op"]
    if op == "weights":
        sectors = (tokens - case["padded"]) * TOP_K * 4
        return {"bytes": sectors + tokens * (TOP_K * 12 + EXPERTS * 4), "flops": tokens * TOP_K * 20}
    width, size = case["width"], SIZE[case["dtype"]]
    if op != "tokens":
        stream = SIZE[case["stream"]]
        per = size + 2 * stream                              # x, the residual stream in and out
        if op == "norm_fp8":
            per += 1 + 4 / QBLOCK + (size if case["normed"] else 0)
        else:
            per += 3 * size + 2 * stream - (size if stream == size else 0)   # y, its gradient, dx; the stream's gradients
        return {"bytes": tokens * width * per, "flops": tokens * width * (10 if op == "norm_fp8" else 20)}
    _, idx = _select(tokens, case["skew"], case["padded"], torch.Generator().manual_seed(7))
    local = (idx >= case["offset"]) & (idx < case["offset"] + case["experts"])
    rows = _capacity(case)
    pairs, active = min(rows, int(local.sum())), int(local.any(dim=1).sum())
    moved = active + rows + pairs + tokens                   # x in, xs out, h in, y out
    if case["train"]:
        moved += active + rows + pairs + tokens              # grad_y in, grad_h out, grad_xs in, grad_x out
    plan = 4 * (tokens * TOP_K * 3 + rows + 2 * case["experts"])
    return {"bytes": moved * width * size + plan, "flops": (4 if not case["train"] else 10) * pairs * width}
