"""GPU: tokens sorted by expert and back with their gradients, and the weights of the selected experts with theirs, against plain
implementations (whole numbers and copies exactly, sums in 64 bits).

Tolerances.  u(t) is half a step of type t.  A combined row is a float32 chain of at most eight multiply-adds: 8 * 2^-24 of the sum
of the terms' magnitudes, and u(t) of the result.  A weight's gradient is a dot product over n columns that at least 32 threads
share: a chain of n / 32 + 8 terms, then 5 + 8 levels."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS24 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def tok():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from fused_moe_b200 import tokens as module
    return module


def assert_within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(err / tol)[bad].max().item():.3f} x"


def poison(rows, n, dtype):
    torch.full((rows, n), float("nan"), device="cuda", dtype=F32).to(dtype)


def select(T, K=8, seed=0, kind="uniform", E=256):
    """Expert ids [T, K]: uniform (distinct per token), hot (a few experts take most), repeats (an expert twice), padded (trailing
    -1), one (all tokens one set), none."""
    rng = np.random.default_rng(seed * 7919 + T * 31 + K)
    ids = np.argsort(rng.random((T, E)), axis=1)[:, :K].astype(np.int32) if T * E < 1 << 23 else \
        (rng.integers(0, E, (T, 1)) + np.arange(K) * 31).astype(np.int32) % E
    if kind == "hot":
        hot = rng.random(T) < 0.7
        ids[hot] = np.arange(K, dtype=np.int32) + 64
    elif kind == "repeats":
        ids = rng.integers(60, 70, (T, K)).astype(np.int32)
    elif kind == "padded":
        ids[T - T // 3:] = -1
        ids[::5, K // 2] = -1
    elif kind == "wild":      # ids that are none: far outside, and the extremes of the type
        ids[::2, 0] = 2 ** 31 - 1
        ids[1::2, 0] = -2 ** 31
        ids[::3, -1] = 256
    elif kind == "one":
        ids[:] = np.arange(K, dtype=np.int32) * 31 % E
    elif kind == "none":
        ids[:] = -1
    return torch.from_numpy(ids).cuda()


def plain_sort(idx, E, offset, align, rows):
    """numpy, stable by expert."""
    ids = idx.cpu().numpy().astype(np.int64)
    flat = ids.reshape(-1) - offset
    flat = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(flat, kind="stable")
    counts = np.bincount(flat, minlength=E + 1)[:E]
    starts = np.concatenate([[0], np.cumsum(-(-counts // align) * align)])
    row_pairs = np.full(rows, -1, np.int64)
    scatter = np.full(flat.shape, -1, np.int64)
    at = 0
    for e in range(E):
        for j, p in enumerate(order[at:at + counts[e]]):
            r = starts[e] + j
            if r < rows:
                row_pairs[r], scatter[p] = p, r
        at += counts[e]
    as_gpu = lambda a: torch.from_numpy(a.astype(np.int32)).cuda()  # noqa: E731
    return as_gpu(counts), as_gpu(np.minimum(starts, rows)), as_gpu(row_pairs), as_gpu(scatter.reshape(ids.shape))


def assert_sorted(plan, want):
    for name, w in zip(("counts", "offsets", "row_pairs", "scatter_map"), want):
        got = getattr(plan, name)
        assert got.dtype is torch.int32 and torch.equal(got, w), name


SORTS = [(1, 8, 256, 0, 1, "uniform"), (1, 1, 1, 255, 1, "none"), (2, 3, 32, 64, 16, "uniform"), (7, 8, 32, 64, 128, "hot"),
         (31, 5, 8, 60, 4, "repeats"), (127, 8, 256, 0, 1, "padded"), (128, 8, 256, 0, 128, "uniform"), (129, 8, 64, 64, 128, "hot"),
         (333, 8, 256, 0, 7, "wild"), (640, 8, 16, 62, 1, "repeats"), (1000, 2, 256, 0, 1, "one"), (1500, 8, 64, 64, 128, "hot"),
         (2050, 8, 256, 0, 1, "uniform"), (4096, 8, 32, 96, 1, "none"), (9001, 7, 256, 0, 16, "padded"),
         (40000, 8, 256, 0, 128, "hot")]


@pytest.mark.parametrize("T, K, E, offset, align, kind", SORTS)
def test_sort(tok, T, K, E, offset, align, kind):
    idx = select(T, K, 1, kind)
    plan = tok.sort_tokens(idx, E, offset, align=align)
    assert plan.rows % align == 0
    assert_sorted(plan, plain_sort(idx, E, offset, align, plan.rows))
    total = int(plan.offsets[-1])
    for rows in {0, 1, max(0, total - 1), total, total // 2 + 1, total + 77}:   # capacities that do not suffice, and more than enough
        assert_sorted(tok.sort_tokens(idx, E, offset, align=align, rows=rows), plain_sort(idx, E, offset, align, rows))


def test_sort_of_many_pairs(tok):
    """More than 256 rounds of 1024 pairs: a CTA ranks several rounds one after the other."""
    idx = select(70001, 8, 2, "hot")
    idx[::3] = select(70001, 8, 3, "uniform")[::3]
    plan = tok.sort_tokens(idx, 256, align=16)
    assert_sorted(plan, plain_sort(idx, 256, 0, 16, plan.rows))


def test_sort_matches_the_layers_sort(tok):
    """Padded to 128 rows, the counts, segments and rows are those of the layer's own sort."""
    from fused_moe_b200 import kernel as K, synth
    T, E, offset = 300, 32, 64
    inp = synth.make_inputs(T, E, seed=4, local_expert_offset=offset, skew=True, device="cuda", only_experts=[])
    idx, w = K.route(inp["routing_logits"], inp["routing_bias"], 2.5)
    K.kernel_from_topk(idx, w, *[inp[k] for k in ("hidden_states", "hidden_states_scale", "gemm1_weights",
                                                  "gemm1_weights_scale", "gemm2_weights", "gemm2_weights_scale")], offset)
    ws = K.last_workspace()
    plan = tok.sort_tokens(idx, E, offset, align=128)
    assert torch.equal(plan.counts, ws.view("counts", torch.int32, (E,)))
    assert torch.equal(plan.offsets, ws.view("block_offsets", torch.int32, (E + 1,)) * 128)
    assert torch.equal(plan.scatter_map, ws.view("scatter_map", torch.int32, (T, 8)))


def test_strided_ids(tok):
    wide = torch.cat([select(50, 8, 5), select(50, 8, 6)], dim=1)
    assert_sorted(tok.sort_tokens(wide[:, 3:11], 256), plain_sort(wide[:, 3:11], 256, 0, 1, 400))
    assert_sorted(tok.sort_tokens(wide.t().contiguous().t()[:, :8], 256), plain_sort(wide[:, :8], 256, 0, 1, 400))


BATCHES = [(1, 8, 256, 0, 1, "uniform", 7168), (1, 8, 32, 64, 128, "none", 8), (3, 2, 32, 64, 16, "repeats", 256),
           (7, 8, 32, 64, 1, "hot", 7168), (33, 8, 256, 0, 128, "uniform", 2048), (80, 8, 64, 64, 1, "padded", 2056),
           (257, 8, 256, 0, 1, "padded", 7168), (500, 5, 8, 62, 128, "repeats", 520), (1001, 8, 256, 0, 16, "uniform", 136),
           (1300, 8, 64, 64, 1, "hot", 4096)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("T, K, E, offset, align, kind, n", BATCHES)
def test_gather_and_combine_with_gradients(tok, T, K, E, offset, align, kind, n, dtype):
    idx = select(T, K, 7, kind)
    g = torch.Generator(device="cuda").manual_seed(T + n)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    for rows in (None, max(1, T * K * E // 600)):
        plan = tok.sort_tokens(idx, E, offset, align=align, rows=rows)
        R, has = plan.rows, (plan.scatter_map >= 0)
        used = plan.row_pairs >= 0
        token = (plan.row_pairs.clamp(min=0) // K).long()
        row = plan.scatter_map.clamp(min=0).long()
        x, h, w = rnd(T, n).to(dtype), rnd(R, n).to(dtype), rnd(T, K)
        h[~used] = float("nan")   # rows without a pair are not read
        gxs, gy = rnd(R, n).to(dtype), rnd(T, n).to(dtype)
        gxs[~used] = float("nan")
        for t in (x, h, w):
            t.requires_grad_()
        poison(R, n, dtype)
        xs = tok.gather_tokens(x, plan)
        assert torch.equal(xs, torch.where(used[:, None], x.detach()[token], 0.0))
        poison(T, n, dtype)
        y = tok.combine_tokens(h, w, plan)
        h64 = torch.where(has[:, :, None], h.detach()[row], 0.0).double() if R else torch.zeros((T, K, n), device="cuda").double()
        want = (h64 * w.detach().double()[:, :, None]).sum(dim=1)
        size = (h64 * w.detach().double()[:, :, None]).abs().sum(dim=1)
        assert_within(y, want, u(dtype) * want.abs() + 8 * EPS24 * size + tiny(dtype), "combined")
        poison(T, n, dtype), poison(R, n, dtype), poison(T, K, F32)
        gx, gh, gw = torch.autograd.grad((xs, y), (x, h, w), (gxs, gy))
        gxs64 = torch.where(has[:, :, None], gxs[row], 0.0).double()
        assert_within(gx, gxs64.sum(dim=1), u(dtype) * gxs64.sum(dim=1).abs() + 8 * EPS24 * gxs64.abs().sum(dim=1) + tiny(dtype),
                      "grad of x")
        flat_w = w.detach().flatten()[plan.row_pairs.clamp(min=0).long()].double()
        gh64 = torch.where(used[:, None], flat_w[:, None] * gy.double()[token], 0.0)
        assert_within(gh, gh64, (u(dtype) + 2 * EPS24) * gh64.abs() + tiny(dtype), "grad of rows")
        dots = h64 * gy.double()[:, None]
        assert_within(gw, dots.sum(dim=2), (n / 32 + 21) * EPS24 * dots.abs().sum(dim=2), "grad of weights")
        assert gw[~has].eq(0).all() and gh[~used].eq(0).all()
        # the explicit forms: the same bits
        with torch.no_grad():
            assert torch.equal(tok.gather_tokens(x, plan), xs) and torch.equal(tok.combine_tokens(h, w, plan), y)
        assert torch.equal(tok.gather_tokens_backward(gxs, plan), gx)
        a, b = tok.combine_tokens_backward(gy, h, w, plan)
        assert torch.equal(a, gh) and torch.equal(b, gw)


def test_gradients_against_differences(tok):
    """Both operators are linear in each argument: a central difference of the 64-bit function is its derivative."""
    idx = select(40, 8, 8, "repeats")
    plan = tok.sort_tokens(idx, 8, 61, align=4)
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
    n, R = 64, plan.rows
    x, h, w, gxs, gy = rnd(40, n), rnd(R, n), rnd(40, 8), rnd(R, n), rnd(40, n)
    used, has = (plan.row_pairs >= 0)[:, None], (plan.scatter_map >= 0)[:, :, None]

    def f(x, h, w):
        xs = torch.where(used, x[(plan.row_pairs.clamp(min=0) // 8).long()], 0.0)
        y = (torch.where(has, h[plan.scatter_map.clamp(min=0).long()], 0.0) * w[:, :, None]).sum(dim=1)
        return (xs * gxs).sum() + (y * gy).sum()

    f32 = [t.float() for t in (x, h, w, gxs, gy)]
    x, h, w, gxs, gy = (t.double() for t in f32)
    got = [tok.gather_tokens_backward(f32[3], plan), *tok.combine_tokens_backward(f32[4], f32[1], f32[2], plan)]
    for i, grad in enumerate(got):
        d = rnd(*(x, h, w)[i].shape)
        step = lambda s: [a + s * d if j == i else a for j, a in enumerate((x, h, w))]  # noqa: E731
        diff = (f(*step(0.5)) - f(*step(-0.5)))
        size = (d.abs() * (1 + grad.double().abs())).sum()
        # float32 gradients: at most 8 terms of size ~1, or 64 / 32 + 21 in the dot product
        assert abs((grad.double() * d).sum() - diff) <= 40 * EPS24 * size * 8


def test_what_lies_in_masked_places_is_not_used(tok):
    """NaN and infinities in the weights and gradients of pairs without a row, in rows without a pair and in the logits of experts
    that no pair names leave no trace."""
    T, n = 50, 136
    idx = select(T, 8, 17, "padded")
    g = torch.Generator(device="cuda").manual_seed(21)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    plan = tok.sort_tokens(idx, 128, 64, align=16, rows=100)
    has, used = plan.scatter_map >= 0, plan.row_pairs >= 0
    assert not has.all() and not used.all() and has.any()
    x, h, w, gy, gxs = rnd(T, n), rnd(100, n), rnd(T, 8), rnd(T, n), rnd(100, n)
    idle = ~has.any(dim=1)   # tokens without any row
    assert idle.any()

    def results(x, h, w, gy, gxs):
        return (tok.gather_tokens(x, plan), tok.combine_tokens(h, w, plan), tok.gather_tokens_backward(gxs, plan),
                *tok.combine_tokens_backward(gy, h, w, plan))

    want = results(x, h, w, gy, gxs)
    for bad in (float("nan"), float("inf"), -3.4e38):
        x2, h2, w2, gy2, gxs2 = (t.clone() for t in (x, h, w, gy, gxs))
        x2[idle], gy2[idle], h2[~used], gxs2[~used], w2[~has] = bad, bad, bad, bad, bad
        assert all(torch.equal(a, b) for a, b in zip(results(x2, h2, w2, gy2, gxs2), want))
    logits, gw = rnd(T, 256), rnd(T, 8)
    want = tok.route_weights(logits, idx, 2.5), tok.route_weights_backward(logits, idx, gw, 2.5)
    named = torch.zeros((T, 257), dtype=torch.bool, device="cuda").scatter_(1, torch.where(idx >= 0, idx, 256).long(), True)
    for bad in (float("nan"), float("inf"), -3.4e38):
        l2, gw2 = torch.where(named[:, :256], logits, bad), torch.where(idx >= 0, gw, bad)
        assert torch.equal(tok.route_weights(l2, idx, 2.5), want[0])
        assert torch.equal(tok.route_weights_backward(l2, idx, gw2, 2.5), want[1])


def test_partial_gradients(tok):
    idx = select(20, 8, 9)
    plan = tok.sort_tokens(idx, 256)
    h, w, gy = torch.randn(160, 64, device="cuda"), torch.randn(20, 8, device="cuda"), torch.randn(20, 64, device="cuda")
    want = tok.combine_tokens_backward(gy, h, w, plan)
    for i in range(2):
        args = [h.clone(), w.clone()]
        args[i].requires_grad_()
        got = torch.autograd.grad(tok.combine_tokens(*args, plan), args[i], gy)[0]
        assert torch.equal(got, want[i])
    leaf = h.clone().requires_grad_()
    one = torch.autograd.grad(tok.combine_tokens(leaf, w, plan).sum(), leaf)[0]   # a broadcast gradient
    assert torch.equal(one, tok.combine_tokens_backward(torch.ones_like(gy), h, w, plan)[0])


def test_second_derivatives_are_refused(tok):
    idx = select(6, 8, 15)
    plan = tok.sort_tokens(idx, 256)
    x, h, w, logits = (torch.randn(s, device="cuda").requires_grad_() for s in ((6, 64), (48, 64), (6, 8), (6, 256)))
    for out, leaves in ((tok.gather_tokens(x, plan), (x,)), (tok.combine_tokens(h, w, plan), (h, w)),
                        (tok.route_weights(logits, idx, 2.5), (logits,))):
        grads = torch.autograd.grad(out.square().sum(), leaves, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            sum((g.sum() + leaf.square().sum()) for g, leaf in zip(grads, leaves)).backward()


def test_strided_and_unaligned_rows(tok):
    idx = select(30, 8, 10, "padded")
    plan = tok.sort_tokens(idx, 256, align=16)
    wide = torch.randn(plan.rows, 1000, device="cuda").bfloat16()
    w = torch.randn(30, 16, device="cuda")[:, ::2]
    for cut in (lambda t: t[:, 8:264], lambda t: t[:, 3:259], lambda t: t[:, ::2][:, :256], lambda t: t[:1].expand(t.shape)[:, :256]):
        x, h = cut(wide[:30]), cut(wide)
        assert torch.equal(tok.gather_tokens(x, plan), tok.gather_tokens(x.contiguous().clone(), plan))
        assert torch.equal(tok.combine_tokens(h, w, plan), tok.combine_tokens(h.contiguous().clone(), w.contiguous(), plan))
        for a, b in zip(tok.combine_tokens_backward(x, h, w, plan),
                        tok.combine_tokens_backward(x.contiguous().clone(), h.contiguous().clone(), w.contiguous(), plan)):
            assert torch.equal(a, b)


def test_rows_of_another_batch_do_no_harm(tok):
    """A map whose entries lie outside the buffers: such a pair counts as one without a row."""
    plan = tok.sort_tokens(select(10, 8, 11), 256)
    bad = plan.scatter_map.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = 80, -7, 2 ** 31 - 1
    x, w = torch.randn(10, 64, device="cuda"), torch.randn(10, 8, device="cuda")
    h = torch.randn(80, 64, device="cuda")
    keep = (bad >= 0) & (bad < 80)
    got = tok.combine_tokens(h, w, plan._replace(scatter_map=bad))
    want = (torch.where(keep[:, :, None], h[torch.where(keep, bad, 0).long()], 0.0).double() * w.double()[:, :, None])
    assert_within(got, want.sum(dim=1), 9 * EPS24 * want.abs().sum(dim=1), "combined")
    assert tok.gather_tokens(x, plan._replace(scatter_map=bad)).shape == (80, 64)
    assert tok.combine_tokens_backward(x, h, w, plan._replace(scatter_map=bad))[1][~keep].eq(0).all()
    torch.cuda.synchronize()


def test_offsets_past_32_bits(tok):
    """More than 2^31 elements and 2^32 bytes of sorted rows."""
    T, n = 40_100, 7168
    idx = select(T, 8, 16)
    plan = tok.sort_tokens(idx, 256)
    assert plan.rows * n > 2 ** 31
    torch.manual_seed(20)
    x = torch.randn(T, n, device="cuda", dtype=BF16)
    xs = tok.gather_tokens(x, plan)
    pick = torch.tensor([0, 1, plan.rows // 2, plan.rows - 2, plan.rows - 1], device="cuda")
    assert torch.equal(xs[pick], x[(plan.row_pairs[pick] // 8).long()])
    w = torch.rand(T, 8, device="cuda")
    y = tok.combine_tokens(xs, w, plan)
    some = torch.tensor([0, 7, T // 2, T - 1], device="cuda")
    want = x[some].double() * w[some].double().sum(dim=1, keepdim=True)
    assert_within(y[some], want, (u(BF16) + 8 * EPS24) * want.abs() + 8 * EPS24 * want.abs(), "combined")
    gh, gw = tok.combine_tokens_backward(x, xs, w, plan)
    pair = plan.row_pairs[pick].long()
    want = w.flatten()[pair].double()[:, None] * x[pair // 8].double()
    assert_within(gh[pick], want, (u(BF16) + 2 * EPS24) * want.abs() + tiny(BF16), "grad of rows")
    dots = x[some].double().square().sum(dim=1, keepdim=True).expand(-1, 8)
    assert_within(gw[some], dots, (n / 32 + 21) * EPS24 * dots, "grad of weights")


def test_empty_batches(tok):
    idx = torch.empty((0, 8), dtype=torch.int32, device="cuda")
    plan = tok.sort_tokens(idx, 32, 64, align=128)
    assert plan.rows == 0 and plan.counts.eq(0).all() and plan.offsets.eq(0).all()
    x = torch.empty((0, 256), device="cuda", requires_grad=True)
    assert tok.gather_tokens(x, plan).shape == (0, 256)
    plan = tok.sort_tokens(idx, 32, 64, rows=20)   # rows without any token are zeros
    poison(20, 256, F32)
    xs = tok.gather_tokens(x, plan)
    assert xs.eq(0).all() and torch.autograd.grad(xs, x, torch.ones_like(xs))[0].shape == (0, 256)
    w = torch.empty((0, 8), device="cuda")
    h = torch.ones((20, 256), device="cuda")
    assert tok.combine_tokens(h, w, plan).shape == (0, 256)
    poison(20, 256, F32)
    gh, gw = tok.combine_tokens_backward(x.detach(), h, w, plan)
    assert gh.eq(0).all() and gw.shape == (0, 8)
    plan = tok.sort_tokens(select(4, 8, 12), 256, rows=0)   # no room at all
    y = tok.combine_tokens(torch.empty((0, 256), device="cuda"), torch.ones((4, 8), device="cuda"), plan)
    assert y.eq(0).all() and tok.gather_tokens(torch.ones((4, 256), device="cuda"), plan).shape == (0, 256)
    gh, gw = tok.combine_tokens_backward(torch.ones((4, 256), device="cuda"), torch.empty((0, 256), device="cuda"),
                                         torch.ones((4, 8), device="cuda"), plan)
    assert gh.shape == (0, 256) and gw.eq(0).all()
    assert tok.route_weights(torch.empty((0, 256), device="cuda"), idx, 2.5).shape == (0, 8)


# ---- weights of the selected experts -----------------------------------------------------------------------------------------
def weights64(logits, idx, scale):
    has = (idx >= 0) & (idx < 256)
    s = torch.sigmoid(logits.double()).gather(1, torch.where(has, idx, 0).long()) * has
    return s / (s.sum(dim=1, keepdim=True) + 1e-20) * scale


@pytest.mark.parametrize("T, scale", [(1, 2.5), (7, 1.0), (33, 2.5), (1000, 2.5)])
def test_route_weights_are_those_of_route(tok, T, scale):
    from fused_moe_b200 import kernel as K
    g = torch.Generator(device="cuda").manual_seed(T)
    logits = 3 * torch.randn(T, 256, generator=g, device="cuda")
    bias = (0.1 * torch.randn(256, generator=g, device="cuda")).bfloat16()
    idx, w = K.route(logits, bias, scale)
    assert torch.equal(tok.route_weights(logits, idx, scale), w)


@pytest.mark.parametrize("T, K, kind, spread", [(1, 8, "uniform", 1.0), (5, 3, "repeats", 4.0), (64, 8, "padded", 1.0),
                                                (333, 8, "wild", 8.0), (1001, 7, "repeats", 1.0), (2000, 1, "uniform", 2.0)])
def test_route_weights_and_gradient(tok, T, K, kind, spread):
    """The sigmoid's operations are within 4.2e-7 relative (polynomial 5e-9, Horner and argument reduction 3e-7, sum and division
    1.2e-7) for |x| < 87; weights take two of them and ten roundings: 2^-19.  The gradient's terms take four: 2^-18 of them."""
    idx = select(T, K, 13, kind)
    g = torch.Generator(device="cuda").manual_seed(T)
    logits = (spread * torch.randn(T, 256, generator=g, device="cuda")).requires_grad_()
    grad = torch.randn(T, K, generator=g, device="cuda")
    w = tok.route_weights(logits, idx, 2.5)
    want = weights64(logits.detach(), idx, 2.5)
    assert_within(w, want, 2.0 ** -19 * want, "weights")
    poison(T, 256, F32)
    got = torch.autograd.grad(w, logits, grad)[0]
    l64 = logits.detach().double()
    ref, size = logits_grad64(l64, idx, grad, 2.5)
    assert_within(got, ref, 2.0 ** -18 * size, "grad of logits")
    assert torch.equal(got, tok.route_weights_backward(logits.detach(), idx, grad, 2.5))
    # differences: the function is smooth, third derivatives of order 1; h = 1e-4 gives h^2 = 1e-8 of the terms
    d = torch.randn(l64.shape, dtype=torch.float64, device="cuda")
    f = lambda a: (weights64(a, idx, 2.5) * grad.double()).sum()  # noqa: E731
    diff = (f(l64 + 1e-4 * d) - f(l64 - 1e-4 * d)) / 2e-4
    assert abs((got.double() * d).sum() - diff) <= (size * d.abs()).sum() * 2.0 ** -18 + 1e-7 * size.sum() * 64


def logits_grad64(l64, idx, grad, scale):
    """The gradient by the formula, and the magnitudes of its terms.  1 - s is taken as sigmoid(-x): s * (1 - s), as torch's own
    gradient has it, loses what it is near x = 30 even in 64 bits."""
    has = (idx >= 0) & (idx < 256)
    key, grad = torch.where(has, idx, 0).long(), grad.double()
    s = torch.sigmoid(l64).gather(1, key) * has
    total = s.sum(dim=1, keepdim=True) + 1e-20
    front = scale * s * torch.sigmoid(-l64).gather(1, key) / total * has
    inner = front * (grad - (grad * s).sum(dim=1, keepdim=True) / total)
    terms = front * (grad.abs() + (grad.abs() * s).sum(dim=1, keepdim=True) / total)
    return tuple(torch.zeros_like(l64).scatter_add_(1, key, v) for v in (inner, terms))


def test_route_weights_at_the_extremes(tok):
    """Saturated logits: weights and gradients stay finite, and a gradient of 1 - s does not cancel."""
    logits = torch.zeros(4, 256, device="cuda")
    logits[0] = 30.0
    logits[1] = -80.0
    logits[2] = 1e4
    logits[3] = -1e4
    idx = select(4, 8, 14)
    w = tok.route_weights(logits, idx, 2.5)
    assert_within(w[:2], weights64(logits, idx, 2.5)[:2], 2.0 ** -19 * 2.5, "weights")
    assert w.isfinite().all()
    up = torch.arange(32.0, device="cuda").view(4, 8)
    grad = tok.route_weights_backward(logits, idx, up, 2.5)
    assert grad.isfinite().all()
    ref, size = logits_grad64(logits.double(), idx, up, 2.5)
    assert_within(grad[0], ref[0], 2.0 ** -18 * size[0], "grad at 30")
    logits[0, int(idx[0, 0])] = float("nan")   # a NaN stays in its token
    w2 = tok.route_weights(logits, idx, 2.5)
    assert w2[0].isnan().all() and torch.equal(w2[1:], w[1:])


# ---- streams, graphs, and all of it together -------------------------------------------------------------------------------
def _step(tok, logits, idx, x, h, w, gxs, gy):
    plan = tok.sort_tokens(idx, 256, align=16)
    weights = tok.route_weights(logits, idx, 2.5)
    xs, y = tok.gather_tokens(x, plan), tok.combine_tokens(h, weights, plan)
    gx = tok.gather_tokens_backward(gxs, plan)
    gh, gw = tok.combine_tokens_backward(gy, h, weights, plan)
    return [plan.counts, plan.offsets, plan.row_pairs, plan.scatter_map, weights, xs, y, gx, gh, gw,
            tok.route_weights_backward(logits, idx, gw, 2.5)]


def _values(T, seed, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R = (T * 8 // 16 + min(256, T * 8)) * 16
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return [rnd(T, 256), select(T, 8, seed), rnd(T, 512).to(dtype), rnd(R, 512).to(dtype), rnd(T, 8), rnd(R, 512).to(dtype),
            rnd(T, 512).to(dtype)]


def test_repeats_bit_for_bit_and_on_another_stream(tok):
    args = _values(777, 1)
    first = _step(tok, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _step(tok, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_two_graphs_replayed_at_once(tok):
    """Captured steps share no scratch: replayed on two streams, over and over and on new values, each gives what it gives alone."""
    sizes, graphs = (130, 2100), []
    for T in sizes:
        static = _values(T, 2)
        _step(tok, *static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(tok, *static)
        graphs.append((graph, static, out, torch.cuda.Stream()))
    for seed in (3, 4):
        want = []
        for T, (graph, static, out, _) in zip(sizes, graphs):
            for a, b in zip(static, _values(T, seed)):
                a.copy_(b)
            want.append(_step(tok, *static))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, _, _, stream in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, out, _), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_refuses_to_record_under_capture(tok):
    logits, idx, x, h, w, gxs, gy = _values(20, 5)
    plan = tok.sort_tokens(idx, 256, align=16)
    leaf, rows_leaf, logits_leaf = (t.clone().requires_grad_() for t in (x, h, logits))
    alive = tok.gather_tokens(leaf, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call, name in ((lambda: tok.gather_tokens(leaf, plan), "gather_tokens_backward"),
                           (lambda: tok.combine_tokens(rows_leaf, w, plan), "combine_tokens_backward"),
                           (lambda: tok.route_weights(logits_leaf, idx, 2.5), "route_weights_backward")):
            with pytest.raises(RuntimeError, match=name):
                call()
        with torch.no_grad():
            out = tok.gather_tokens(leaf, plan)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive)


def test_training_block(tok):
    """The run as it is used: norm -> router -> selected weights -> sort -> gather -> experts (torch products) -> combine, and
    back, in float32, against the same graph in 64 bits with torch's own gradients.

    Each product of length n = 256 is off by at most n * 2^-24 = 1.5e-5 of its absolute sum, which is about sqrt(n) = 16 times
    the result's norm: 2.4e-4.  The results pass through at most three products forward and three back: 1.5e-3 in the 2-norm."""
    from fused_moe_b200 import kernel as K, norm
    T, n, E, offset = 150, 256, 6, 96
    g = torch.Generator(device="cuda").manual_seed(6)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, res, w = rnd(T, n), rnd(T, n), 1 + 0.1 * rnd(n)
    gate = rnd(256, n) / 16
    gate[offset:offset + E] *= 3   # the local experts are chosen often
    experts = rnd(E, n, n) / 16
    bias = torch.zeros(256, dtype=BF16, device="cuda")
    gy, gr = rnd(T, n), rnd(T, n)

    def block(x, res, w, gate, experts, ours, idx=None):
        if ours:
            y, r = norm.add_rms_norm(x, res, w)
            logits = y @ gate.t()
            idx, _ = K.route(logits.detach(), bias, 2.5)
            weights = tok.route_weights(logits, idx, 2.5)
            plan = tok.sort_tokens(idx, E, offset, align=16)
            xs = tok.gather_tokens(y, plan)
            segment = torch.searchsorted(plan.offsets[1:].contiguous(), torch.arange(plan.rows, device="cuda", dtype=torch.int32),
                                         right=True).clamp(max=E - 1)
            parts = torch.stack([torch.tanh(xs @ experts[e]) for e in range(E)])
            return tok.combine_tokens(parts[segment, torch.arange(plan.rows, device="cuda")], weights, plan), r, idx
        r = x + res
        y = r / torch.sqrt(r.square().mean(dim=1, keepdim=True) + 1e-6) * w
        s = torch.sigmoid(y @ gate.t()).gather(1, idx.long())
        weights = s / (s.sum(dim=1, keepdim=True) + 1e-20) * 2.5
        out = torch.zeros_like(x)
        for e in range(E):
            share = (weights * (idx == offset + e)).sum(dim=1, keepdim=True)
            out = out + share * torch.tanh(y @ experts[e])
        return out, r, idx

    leaves = [t.clone().requires_grad_() for t in (x, res, w, gate, experts)]
    out, r, idx = block(*leaves, True)
    assert ((idx >= offset) & (idx < offset + E)).sum() > T // 2
    got = [out, *torch.autograd.grad((out, r), leaves, (gy, gr))]
    leaves64 = [t.double().requires_grad_() for t in (x, res, w, gate, experts)]
    out64, r64, _ = block(*leaves64, False, idx)
    want = [out64, *torch.autograd.grad((out64, r64), leaves64, (gy.double(), gr.double()))]
    for name, a, b in zip(("out", "x", "res", "w", "gate", "experts"), got, want):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= 1.5e-3, (name, rel)


@pytest.mark.parametrize("T, n, align, K", [(10, 64, 1, 8), (200, 520, 16, 8), (700, 2048, 1, 3)])
def test_rows_whose_pair_has_lost_them_are_zeros(tok, T, n, align, K):
    """A map that has been edited behind the sort (pairs dropped with -1, entries outside the
    buffers): the rows that no pair names any more are zeros, like all rows without a pair."""
    idx = select(T, K, 30, "uniform")
    plan = tok.sort_tokens(idx, 256, align=align)
    R = plan.rows
    g = torch.Generator(device="cuda").manual_seed(22)
    x, gy = torch.randn(T, n, generator=g, device="cuda"), torch.randn(T, n, generator=g, device="cuda")
    h, w = torch.randn(R, n, generator=g, device="cuda"), torch.randn(T, K, generator=g, device="cuda")
    edited = plan.scatter_map.clone()
    edited[::3, 0], edited[1::3, 1], edited[2::3, 2] = -1, R, -2 ** 31
    named = torch.zeros(R, dtype=torch.bool, device="cuda")
    named[edited[(edited >= 0) & (edited < R)].long()] = True
    full = tok.gather_tokens(x, plan), tok.combine_tokens_backward(gy, h, w, plan)[0]
    for pairs in (plan.row_pairs, plan.row_pairs.clone().fill_(2 ** 31 - 1)):
        plan2 = plan._replace(scatter_map=edited, row_pairs=pairs)
        if pairs is not plan.row_pairs:   # pairs that are none of the batch's: no row is anybody's
            plan2 = plan2._replace(scatter_map=torch.full_like(edited, -1))
            named = torch.zeros_like(named)
        poison(R, n, F32)
        xs = tok.gather_tokens(x, plan2)
        assert torch.equal(xs, torch.where(named[:, None], full[0], 0.0))
        poison(R, n, F32)
        gh, gw = tok.combine_tokens_backward(gy, h, w, plan2)
        assert torch.equal(gh, torch.where(named[:, None], full[1], 0.0))
        assert gw[(plan2.scatter_map < 0) | (plan2.scatter_map >= R)].eq(0).all()


def test_rows_of_a_larger_batch_are_zeros(tok):
    """row_pairs of a batch with more tokens: pairs behind the batch's own are none of it."""
    big, small = tok.sort_tokens(select(40, 8, 31), 256), tok.sort_tokens(select(20, 8, 32), 256, rows=320)
    x = torch.randn(20, 64, device="cuda")
    behind = (big.row_pairs >= 160) & ~torch.isin(torch.arange(320, device="cuda", dtype=torch.int32), small.scatter_map.flatten())
    assert behind.any()
    poison(320, 64, F32)
    xs = tok.gather_tokens(x, small._replace(row_pairs=big.row_pairs))
    assert xs[behind].eq(0).all()


def test_every_backward_pass_asks_for_a_capture_first(tok, monkeypatch):
    """Under capture autograd's backward passes are refused before they launch anything: each of the four asks, and names the
    explicit function that is there instead."""
    from fused_moe_b200 import norm

    class Asked(RuntimeError):
        pass

    def ask(instead, device):
        raise Asked(f"{instead} {device.type}")

    idx = select(6, 8, 33)
    plan = tok.sort_tokens(idx, 256)
    x, h, w, logits, res, weight = (torch.randn(s, device="cuda").requires_grad_()
                                    for s in ((6, 64), (48, 64), (6, 8), (6, 256), (6, 64), (64,)))
    y, r = norm.add_rms_norm(x, res, weight)
    outs = ((y, "add_rms_norm_backward"), (r, "add_rms_norm_backward"), (norm.add_rms_norm(x, None, weight)[0], "add_rms_norm_backward"),
            (tok.gather_tokens(x, plan), "gather_tokens_backward"), (tok.combine_tokens(h, w, plan), "combine_tokens_backward"),
            (tok.route_weights(logits, idx, 2.5), "route_weights_backward"))
    with monkeypatch.context() as m:
        m.setattr(norm, "refuse_capture", ask)
        m.setattr(tok, "refuse_capture", ask)
        for out, name in outs:
            with pytest.raises(Asked, match=name + " cuda"):
                out.sum().backward(retain_graph=True)
    for out, _ in outs:   # and without a capture they run (y and r are of one node)
        out.sum().backward(retain_graph=True)
    assert all(t.grad is not None and t.grad.isfinite().all() for t in (x, h, w, logits, res, weight))
