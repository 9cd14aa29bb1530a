"""GPU: residual addition + RMS norm (and its e4m3 form, and its gradient) against the formulas in 64 bits.

Tolerances.  u(t) is half a step of type t (its relative rounding error).  The residual stream is one float32 addition and one
rounding, which torch repeats bit for bit.  The mean square is a float32 sum of non-negative terms: at most 32 in a
thread's chain, 5 + 5 levels of the tree, and a few roundings for the division, the root and the two products, together below
2^-19 relative.  Products of signed terms are bounded by the same factor times the sum of the terms' magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6
ARITH = 2.0 ** -19


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of the type: what a rounding among its subnormal values may be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def norm():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from fused_moe_b200 import norm as module
    return module


def make(T, n, dtype, stream, weight_type=None, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + T + n)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = (scale * rnd(T, n)).to(dtype)
    res = None if stream is None else (3 * scale * rnd(T, n)).to(stream)
    w = (1 + 0.1 * rnd(n)).to(weight_type or dtype)
    return x, res, w, rnd


def ref64(x, res, w, eps=EPS):
    """(r as its type holds it, y in 64 bits)."""
    r = x if res is None else (x.float() + res.float()).to(res.dtype)
    h = r.double()
    return r, h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps) * w.double()


def assert_within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(err / tol)[bad].max().item():.3f} x"


def poison(*shapes):
    """Leaves NaN in the memory that the next allocations of these sizes will get."""
    for shape, dtype in shapes:
        torch.full(shape, float("nan"), device="cuda", dtype=F32).to(dtype)


SHAPES = [(1, 8), (1, 7168), (2, 128), (3, 200), (7, 512), (5, 2048), (33, 2056), (17, 4096), (4, 4104), (3, 8192), (2, 16384),
          (333, 7168), (1025, 264), (1030, 7168), (1026, 2056), (1100, 1024), (2000, 576), (70001, 128)]
TYPES = [(BF16, BF16), (BF16, F32), (BF16, None), (F16, F16), (F16, F32), (F32, F32), (F32, None)]


@pytest.mark.parametrize("dtype, stream", TYPES, ids=str)
@pytest.mark.parametrize("T, n", SHAPES)
def test_forward(norm, T, n, dtype, stream):
    x, res, w, _ = make(T, n, dtype, stream, F32 if T % 2 else None)
    r, y = ref64(x, res, w)
    poison(((T, n), dtype), ((T, n), stream or dtype))
    got_y, got_r = norm.add_rms_norm(x, res, w, EPS)
    assert got_y.dtype is dtype and torch.equal(got_r, r)
    if res is None:
        assert got_r is x
    assert_within(got_y, y, (u(dtype) + ARITH) * y.abs() + tiny(dtype), "y")


@pytest.mark.parametrize("dtype, stream", TYPES, ids=str)
@pytest.mark.parametrize("T, n", [s for s in SHAPES if s[1] % 128 == 0] + [(260, 7168), (9, 2176), (6, 16256)])
def test_quantize(norm, T, n, dtype, stream):
    """Every e4m3 value within half a step of y / scale (2^-4 relative, 2^-10 among the subnormals), the scales within the
    arithmetic's bound of amax / 448; and r and y as the float form gives them."""
    x, res, w, _ = make(T, n, dtype, stream, seed=1)
    _, y = ref64(x, res, w)
    want_y, want_r = norm.add_rms_norm(x, res, w, EPS)
    q, s, r, got_y = norm.add_rms_norm_quantize(x, res, w, EPS, with_normed=True)
    assert q.dtype is torch.float8_e4m3fn and s.shape == (n // 128, T)
    assert torch.equal(r, want_r) and torch.equal(got_y, want_y)
    scale = (y.abs().view(T, -1, 128).amax(dim=2) / 448).clamp_min(1e-12)
    assert_within(s.t(), scale, 2 * ARITH * scale, "scales")
    v = y / scale.repeat_interleave(128, dim=1)
    assert_within(q, v, torch.maximum(2.0 ** -4 * (1 + 2.0 ** -10) * v.abs(), torch.full_like(v, 2.0 ** -10 * (1 + 2.0 ** -10))), "q")
    q2, s2, _ = norm.add_rms_norm_quantize(x, res, w, EPS)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


def test_quantize_is_the_layers_rule_on_the_float32_rows(norm):
    """With float32 rows y itself is an output, so the rule of the quantiser (every operation rounded to float32) can be repeated
    on the CPU, bit for bit."""
    x, res, w, _ = make(37, 7168, F32, F32, seed=2)
    x[3] = 0
    res[3] = 0
    res[4, :256] *= 1e4
    q, s, _, y = norm.add_rms_norm_quantize(x, res, w, EPS, with_normed=True)
    y = y.cpu().view(37, 56, 128)
    scale = (y.abs().amax(dim=2) * (1.0 / 448.0)).clamp_min(1e-12)
    want = (y * (1.0 / scale).unsqueeze(2)).clamp(-448, 448).to(torch.float8_e4m3fn).view(37, 7168)
    assert torch.equal(s.cpu(), scale.t())
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))
    assert s.cpu()[:, 3].eq(1e-12).all()   # a row of zeros


def test_rows_that_are_not_finite_stay_by_themselves(norm):
    """A NaN or an infinity spoils its own row (scales included) and no other."""
    x, res, w, _ = make(6, 1024, BF16, BF16, seed=3)
    clean = norm.add_rms_norm_quantize(x, res, w, EPS, with_normed=True)
    x[1, 5] = float("nan")
    res[3, 900] = float("inf")
    q, s, r, y = norm.add_rms_norm_quantize(x, res, w, EPS, with_normed=True)
    keep = [0, 2, 4, 5]
    assert torch.equal(q.view(torch.uint8)[keep], clean[0].view(torch.uint8)[keep])
    assert torch.equal(s[:, keep], clean[1][:, keep]) and torch.equal(y[keep], clean[3][keep])
    assert y[1].isnan().all() and s[:, 1].isnan().all() and q[1].float().isnan().all()
    assert y[3, 900].isnan() and s[7, 3].isnan() and y[3, :900].eq(0).all() and s[0, 3] == 1e-12


def test_large_and_small_rows(norm):
    """Magnitudes at which the mean square is far from 1; eps decides where rows vanish."""
    for scale, dtype in ((1e-4, BF16), (1e4, BF16), (1e-18, F32), (1e16, F32), (1e-3, F16), (100.0, F16)):
        x, res, w, _ = make(9, 2048, dtype, dtype, seed=4, scale=scale)
        r, y = ref64(x, res, w)
        got, got_r = norm.add_rms_norm(x, res, w, EPS)
        assert torch.equal(got_r, r)
        assert_within(got, y, (u(dtype) + ARITH) * y.abs() + tiny(dtype), f"y at {scale}")
    x = torch.zeros((2, 256), dtype=F32, device="cuda")
    assert norm.add_rms_norm(x, None, torch.ones(256, device="cuda"), EPS)[0].eq(0).all()


def test_strided_and_unaligned_inputs(norm):
    """Row slices of wider tensors are read in place; other layouts through a copy: the same bits as dense inputs."""
    T, n = 21, 640
    wide, wide_res, w, _ = make(T, 3 * n, BF16, BF16, seed=5)
    w = w[:n].clone()
    layouts = [(wide[:, n:2 * n], wide_res[:, :n]),                       # in place
               (wide[:, 4:4 + n], wide_res[:, 1:1 + n]),                  # rows not on 16 bytes
               (wide[:, ::2][:, :n], wide_res.t().contiguous().t()[:, :n]),
               (wide[:1].expand(T, 3 * n)[:, :n], wide_res[:, :n]),       # one row for all
               (wide.flatten()[8:8 + T * n].view(T, n), wide.flatten()[3:3 + T * n].view(T, n)),
               (wide[::3, :n][:7], wide_res[1:8, :n])]
    for x, res in layouts:
        dx, dres = x.contiguous().clone(), res.contiguous().clone()
        for a, b in zip(norm.add_rms_norm_quantize(x, res, w, EPS, with_normed=True),
                        norm.add_rms_norm_quantize(dx, dres, w, EPS, with_normed=True)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                               b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
        gy = torch.randn(x.shape, device="cuda").bfloat16()
        for a, b in zip(norm.add_rms_norm_backward(gy, x, res, w), norm.add_rms_norm_backward(gy, dx, dres, w)):
            assert torch.equal(a, b)
    odd = torch.randn(n + 1, device="cuda").bfloat16()[1:]                # a weight that is not on 16 bytes
    x, res = wide[:, :n].contiguous(), wide_res[:, :n].contiguous()
    assert torch.equal(norm.add_rms_norm(x, res, odd)[0], norm.add_rms_norm(x, res, odd.clone())[0])


def test_destinations(norm):
    x, res, w, _ = make(40, 7168, BF16, BF16, seed=6)
    q, s, r = norm.add_rms_norm_quantize(x, res, w)
    out = torch.full_like(res, float("nan"))
    q1, s1, r1 = norm.add_rms_norm_quantize(x, res, w, residual_out=out)
    assert r1 is out and torch.equal(out, r)
    own = res.clone()
    q2, s2, r2 = norm.add_rms_norm_quantize(x, own, w, residual_out=own)
    assert r2 is own and torch.equal(own, r)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s1) and torch.equal(s, s2)
    wide = torch.full((42, 7168), 3.0, dtype=BF16, device="cuda")          # nothing beside the rows is written
    norm.add_rms_norm_quantize(x, res, w, residual_out=wide[1:41])
    assert wide[0].eq(3).all() and wide[41].eq(3).all() and torch.equal(wide[1:41], r)
    both = res.clone()                                                      # x and the residual are one tensor, and so is r
    want = norm.add_rms_norm(both, both, w)
    assert torch.equal(norm.add_rms_norm_quantize(both, both, w, residual_out=both)[2], want[1])


def grads64(gy, gs, r, w, eps=EPS):
    """Gradients by the formula, and the magnitudes of the terms that make them up."""
    g, h, w = gy.double(), r.double(), w.double()
    n = h.shape[1]
    rstd = 1 / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps)
    up = g * w
    dr = rstd * (up - h * rstd.square() * (up * h).mean(dim=1, keepdim=True))
    size = rstd * (up.abs() + h.abs() * rstd.square() * (up * h).abs().mean(dim=1, keepdim=True))
    if gs is not None:
        dr, size = dr + gs.double(), size + gs.double().abs()
    unit = h * rstd
    return dr, size, (g * unit).sum(dim=0), (g * unit).abs().sum(dim=0)


@pytest.mark.parametrize("dtype, stream", TYPES, ids=str)
@pytest.mark.parametrize("T, n", SHAPES + [(700, 512), (1500, 72)])
def test_backward(norm, T, n, dtype, stream):
    """The weight's gradient is a float32 sum over tokens: at most ceil(T / 148) + 64 + 8 terms in a chain behind the 2^-19 of its
    terms."""
    x, res, w, rnd = make(T, n, dtype, stream, F32 if n % 3 == 0 else None, seed=7)
    gy = rnd(T, n).to(dtype)
    gs = None if stream is None else rnd(T, n).to(stream)
    leaves = [t.requires_grad_() for t in (x, res, w) if t is not None]
    y, r = norm.add_rms_norm(x, res, w, EPS)
    poison(((T, n), dtype), ((T, n), stream or dtype), ((min(T, 512), n), F32))
    outs = (y,) if res is None else (y, r)
    grads = torch.autograd.grad(outs, leaves, (gy,) if res is None else (gy, gs))
    dr, size, dw, dw_size = grads64(gy, gs, r.detach(), w.detach())
    for got, leaf in zip(grads[:-1], leaves):
        assert got.dtype is leaf.dtype
        assert_within(got, dr, u(got.dtype) * dr.abs() + 2 * ARITH * size + tiny(got.dtype), "grad of x or residual")
    chain = (T / 148 + 73) * 2.0 ** -24
    assert grads[-1].dtype is w.dtype
    assert_within(grads[-1], dw, u(w.dtype) * dw.abs() + (ARITH + chain) * dw_size + tiny(w.dtype), "grad of weight")
    again = norm.add_rms_norm_backward(gy, gs, r.detach(), w.detach(), EPS)   # the explicit form: the same bits
    assert torch.equal(again[0], grads[0]) and torch.equal(again[2], grads[-1])
    if res is not None:
        assert torch.equal(again[1], grads[1])


def test_backward_against_differences(norm):
    """Directional derivatives of the 64-bit function.  With step h the central difference is off by h^2 / 6 times the third
    derivative (of order 1 per unit of sum |g|, h = 1e-5: 1e-10) and by 2^-52 / h (2e-11) of the same."""
    T, n = 5, 264
    x, res, w, rnd = make(T, n, F32, F32, seed=8)
    gy, gs = rnd(T, n), rnd(T, n)
    got = norm.add_rms_norm_backward(gy, gs, x + res, w, EPS)

    def f(x, res, w):
        r = x + res
        return ((r / torch.sqrt(r.square().mean(dim=1, keepdim=True) + EPS) * w) * gy.double()).sum() + (r * gs.double()).sum()

    args = [t.double() for t in (x, res, w)]
    _, size, _, dw_size = grads64(gy, gs, x + res, w)
    for i, grad in enumerate(got):
        d = torch.randn(args[i].shape, dtype=torch.float64, device="cuda")
        step = lambda h: [a + h * d if j == i else a for j, a in enumerate(args)]  # noqa: E731
        diff = (f(*step(1e-5)) - f(*step(-1e-5))) / 2e-5
        budget = ((size if i < 2 else dw_size) * d.abs()).sum() * (2 * ARITH + 2.0 ** -17)
        # x + res rounds to float32 in `got` and not here: 2^-24 relative in r, which the budget's last term covers
        assert abs((grad.double() * d).sum() - diff) <= budget + 1e-8 * (gy.abs().sum() + gs.abs().sum())


def test_partial_uses_of_the_results(norm):
    """Only y, only r, or not all inputs differentiable."""
    x, res, w, rnd = make(19, 512, BF16, F32, seed=9)
    gy, gs = rnd(19, 512).bfloat16(), rnd(19, 512)
    xl, rl, wl = (t.clone().requires_grad_() for t in (x, res, w))
    y, r = norm.add_rms_norm(xl, rl, wl)
    only_y = torch.autograd.grad(y, (xl, rl, wl), gy, retain_graph=True)
    want = norm.add_rms_norm_backward(gy, None, r.detach(), w)
    assert all(torch.equal(a, b) for a, b in zip(only_y, want))
    only_r = torch.autograd.grad(r, (xl, rl, wl), gs, allow_unused=True, retain_graph=True)
    assert torch.equal(only_r[0], gs.bfloat16()) and torch.equal(only_r[1], gs) and (only_r[2] is None or not only_r[2].any())
    full = norm.add_rms_norm_backward(gy, gs, r.detach(), w)
    for which in range(3):
        leaf = (x, res, w)[which].clone().requires_grad_()
        args = [leaf if i == which else t for i, t in enumerate((x, res, w))]
        y, r = norm.add_rms_norm(*args)
        assert torch.equal(torch.autograd.grad((y, r), leaf, (gy, gs))[0], full[which])
    broadcast = torch.ones(1, device="cuda", requires_grad=True)           # a gradient that is one value for all
    y, r = norm.add_rms_norm(xl, rl, wl)
    a = torch.autograd.grad((y * broadcast).sum(), wl)[0]
    b = norm.add_rms_norm_backward(torch.ones_like(y), None, r.detach(), w)[2]
    assert torch.equal(a, b)


def test_one_tensor_as_x_and_residual(norm):
    x, _, w, rnd = make(6, 512, F32, None, seed=10)
    gy, gs = rnd(6, 512), rnd(6, 512)
    leaf = x.clone().requires_grad_()
    y, r = norm.add_rms_norm(leaf, leaf, w)
    got = torch.autograd.grad((y, r), leaf, (gy, gs))[0]
    a, b, _ = norm.add_rms_norm_backward(gy, gs, r.detach(), w)
    assert torch.equal(got, a + b)


def test_offsets_past_32_bits(norm):
    """More than 2^31 elements and 2^32 bytes: the last rows are those of a call on themselves.  (The parts have more than 1024
    rows: below, a row's squares are added by more threads in another order, and a scale may differ in its last bit.)"""
    T, n = 300_032, 7168
    torch.manual_seed(19)
    x = torch.randn(T, n, device="cuda", dtype=BF16)
    res = torch.randn(T, n, device="cuda", dtype=BF16)
    w = torch.randn(n, device="cuda", dtype=BF16)
    q, s, r, y = norm.add_rms_norm_quantize(x, res, w, with_normed=True)
    for part in (slice(0, 1030), slice(T // 2, T // 2 + 1030), slice(T - 1030, T)):
        want = norm.add_rms_norm_quantize(x[part], res[part], w, with_normed=True)
        assert torch.equal(q[part].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s[:, part], want[1])
        assert torch.equal(r[part], want[2]) and torch.equal(y[part], want[3])
    del q, s, r
    gx, gr, gw = norm.add_rms_norm_backward(y, x, res, w)
    for part in (slice(0, 3), slice(T - 3, T)):
        # another launch shape may add a row's squares in another order: a rounding of the result apart
        want = grads64(y[part], x[part], res[part], w)
        assert_within(gx[part], want[0], u(BF16) * want[0].abs() + 2 * ARITH * want[1] + tiny(BF16), "grad")
    assert gr is gx and gw.isfinite().all()


def test_a_destination_counts_the_write(norm):
    """A tensor that autograd has saved notices that it was overwritten; one that requires a gradient is refused."""
    x, res, w, _ = make(4, 256, F32, F32, seed=18)
    leaf = x.clone().requires_grad_()
    y = leaf * res
    norm.add_rms_norm_quantize(x, res, w, residual_out=res)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="must not require"):
        norm.add_rms_norm_quantize(x, res, w, residual_out=res.clone().requires_grad_())


def test_empty_batch(norm):
    w = torch.ones(256, dtype=BF16, device="cuda", requires_grad=True)
    x = torch.empty((0, 256), dtype=BF16, device="cuda", requires_grad=True)
    y, r = norm.add_rms_norm(x, x.detach(), w)
    assert y.shape == r.shape == (0, 256)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert gx.shape == (0, 256) and gw.eq(0).all()
    q, s, _ = norm.add_rms_norm_quantize(x, None, w)
    assert q.shape == (0, 256) and s.shape == (2, 0)


def test_repeats_bit_for_bit_and_on_another_stream(norm):
    x, res, w, rnd = make(777, 2048, BF16, BF16, seed=11)
    gy, gs = rnd(777, 2048).bfloat16(), rnd(777, 2048).bfloat16()
    first = (*norm.add_rms_norm(x, res, w), *norm.add_rms_norm_backward(gy, gs, res, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_()
        other = (*norm.add_rms_norm(x, res, w), *norm.add_rms_norm_backward(gy, gs, res, w))
        y, r = norm.add_rms_norm(leaf, res, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    g = torch.autograd.grad((y, r), leaf, (gy, gs))[0]
    assert torch.equal(g, norm.add_rms_norm_backward(gy, gs, r.detach(), w)[0])


def test_captured_and_replayed(norm):
    """A step without autograd is captured and replayed on new values; a call that would record a gradient is refused and leaves
    the capture usable."""
    x, res, w, rnd = make(50, 7168, BF16, BF16, seed=12)
    gy = rnd(50, 7168).bfloat16()
    leaf = x.clone().requires_grad_()
    y, r = norm.add_rms_norm(leaf, res, w)   # an eager graph of the same leaf stays alive
    norm.add_rms_norm_backward(gy, gy, res, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="add_rms_norm_backward"):
            norm.add_rms_norm(leaf, res, w)
        with torch.no_grad():
            cy, cr = norm.add_rms_norm(leaf, res, w)
        grads = norm.add_rms_norm_backward(gy, gy, cr, w)
        quant = norm.add_rms_norm_quantize(x, res, w)
    for seed in (13, 14):
        nx, nres, _, rnd = make(50, 7168, BF16, BF16, seed=seed)
        x.copy_(nx), res.copy_(nres), gy.copy_(rnd(50, 7168))
        leaf.data.copy_(nx)
        graph.replay()
        torch.cuda.synchronize()
        wy, wr = norm.add_rms_norm(x, res, w)
        assert torch.equal(cy, wy) and torch.equal(cr, wr)
        assert all(torch.equal(a, b) for a, b in zip(grads, norm.add_rms_norm_backward(gy, gy, wr, w)))
        want = norm.add_rms_norm_quantize(x, res, w)
        assert torch.equal(quant[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(quant[1], want[1])


def test_refuses_an_autograd_pass_under_capture(norm):
    x, res, w, rnd = make(4, 256, BF16, BF16, seed=15)
    leaf = x.clone().requires_grad_()
    y, r = norm.add_rms_norm(leaf, res, w)
    ones = torch.ones_like(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    held = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        held += 1
        with pytest.raises(RuntimeError, match="stream capture"):
            from fused_moe_b200 import rows
            rows.refuse_capture("add_rms_norm_backward", x.device)   # what the backward pass calls first
    graph.replay()
    torch.cuda.synchronize()
    assert held.eq(1).all()
    want = norm.add_rms_norm_backward(ones, None, r.detach(), w)[0]
    assert torch.equal(torch.autograd.grad(y, leaf, ones)[0], want)


@pytest.mark.parametrize("T", [3, 80])
def test_feeds_the_layer(norm, oracle, T):
    """The run as it is used: residual stream -> norm and quantisation -> router -> layer, against the oracle's layer on the
    quantised rows that the norm gave."""
    from conftest import assert_close
    from fused_moe_b200 import kernel as K, synth
    base = synth.make_inputs(T, 2, seed=21, local_expert_offset=64, device="cuda")
    x, res, w, rnd = make(T, 7168, BF16, BF16, seed=16)
    q, s, r, y = norm.add_rms_norm_quantize(x, res, w, with_normed=True)
    gate = 0.02 * rnd(256, 7168)
    logits = y.float() @ gate.t()
    logits[:, 64:66] += 2.0   # the local experts see tokens
    args = dict(base, routing_logits=logits, hidden_states=q, hidden_states_scale=s)
    out = K.kernel(**args)
    K.check_status()
    keys = ("routing_logits", "routing_bias", "hidden_states", "hidden_states_scale", "gemm1_weights", "gemm1_weights_scale",
            "gemm2_weights", "gemm2_weights_scale", "local_expert_offset", "routed_scaling_factor")
    want = oracle.kernel(*[args[k].cpu() if torch.is_tensor(args[k]) else args[k] for k in keys])
    assert want["pairs"] > 0 and r.isfinite().all()
    assert_close(out.cpu(), want["out_f32"])


def test_second_derivatives_are_refused(norm):
    """Also where the first gradient came from a constant: it must not pass for a constant of the inputs."""
    x, res, w, rnd = make(3, 128, F32, F32, seed=17)
    x.requires_grad_()
    y, _ = norm.add_rms_norm(x, res, w)
    g = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    assert torch.equal(g, norm.add_rms_norm_backward(torch.ones_like(y), None, (x + res).detach(), w)[0])
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g.sum() + x.square().sum()).backward()


@pytest.mark.parametrize("dtype, stream, scale, grad_scale, eps", [
    (F32, F32, 1e14, 1.0, EPS), (F32, F32, 1e15, 1.0, EPS), (F32, F32, 1e16, 1.0, EPS), (F32, F32, 1e16, 1e-8, EPS),
    (F32, None, 1e-18, 1.0, EPS), (F32, F32, 1e-13, 1.0, 0.0), (F32, None, 1e-16, 1e-3, 0.0), (BF16, BF16, 1e16, 1.0, EPS),
    (BF16, F32, 1e15, 1.0, EPS), (BF16, BF16, 1e-13, 1.0, 0.0), (BF16, BF16, 1e4, 1.0, EPS), (BF16, None, 1e-4, 1.0, EPS),
    (F16, F16, 100.0, 1.0, EPS), (F16, F16, 1e-3, 1.0, EPS)], ids=str)
@pytest.mark.parametrize("T, n", [(9, 2048), (3, 264), (200, 1024)])
def test_backward_of_large_and_small_rows(norm, T, n, dtype, stream, scale, grad_scale, eps):
    """Rows far from magnitude 1, with gradients that have a component along the row, so that both terms of the gradient count.
    No factor leaves the type's range where the result does not.  Rounding errors, in units of 2^-24 of the terms' magnitudes:
    a sum over a row is at most 16 terms in a thread's chain and 10 levels of the tree, once whole for mean(g r) and twice
    half for 1 / sqrt; with the products, divisions and roots at most 64, which is 2^-18."""
    x, res, w, rnd = make(T, n, dtype, stream, seed=20, scale=scale)
    r, _ = ref64(x, res, w, eps)
    unit = r.double() / r.double().square().mean(dim=1, keepdim=True).sqrt()
    gy = (grad_scale * (rnd(T, n) + 0.5 * unit)).to(dtype)
    gs = None if stream is None else (grad_scale * rnd(T, n) / (3 * scale)).to(stream)
    if dtype is F16:
        gs = None   # of the size of the rest of the gradient, it would leave the type's range
    grads = norm.add_rms_norm_backward(gy, gs, r, w, eps)
    dr, size, dw, dw_size = grads64(gy, gs, r, w, eps)
    assert dr.abs().max() > 0.1 * size.max()
    for got in grads[:2]:
        assert got.isfinite().all()
        assert_within(got, dr, u(got.dtype) * dr.abs() + 2.0 ** -18 * size + tiny(got.dtype), "grad of x or residual")
    chain = (T / 148 + 73) * 2.0 ** -24
    assert_within(grads[2], dw, u(w.dtype) * dw.abs() + (ARITH + chain) * dw_size + tiny(w.dtype), "grad of weight")


@pytest.mark.parametrize("dtype, eps", [(F32, 1e-26), (F32, 1e-30), (BF16, 1e-30), (F32, 1e-36)], ids=str)
def test_backward_of_a_row_of_zeros(norm, dtype, eps):
    """dr = g / sqrt(eps), also where eps^(-3/2) would leave float32."""
    r = torch.zeros((3, 512), dtype=dtype, device="cuda")
    r[1] = torch.randn(512, device="cuda").to(dtype)
    gy, w = torch.randn(3, 512, device="cuda").to(dtype), torch.ones(512, dtype=dtype, device="cuda")
    got = norm.add_rms_norm_backward(gy, None, r, w, eps)
    dr, size, dw, dw_size = grads64(gy, None, r, w, eps)
    assert_within(got[0], dr, u(dtype) * dr.abs() + 2.0 ** -18 * size, "grad of x")
    assert_within(got[2], dw, u(dtype) * dw.abs() + 2.0 ** -18 * dw_size, "grad of weight")


@pytest.mark.parametrize("dtype, stream", [(BF16, BF16), (BF16, F32), (F32, F32)], ids=str)
@pytest.mark.parametrize("n", [128, 512, 2048, 7168, 8320])
def test_a_tokens_results_do_not_depend_on_its_neighbours(norm, n, dtype, stream):
    """Bit for bit: the forward among batches of up to 1024 tokens and among larger ones (and, for rows of at most 512 columns or more
    than 8192, across the two), the gradient of a row in any batch."""
    x, res, w, rnd = make(2500, n, dtype, stream, seed=23)
    gy, gs = rnd(2500, n).to(dtype), rnd(2500, n).to(stream)

    def forward(T):
        q, s, r, y = norm.add_rms_norm_quantize(x[:T], res[:T], w, with_normed=True)
        return q.view(torch.uint8), s.t(), r, y

    small, large = {T: forward(T) for T in (1, 5, 333, 1024)}, {T: forward(T) for T in (1025, 2500)}
    for group in (small, large) if 512 < n <= 8192 else (small | large,):
        most = max(group)
        for T, got in group.items():
            assert all(torch.equal(a, b[:T]) for a, b in zip(got, group[most])), (T, most)
    back = {T: norm.add_rms_norm_backward(gy[:T], gs[:T], res[:T], w)[:2] for T in (1, 64, 65, 333, 1100, 2500)}
    for T, got in back.items():
        assert all(torch.equal(a, b[:T]) for a, b in zip(got, back[2500])), T
