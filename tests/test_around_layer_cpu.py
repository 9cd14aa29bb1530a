"""CPU: what the operators around the layer (norm, token permutation, routing weights) refuse, in Python and at the C ABI.  Every
call here ends before a launch."""
import ctypes as C

import pytest
import torch

from fused_moe_b200 import _lib, norm, tokens

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(T=3, n=256, dtype=BF16):
    return torch.zeros((T, n), dtype=dtype)


NORM_REFUSED = [
    (TypeError, dict(x=None)),
    (TypeError, dict(x=rows(dtype=torch.float64))),
    (ValueError, dict(x=torch.zeros(256, dtype=BF16))),
    (ValueError, dict(x=rows(n=252), residual=rows(n=252), weight=torch.zeros(252))),
    (ValueError, dict(x=rows(n=16512), residual=None, weight=torch.zeros(16512))),
    (ValueError, dict(x=rows(n=0), residual=None, weight=torch.zeros(0))),
    (TypeError, dict(residual=rows(dtype=F16))),
    (ValueError, dict(residual=rows(T=4))),
    (TypeError, dict(residual=1.0)),
    (TypeError, dict(weight=None)),
    (TypeError, dict(weight=torch.zeros(256, dtype=torch.int32))),
    (TypeError, dict(weight=torch.zeros(256, dtype=F16))),
    (ValueError, dict(weight=torch.zeros(128))),
    (ValueError, dict(eps=-1e-6)),
    (ValueError, dict(eps=float("nan"))),
    (RuntimeError, {}),   # all is well but for the device: no CPU path
]


@pytest.mark.parametrize("error, change", NORM_REFUSED, ids=range(len(NORM_REFUSED)))
@pytest.mark.parametrize("call", [norm.add_rms_norm, norm.add_rms_norm_quantize])
def test_norm_refuses(call, error, change):
    args = dict(x=rows(), residual=rows(), weight=torch.zeros(256), eps=1e-6) | change
    with pytest.raises(error):
        call(args["x"], args["residual"], args["weight"], args["eps"])


def test_quantize_refuses():
    with pytest.raises(ValueError, match="multiple of 128"):
        norm.add_rms_norm_quantize(rows(n=72), None, torch.zeros(72))
    with pytest.raises(ValueError, match="residual_out needs"):
        # a meta tensor passes for a CUDA one nowhere: the device check comes first
        norm.add_rms_norm_quantize(_cuda_like(rows()), None, _cuda_like(torch.zeros(256)), residual_out=rows())


class _Fake(torch.Tensor):
    """A CPU tensor that reports a CUDA device, for checks behind the device check."""

    @property
    def device(self):
        return torch.device("cuda", 0)

    @property
    def is_cuda(self):
        return True


def _cuda_like(t):
    return t.as_subclass(_Fake)


def test_quantize_refuses_bad_destinations():
    x, w = _cuda_like(rows()), _cuda_like(torch.zeros(256))
    res = _cuda_like(rows())
    for out, error in ((rows(T=4), ValueError), (rows(dtype=F32), TypeError), (rows(n=512)[:, ::2], ValueError),
                       (torch.zeros(3 * 256 + 1, dtype=BF16)[1:].view(3, 256), ValueError)):
        with pytest.raises(error):
            norm.add_rms_norm_quantize(x, res, w, residual_out=_cuda_like(out))
    both = torch.zeros(5 * 256, dtype=BF16)
    with pytest.raises(ValueError, match="overlaps residual"):
        norm.add_rms_norm_quantize(x, _cuda_like(both[:768].view(3, 256)), w, residual_out=_cuda_like(both[256:1024].view(3, 256)))
    with pytest.raises(ValueError, match="overlaps x"):
        norm.add_rms_norm_quantize(_cuda_like(both[:768].view(3, 256)), res, w,
                                   residual_out=_cuda_like(both[512:].view(3, 256)))
    with pytest.raises(ValueError, match="overlaps weight"):
        norm.add_rms_norm_quantize(x, res, _cuda_like(both[:256]), residual_out=_cuda_like(both[:768].view(3, 256)))


def test_overlap_of_ranges():
    t = torch.zeros(100)
    assert norm._overlap(t, t) and norm._overlap(t[10:20], t[19:21]) and not norm._overlap(t[:10], t[10:])
    assert norm._overlap(t.view(10, 10)[:, :5], t.view(10, 10)[:, 5:]) and not norm._overlap(t[5:5], t)


def test_norm_backward_refuses():
    g, r, w = rows(), rows(), torch.zeros(256)
    for args, error in (((g, None, None, w), TypeError), ((g, rows(T=4), r, w), ValueError),
                        ((g, rows(dtype=F32), r, w), TypeError), ((g, None, rows(dtype=F16), w), TypeError),
                        ((g, None, r, w), RuntimeError)):
        with pytest.raises(error):
            norm.add_rms_norm_backward(*args)


def ids(T=3, K=8, dtype=torch.int32):
    return torch.zeros((T, K), dtype=dtype)


@pytest.mark.parametrize("error, args, more", [
    (TypeError, (None, 32), {}),
    (TypeError, (ids(dtype=torch.int64), 32), {}),
    (ValueError, (ids(K=9), 32), {}),
    (ValueError, (ids(K=0), 32), {}),
    (ValueError, (torch.zeros(8, dtype=torch.int32), 32), {}),
    (ValueError, (ids(), 0), {}),
    (ValueError, (ids(), 257), {}),
    (ValueError, (ids(), 32, 225), {}),
    (ValueError, (ids(), 32, -1), {}),
    (ValueError, (ids(), 32), {"align": 0}),
    (ValueError, (ids(), 256), {"align": 1 << 23}),
    (ValueError, (ids(), 32), {"rows": -1}),
    (ValueError, (ids(), 32), {"rows": (1 << 30) + 1}),
    (RuntimeError, (ids(), 32), {}),
], ids=range(14))
def test_sort_refuses(error, args, more):
    with pytest.raises(error):
        tokens.sort_tokens(*args, **more)


def plan(T=3, K=8, n=24):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return tokens.TokenSort(i(32), i(33), i(n), i(T, K), n, 1)


def test_gather_and_combine_refuse():
    w = torch.zeros((3, 8))
    for call, error in (
            (lambda: tokens.gather_tokens(rows(), "plan"), TypeError),
            (lambda: tokens.gather_tokens(rows(T=4), plan()), ValueError),
            (lambda: tokens.gather_tokens(rows(n=4), plan()), ValueError),              # 8 bytes
            (lambda: tokens.gather_tokens(rows(n=6, dtype=F32), plan()), ValueError),   # 24 bytes
            (lambda: tokens.gather_tokens(rows(n=0), plan()), ValueError),
            (lambda: tokens.gather_tokens(rows(dtype=torch.int32), plan()), TypeError),
            (lambda: tokens.gather_tokens(rows(), plan()), RuntimeError),
            (lambda: tokens.gather_tokens_backward(rows(T=3), plan()), ValueError),
            (lambda: tokens.combine_tokens(rows(T=23), w, plan()), ValueError),
            (lambda: tokens.combine_tokens(rows(T=24), w.bfloat16(), plan()), RuntimeError),   # the device comes first
            (lambda: tokens.combine_tokens(rows(T=24), w, plan()), RuntimeError),
            (lambda: tokens.combine_tokens(_cuda_like(rows(T=24)), w.bfloat16(), _cuda_plan()), TypeError),
            (lambda: tokens.combine_tokens(_cuda_like(rows(T=24)), w[:, :4], _cuda_plan()), ValueError),
            (lambda: tokens.combine_tokens_backward(_cuda_like(rows()), rows(T=24, dtype=F32), w, _cuda_plan()), TypeError),
            (lambda: tokens.combine_tokens_backward(_cuda_like(rows()), rows(T=23), w, _cuda_plan()), ValueError),
            (lambda: tokens.combine_tokens_backward(rows(T=24), rows(T=24), w, plan()), ValueError)):
        with pytest.raises(error):
            call()


def _cuda_plan():
    p = plan()
    return tokens.TokenSort(*(_cuda_like(t) for t in (p.counts, p.offsets, p.row_pairs, p.scatter_map)), p.rows, p.align)


def test_route_weights_refuses():
    logits = torch.zeros((3, 256))
    for args, error in (((logits, ids(dtype=torch.int64), 1.0), TypeError), ((logits.bfloat16(), ids(), 1.0), TypeError),
                        ((logits[:, :128], ids(), 1.0), ValueError), ((logits, ids(T=4), 1.0), ValueError),
                        ((logits, ids(K=9), 1.0), ValueError), ((logits, ids(), 1.0), RuntimeError)):
        with pytest.raises(error):
            tokens.route_weights(*args)
    with pytest.raises(RuntimeError):
        tokens.route_weights_backward(logits, ids(), torch.zeros((3, 8)), 1.0)


# ---- the C ABI: every refusal comes before the device is looked at --------------------------------------------------------
A = 1 << 20   # an address that is never followed


@pytest.fixture(scope="module")
def lib():
    from fused_moe_b200 import build
    build.build()
    return _lib.load()


def with_args(base, **change):
    d = dict(base)
    assert set(change) <= set(d)
    d.update(change)
    return tuple(d.values())


def test_norm_abi_refuses(lib):
    base = dict(x=A, x_pitch=0, x_type=0, residual=A, r_pitch=0, r_type=0, weight=A, w_type=0, T=4, columns=256, eps=1e-6,
                stream_out=A, y=A, q=A, scale=A, stream=None)
    for change in (dict(x=None), dict(x=A + 8), dict(x_pitch=8), dict(x_pitch=-16), dict(x_type=3), dict(x_type=-1),
                   dict(r_type=1), dict(residual=A + 2), dict(weight=None), dict(weight=A + 4), dict(w_type=7), dict(w_type=1), dict(T=-1),
                   dict(T=(1 << 24) + 1), dict(columns=0), dict(columns=260), dict(columns=264), dict(columns=16512),
                   dict(eps=-1.0), dict(eps=float("nan")), dict(stream_out=None), dict(q=None), dict(scale=None),
                   dict(y=None, q=None, scale=None), dict(y=A + 1), dict(q=A + 8)):
        assert lib.b200moe_add_rms_norm(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_add_rms_norm(*with_args(base, T=0, x=None, weight=None)) == 0   # nothing to do
    base = dict(gy=A, gy_pitch=0, type=0, gs=A, gs_pitch=0, r=A, r_pitch=0, r_type=2, weight=A, w_type=2, T=4, columns=256,
                eps=1e-6, gx=A, gr=A, gw=A, partial=A, stream=None)
    for change in (dict(gy=None), dict(r=None), dict(weight=None), dict(partial=None), dict(gx=None, gr=None, gw=None),
                   dict(r_type=1), dict(type=5), dict(gs=A + 4), dict(gs_pitch=4), dict(columns=4), dict(columns=16392),
                   dict(gw=A + 2), dict(T=-1), dict(eps=-1.0)):
        assert lib.b200moe_add_rms_norm_backward(*with_args(base, **change)) == _lib.EINVAL, change


def test_token_abi_refuses(lib):
    n = C.c_size_t(0)
    for T, K, E, rc in ((8, 8, 32, 0), (-1, 8, 32, _lib.EINVAL), (8, 9, 32, _lib.EINVAL), (8, 0, 32, _lib.EINVAL),
                        (8, 8, 0, _lib.EINVAL), (8, 8, 257, _lib.EINVAL), ((1 << 24) + 1, 8, 32, _lib.EINVAL), (0, 8, 32, 0)):
        assert lib.b200moe_token_sort_scratch_bytes(T, K, E, C.byref(n)) == rc, (T, K, E)
    assert lib.b200moe_token_sort_scratch_bytes(8, 8, 32, None) == _lib.EINVAL
    assert lib.b200moe_token_sort_scratch_bytes(1 << 24, 8, 256, C.byref(n)) == 0 and n.value <= 256 * 256 * 4
    base = dict(idx=A, T=8, K=8, E=32, offset=0, align=1, rows=64, scratch=A, bytes=1 << 20, counts=A, offsets=A, row_pairs=A,
                map=A, stream=None)
    for change in (dict(idx=None), dict(K=9), dict(E=0), dict(offset=225), dict(offset=-1), dict(align=0), dict(rows=-1),
                   dict(rows=(1 << 30) + 1), dict(align=1 << 26), dict(counts=None), dict(offsets=None),
                   dict(row_pairs=None), dict(map=None)):
        assert lib.b200moe_token_sort(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_token_sort_scratch_bytes(8, 8, 32, C.byref(n)) == 0 and n.value == 0
    base.update(T=4096)
    assert lib.b200moe_token_sort_scratch_bytes(4096, 8, 32, C.byref(n)) == 0 and n.value > 4
    for change in (dict(scratch=None), dict(scratch=A + 2), dict(bytes=4)):
        assert lib.b200moe_token_sort(*with_args(base, **change)) == _lib.EWORKSPACE, change
    base = dict(x=A, pitch=0, type=0, T=8, K=8, columns=64, rows=64, row_pairs=A, map=A, out=A, stream=None)
    for change in (dict(x=None), dict(x=A + 8), dict(pitch=8), dict(type=3), dict(T=-1), dict(K=0), dict(columns=4),
                   dict(columns=0), dict(rows=-1), dict(row_pairs=None), dict(map=None), dict(out=None), dict(out=A + 4)):
        assert lib.b200moe_token_gather(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_token_gather(*with_args(base, rows=0, out=None)) == 0
    base = dict(x=A, pitch=0, type=0, weights=A, T=8, K=8, columns=64, rows=64, map=A, out=A, stream=None)
    for change in (dict(x=None), dict(x=A + 8), dict(pitch=4), dict(type=-1), dict(T=-1), dict(K=9), dict(columns=12),
                   dict(rows=-1), dict(map=None), dict(out=None), dict(out=A + 4)):
        assert lib.b200moe_token_combine(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_token_combine(*with_args(base, T=0, map=None, out=None)) == 0
    base = dict(g=A, g_pitch=0, x=A, pitch=0, type=0, weights=A, T=8, K=8, columns=64, rows=64, row_pairs=A, map=A, gr=A, gw=A,
                stream=None)
    for change in (dict(g=None), dict(g=A + 8), dict(g_pitch=4), dict(x=None), dict(weights=None), dict(map=None),
                   dict(row_pairs=None), dict(gr=A + 8), dict(K=9), dict(columns=4), dict(rows=-1)):
        assert lib.b200moe_token_combine_backward(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_token_combine_backward(*with_args(base, gr=None, gw=None)) == 0
    for change in (dict(logits=None), dict(idx=None), dict(out=None), dict(K=9), dict(T=-1)):
        base = dict(logits=A, idx=A, T=8, K=8, scale=1.0, out=A, stream=None)
        assert lib.b200moe_route_weights(*with_args(base, **change)) == _lib.EINVAL, change
        base = dict(logits=A, idx=A, grad=A, T=8, K=8, scale=1.0, out=A, stream=None)
        assert lib.b200moe_route_weights_backward(*with_args(base, **change)) == _lib.EINVAL, change
    assert lib.b200moe_route_weights_backward(A, A, None, 8, 8, 1.0, A, None) == _lib.EINVAL
    assert lib.b200moe_route_weights_backward(A, A, A, 8, 8, 1.0, A + 4, None) == _lib.EINVAL


def test_constants_match_the_header():
    import re
    from conftest import ROOT
    header = (ROOT / "include" / "b200moe.h").read_text()
    value = lambda n: eval(re.search(rf"#define {n} (.+)", header).group(1))  # noqa: E731
    assert [value(f"B200MOE_DTYPE_{t}") for t in ("BF16", "F16", "F32")] == [_lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32]
    assert value("B200MOE_NORM_MAX_COLUMNS") == _lib.NORM_MAX_COLUMNS
    assert value("B200MOE_NORM_PARTIAL_ROWS") == _lib.NORM_PARTIAL_ROWS
    assert value("B200MOE_TOKEN_MAX_ROWS") == _lib.TOKEN_MAX_ROWS


def _plan_calls(p):
    """Every call that takes a plan, on tensors that pass for CUDA ones and fit three tokens and 24 rows."""
    x, h, w = (_cuda_like(t) for t in (rows(), rows(T=24), torch.zeros((3, 8))))
    return (lambda: tokens.gather_tokens(x, p), lambda: tokens.gather_tokens_backward(h, p), lambda: tokens.combine_tokens(h, w, p),
            lambda: tokens.combine_tokens_backward(x, h, w, p))


def _ints(*shape, dtype=torch.int32):
    return _cuda_like(torch.zeros(shape, dtype=dtype))


@pytest.mark.parametrize("error, match, change", [
    (ValueError, "plan.rows", lambda: dict(row_pairs=_ints(23))),                    # shorter than the capacity: read past its end
    (ValueError, "plan.rows", lambda: dict(row_pairs=_ints(25))),
    (ValueError, "plan.rows", lambda: dict(row_pairs=_ints(24, 1))),
    (ValueError, "contiguous", lambda: dict(row_pairs=_ints(48)[::2])),
    (TypeError, "row_pairs", lambda: dict(row_pairs=_ints(24, dtype=torch.int64))),
    (TypeError, "row_pairs", lambda: dict(row_pairs=None)),
    (ValueError, "contiguous", lambda: dict(scatter_map=_ints(8, 3).t())),
    (ValueError, "contiguous", lambda: dict(scatter_map=_ints(3, 16)[:, ::2])),
    (TypeError, "scatter_map", lambda: dict(scatter_map=_ints(3, 8, dtype=torch.int64))),
    (TypeError, "scatter_map", lambda: dict(scatter_map=_ints(3, 8, dtype=torch.float32))),
    (TypeError, "scatter_map", lambda: dict(scatter_map=[[0] * 8] * 3)),
    (ValueError, "scatter_map", lambda: dict(scatter_map=_ints(24))),
    (ValueError, "scatter_map", lambda: dict(scatter_map=_ints(3, 9))),
    (ValueError, "scatter_map", lambda: dict(scatter_map=_ints(3, 0))),
    (RuntimeError, "CUDA|device", lambda: dict(row_pairs=torch.zeros(24, dtype=torch.int32))),
    (RuntimeError, "CUDA|device", lambda: dict(scatter_map=torch.zeros((3, 8), dtype=torch.int32))),
], ids=range(16))
@pytest.mark.parametrize("which", range(4))
def test_plans_whose_arrays_do_not_fit_are_refused(which, error, match, change):
    """A plan is a public tuple: its arrays may come from anywhere."""
    with pytest.raises(error, match=match):
        _plan_calls(_cuda_plan()._replace(**change()))[which]()


@pytest.mark.parametrize("which", range(4))
def test_a_plan_with_a_larger_capacity_than_its_arrays_is_refused(which):
    p = _cuda_plan()._replace(rows=1000)
    x, h, w = (_cuda_like(t) for t in (rows(), rows(T=1000), torch.zeros((3, 8))))
    with pytest.raises(ValueError, match="plan.rows"):
        (lambda: tokens.gather_tokens(x, p), lambda: tokens.gather_tokens_backward(h, p), lambda: tokens.combine_tokens(h, w, p),
         lambda: tokens.combine_tokens_backward(x, h, w, p))[which]()


# ---- derivatives that an operator does not have -------------------------------------------------------------------------------
def _operators():
    """(call on a dict of tensors, names of its tensors that have a derivative); on tensors that pass for CUDA ones."""
    t = {k: _cuda_like(v) for k, v in dict(
        x=rows(), res=rows(), w=torch.ones(256), h=rows(T=24), tw=torch.zeros((3, 8)), logits=torch.zeros((3, 256)),
        gy=rows(), gs=rows(), gl=torch.zeros((3, 8))).items()}
    p, i = _cuda_plan(), _cuda_like(ids())
    return t, {
        "add_rms_norm": (lambda a: norm.add_rms_norm(a["x"], a["res"], a["w"]), ("x", "res", "w")),
        "first norm": (lambda a: norm.add_rms_norm(a["x"], None, a["w"]), ("x", "w")),
        "add_rms_norm_backward": (lambda a: norm.add_rms_norm_backward(a["gy"], a["gs"], a["res"], a["w"]), ("gy", "gs", "res", "w")),
        "add_rms_norm_quantize": (lambda a: norm.add_rms_norm_quantize(a["x"], a["res"], a["w"]), ("x", "res", "w")),
        "gather_tokens": (lambda a: tokens.gather_tokens(a["x"], p), ("x",)),
        "gather_tokens_backward": (lambda a: tokens.gather_tokens_backward(a["h"], p), ("h",)),
        "combine_tokens": (lambda a: tokens.combine_tokens(a["h"], a["tw"], p), ("h", "tw")),
        "combine_tokens_backward": (lambda a: tokens.combine_tokens_backward(a["x"], a["h"], a["tw"], p), ("x", "h", "tw")),
        "route_weights": (lambda a: tokens.route_weights(a["logits"], i, 2.5), ("logits",)),
        "route_weights_backward": (lambda a: tokens.route_weights_backward(a["logits"], i, a["gl"], 2.5), ("logits", "gl"))}


@pytest.mark.parametrize("name", list(_operators()[1]))
def test_tangents_are_refused(name):
    """A dual tensor does not require a gradient; its tangent must not get lost."""
    from torch.autograd import forward_ad
    t, calls = _operators()
    call, names = calls[name]
    for which in names:
        with forward_ad.dual_level():
            dual = _cuda_like(forward_ad.make_dual(t[which].as_subclass(torch.Tensor), torch.ones(t[which].shape, dtype=t[which].dtype)))
            assert not dual.requires_grad and forward_ad.unpack_dual(dual).tangent is not None
            with pytest.raises(RuntimeError, match="carries a tangent"):
                call(t | {which: dual})


def test_tangents_of_incoming_gradients_are_refused():
    """Forward over reverse: the gradient of the result carries the tangent, the inputs do not."""
    from torch.autograd import forward_ad
    from fused_moe_b200.rows import differentiable_once

    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return 2 * x

        @staticmethod
        @differentiable_once
        def backward(ctx, g):
            return g.detach() * 2

    x = torch.zeros(3, requires_grad=True)
    y = Double.apply(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="carries a tangent"):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones(3), torch.ones(3)), retain_graph=True)
    assert torch.autograd.grad(y, x, torch.ones(3))[0].eq(2).all()


@pytest.mark.parametrize("which", ["x", "res", "w"])
@pytest.mark.parametrize("residual", [True, False])
def test_the_quantised_norm_refuses_to_drop_a_gradient(monkeypatch, which, residual):
    t, _ = _operators()
    if which == "res" and not residual:
        return
    leaf = t[which].clone().requires_grad_()
    a = t | {which: _cuda_like(leaf) if not isinstance(leaf, _Fake) else leaf}
    call = lambda: norm.add_rms_norm_quantize(a["x"], a["res"] if residual else None, a["w"])  # noqa: E731
    assert a[which].requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        call()
    launched = []
    monkeypatch.setattr(norm, "_forward", lambda *args: launched.append(args))   # no launch from these tensors, wherever this runs
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            call()
    assert len(launched) == 2
    empty = {k: _cuda_like(v[:0].detach().clone().requires_grad_()) if k in ("x", "res") else v for k, v in t.items()}
    norm.add_rms_norm_quantize(empty["x"], empty["res"] if residual else None, empty["w"])   # has no gradient to lose


def test_a_scaling_factor_that_requires_a_gradient_is_refused(monkeypatch):
    from torch.autograd import forward_ad
    t, _ = _operators()
    i, scale = _cuda_like(ids()), torch.tensor(2.5, requires_grad=True)
    calls = (lambda s: tokens.route_weights(t["logits"], i, s), lambda s: tokens.route_weights_backward(t["logits"], i, t["gl"], s))
    for call in calls:
        with pytest.raises(RuntimeError, match="routed_scaling_factor has no gradient"):
            call(scale)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="carries a tangent"):
            call(forward_ad.make_dual(scale.detach(), torch.tensor(1.0)))
    seen = []
    monkeypatch.setattr(tokens, "_route_weights", lambda logits, idx, s: seen.append(s))
    monkeypatch.setattr(tokens, "_route_weights_backward", lambda logits, idx, grad, s: seen.append(s))
    for call in calls:
        call(scale.detach())
        with torch.no_grad():
            call(scale)
    assert seen == [2.5] * 4


def test_the_number_of_multiprocessors_is_the_devices():
    """No launch rule has one GPU's count of SMs (148, or four CTAs on each, 592) written into it."""
    import re
    from conftest import ROOT
    for name in ("norm.cu", "tokens.cu"):
        code = re.sub(r"//[^\n]*", "", (ROOT / "fused_moe_b200" / "csrc" / name).read_text())
        assert not re.search(r"\b(148|296|444|592)\b", code), name
