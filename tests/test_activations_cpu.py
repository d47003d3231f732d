"""The activation operators without a GPU: what they refuse, the rotation's
plan, and the backward formulas against differences."""
import ctypes
import math

import pytest
import torch

import act_ref as ref
import ark_b200 as ab
from ark_b200 import _lib

INVALID, MISALIGNED, UNSUPPORTED = -1, -2, -8
P = 0x7F0000001000      # an aligned address that nothing reads


def act(rows=64, cols=100, kind=0, data=P, scale=P):
    return _lib.Act8(data, scale, rows, cols, kind, 0)


def by(x):
    return ctypes.byref(x)


# ----------------------------------------------------------------- the C ABI's refusals
def test_pitch():
    L = _lib.lib()
    assert [L.ark_cuda_act8_pitch(c) for c in (0, 1, 128, 129, 768)] == [0, 128, 128, 256, 768]


@pytest.mark.parametrize("want,args", [
    (INVALID, lambda: (P, 0, 100, None)),
    (INVALID, lambda: (P, 0, 100, by(act(kind=2)))),
    (INVALID, lambda: (P, 0, 100, by(act(data=None)))),
    (INVALID, lambda: (P, 7, 100, by(act()))),
    (INVALID, lambda: (P, 3, 100, by(act()))),
    (INVALID, lambda: (P, 0, 99, by(act()))),                 # rows overlap
    (INVALID, lambda: (None, 0, 100, by(act()))),
    (INVALID, lambda: (P, 0, 1 << 31, by(act(cols=1 << 31)))),
    (MISALIGNED, lambda: (P + 1, 0, 100, by(act()))),
    (MISALIGNED, lambda: (P + 2, 2, 100, by(act()))),
    (MISALIGNED, lambda: (P, 0, 100, by(act(data=P + 8)))),
    (MISALIGNED, lambda: (P, 0, 100, by(act(scale=P + 2)))),
    (0, lambda: (None, 0, 100, by(act(rows=0)))),
    (0, lambda: (None, 0, 0, by(act(cols=0)))),
])
def test_pack_refuses(want, args):
    assert _lib.lib().ark_cuda_act8_pack(*args(), None) == want


@pytest.mark.parametrize("want,args", [
    (INVALID, lambda: (None, P, 0, 100)),
    (INVALID, lambda: (by(act()), None, 0, 100)),
    (INVALID, lambda: (by(act()), P, 4, 100)),
    (INVALID, lambda: (by(act()), P, 0, 99)),
    (INVALID, lambda: (by(act()), P, 0, 0)),                  # an output row may not repeat
    (MISALIGNED, lambda: (by(act()), P + 1, 1, 100)),
    (0, lambda: (by(act(rows=0)), None, 0, 100)),
])
def test_unpack_refuses(want, args):
    assert _lib.lib().ark_cuda_act8_unpack(*args(), None) == want


def wg(x=None, dy=P, t=0, lddy=64, n=64, dw=P, dt=0, lddw=64, ws=None, wsb=0):
    return _lib.lib().ark_cuda_weight_grad(by(act()) if x is None else x, dy, t, lddy, n, dw, dt, lddw,
                                           0, ws, wsb, None)


def test_weight_grad_refuses():
    assert _lib.lib().ark_cuda_weight_grad(None, P, 0, 64, 64, P, 0, 64, 0, None, 0, None) == INVALID
    assert wg(t=2) == UNSUPPORTED                             # FP32 dY
    assert wg(dt=3) == INVALID and wg(dt=-1) == INVALID
    assert wg(lddw=63) == INVALID and wg(lddy=63) == INVALID
    assert wg(dw=None) == INVALID and wg(dy=None) == INVALID
    assert wg(dw=P + 1) == MISALIGNED and wg(dy=P + 1) == MISALIGNED
    assert wg(x=by(act(rows=(1 << 31) - 1))) == INVALID
    assert wg(n=0) == 0 and wg(x=by(act(cols=0))) == 0
    L, a = _lib.lib(), act()
    need = L.ark_cuda_weight_grad_workspace(by(a), P + 2, 64, 63)
    assert need > 0                                           # rows that have to be realigned
    assert wg(dy=P + 2, n=63) == INVALID
    assert wg(dy=P + 2, n=63, ws=P, wsb=need - 1) == INVALID
    assert wg(dy=P + 2, n=63, ws=P + 4, wsb=need) == MISALIGNED
    assert L.ark_cuda_weight_grad_workspace(by(act(rows=0)), P, 64, 64) == 0
    assert L.ark_cuda_weight_grad_workspace(None, P, 64, 64) == 0


def test_swiglu_refuses():
    f, b = _lib.lib().ark_cuda_swiglu, _lib.lib().ark_cuda_swiglu_backward
    ok = (P, 100, P, 100, 0, 64, 100, P, 100)
    assert f(*ok, by(act()), None, None) == INVALID           # one checkpoint of two
    assert f(*ok, by(act()), by(act(kind=1)), None) == INVALID
    assert f(*ok, by(act(rows=63)), by(act(rows=63)), None) == INVALID
    assert f(P, 99, P, 100, 0, 64, 100, P, 100, None, None, None) == INVALID
    assert f(P, 100, P, 100, 0, 64, 100, P, 0, None, None, None) == INVALID
    assert f(P, 100, P, 100, 5, 64, 100, P, 100, None, None, None) == INVALID
    assert f(None, 100, P, 100, 0, 64, 100, P, 100, None, None, None) == INVALID
    assert f(P, 100, P + 1, 100, 0, 64, 100, P, 100, None, None, None) == MISALIGNED
    assert f(None, 100, None, 100, 0, 0, 100, None, 100, None, None, None) == 0
    assert b(P, 100, 0, None, by(act()), P, 100, P, 100, None, None) == INVALID
    assert b(P, 100, 0, by(act()), by(act(cols=99)), P, 100, P, 100, None, None) == INVALID
    assert b(P, 100, 0, by(act()), by(act()), P, 99, P, 100, None, None) == INVALID
    assert b(P, 100, 0, by(act()), by(act()), P, 100, None, 100, None, None) == INVALID
    assert b(P, 100, 0, by(act()), by(act()), P, 100, P, 100, by(act(rows=1)), None) == INVALID


def heads(p=P, h=4, ts=256, hs=64):
    return by(_lib.Heads(p, h, ts, hs))


def plan_struct(rot=64):
    c = _lib.RopePlan()
    assert _lib.lib().ark_cuda_rope_plan(by(c), rot, 0, 10000.0, 0, 1.0, 0.0, 32.0, 1.0) == 0
    return c


def plan(rot=64):
    return by(plan_struct(rot))


def rope(pl=None, q=None, k=None, oq=None, ok=None, t=0, tokens=8, dim=64, pos=None, pt=0, seq=8):
    return _lib.lib().ark_cuda_rope(pl or plan(), q or heads(), k, oq or heads(), ok, t, tokens, dim, pos, pt,
                                    seq, 0, None)


def test_rope_refuses():
    assert _lib.lib().ark_cuda_rope(None, heads(), None, heads(), None, 0, 8, 64, None, 0, 8, 0, None) == INVALID
    assert rope(dim=32) == INVALID                            # shorter than the rotated part
    assert rope(dim=257) == UNSUPPORTED
    assert rope(t=3) == INVALID
    assert rope(k=heads()) == INVALID                         # no output for k
    assert rope(seq=0) == INVALID                             # neither positions nor a length
    assert rope(pos=P, pt=0) == INVALID
    assert rope(pos=P + 4, pt=4) == MISALIGNED and rope(pos=P + 2, pt=3) == MISALIGNED
    assert rope(q=heads(None)) == INVALID and rope(q=heads(P + 1)) == MISALIGNED
    assert rope(oq=heads(h=3)) == INVALID
    assert rope(oq=heads(hs=63)) == INVALID                   # heads of an output overlap
    assert rope(oq=heads(ts=255)) == INVALID
    assert rope(tokens=0) == 0 and rope(q=heads(h=0), oq=heads(h=0)) == 0
    broken = plan_struct()
    for field, value in (("rotary_dim", 63), ("rotary_dim", 0), ("interleaved", 2)):
        c = type(broken).from_buffer_copy(broken)
        setattr(c, field, value)
        assert rope(pl=by(c)) == INVALID


def test_qk_norm_refuses():
    f = _lib.lib().ark_cuda_qk_norm_rope

    def call(gq=P, gk=None, gt=0, eps=1e-6, k=None, ok=None, q8=None, k8=None, q=None, dim=64, pl=None):
        return f(pl or plan(), q or heads(), k, q or heads(), ok, 0, 8, dim, gq, gk, gt, eps, None, 0, 8, q8, k8,
                 None)

    assert call(gq=None) == INVALID and call(gt=4) == INVALID
    assert call(eps=-1.0) == INVALID and call(eps=math.nan) == INVALID
    assert call(gq=P + 1) == MISALIGNED
    assert call(k=heads(), ok=heads(), gk=None) == INVALID
    c = act(8, 256)
    assert call(k8=by(c)) == INVALID
    assert call(q8=by(act(8, 255))) == INVALID and call(q8=by(act(9, 256))) == INVALID
    assert call(k=heads(), ok=heads(), gk=P, q8=by(c)) == INVALID
    assert call(k=heads(), ok=heads(), gk=P, q8=by(c), k8=by(act(8, 256, kind=1))) == INVALID
    # heads apart, and a head that is not made of whole scale blocks
    assert call(q=heads(hs=72, ts=288), dim=40, pl=plan(40), q8=by(act(8, 160))) == UNSUPPORTED
    b = _lib.lib().ark_cuda_qk_norm_rope_backward

    def back(q8=None, q=None, dgq=P, ws=P, wsb=None, k=None, ok=None, k8=None, xk=None, dgk=None, gk=None):
        need = _lib.lib().ark_cuda_qk_norm_rope_workspace(64) if wsb is None else wsb
        return b(plan(), heads(), k, heads(), ok, 0, 8, 64, q8, k8, q, xk, P, gk, 0, 1e-6, None, 0, 8, dgq, dgk, 0, 0,
                 ws, need, None)

    assert back() == INVALID                                  # no x
    assert back(q8=by(c), q=heads()) == INVALID               # two of them
    assert back(q=heads(), dgq=None) == INVALID
    assert back(q=heads(), ws=None) == INVALID and back(q=heads(), wsb=16) == INVALID
    assert back(q=heads(), ws=P + 2) == MISALIGNED
    assert back(q=heads(h=3)) == INVALID
    assert back(q8=by(c), k=heads(), ok=heads(), xk=heads(), gk=P, dgk=P) == INVALID


# ----------------------------------------------------------------- the Python mirror's refusals
def test_host_tensors_and_types_are_refused():
    x = torch.zeros(4, 64, dtype=torch.float16)
    c = None
    for call in (lambda: ab.act8_pack(x), lambda: ab.swiglu(x, x),
                 lambda: ab.rope(x.view(4, 1, 64), None, ab.RopePlan(64)),
                 lambda: ab.qk_norm_rope(x.view(4, 1, 64), None, x[0], None, ab.RopePlan(64)),
                 lambda: ab.Act8(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: ab.act8_pack(x.double()), lambda: ab.act8_pack([1.0]), lambda: ab.act8_unpack(c),
                 lambda: ab.weight_grad(x, x), lambda: ab.Act8(x, x, 64),
                 lambda: ab.swiglu(x.int(), x.int())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="kind"):
        ab.Act8(None, None, 64, "fp4")
    with pytest.raises(ValueError, match="kind"):
        ab.Act8.empty(4, 64, "fp4")


def test_grad_view_needs_the_buffer():
    opt = object.__new__(ab.Optimizer)
    with pytest.raises(RuntimeError, match="grad_buffer"):
        opt.grad_view("embed")
    from ark_b200 import layout
    opt.layout = layout.decoder_layout("tiny", 1, 8, 16, 32)
    opt._gbuf = torch.zeros(opt.layout.n)
    opt._h = None
    assert opt.grad_view("l0.w1", 8, 16).shape == (8, 16) and opt.grad_view("l0.g1").shape == (8,)
    opt.grad_view("l0.w2", 16, 8)[:] = 1
    lo = opt.layout.offsets["l0.w2"]
    assert opt._gbuf[lo: lo + 128].all() and opt._gbuf.sum() == 128
    with pytest.raises(ValueError):
        opt.grad_view("l0.w1", 8, 8)
    with pytest.raises(KeyError):
        opt.grad_view("l1.w1")


# ----------------------------------------------------------------- plans
@pytest.mark.parametrize("kw", [dict(), dict(base=500000.0), dict(scaling="linear", factor=4.0),
                                dict(scaling="base", factor=8.0), dict(scaling="parts", factor=16.0, original=4096),
                                dict(scaling="parts", factor=2.0, original=40, fast=4.0, slow=1.0),
                                dict(scaling="wave", factor=8.0, original=8192, fast=4.0, slow=1.0)])
@pytest.mark.parametrize("rot", [4, 32, 100, 128, 256])
def test_plan_frequencies(rot, kw):
    p = ab.RopePlan(rot, **kw)
    freq, gain = ref.frequencies(rot, **{"fast": 32.0, **kw})
    # whole 2^-64 of a turn: 2 pi 2^-64 = 3.41e-19; pow and the divisions are off by a few 2^-53
    for got, want in zip(p.frequencies(), freq.tolist()):
        assert abs(got - want) <= 3.42e-19 + 16 * 2.0 ** -53 * want
    assert abs(p.gain - gain) <= 2.0 ** -24 * gain


@pytest.mark.parametrize("bad", [dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=258), dict(layout="x"),
                                 dict(scaling="x"), dict(base=1.0), dict(base=math.inf), dict(scaling="linear", factor=0.5),
                                 dict(scaling="linear", factor=math.nan), dict(scaling="parts", factor=2.0),
                                 dict(scaling="wave", factor=2.0, original=100, fast=1.0, slow=1.0),
                                 dict(rotary_dim=2, scaling="base", factor=2.0)])
def test_plan_refuses(bad):
    with pytest.raises((ValueError, ab.ArkError)):
        ab.RopePlan(**{"rotary_dim": 64, **bad})


# ----------------------------------------------------------------- formulas against differences
def test_swiglu_slope_is_the_derivative():
    a, h = torch.linspace(-30, 30, 601, dtype=torch.float64), 1e-5
    f = lambda x: ref.silu_parts(x)[1]  # noqa: E731
    # central differences: h^2 / 6 times the third derivative (below 1), and 2^-53 |f| / h
    assert torch.allclose(ref.silu_parts(a)[2], (f(a + h) - f(a - h)) / (2 * h), rtol=0, atol=1e-9)


@pytest.mark.parametrize("layout,rot", [("half", 8), ("interleaved", 8), ("half", 4), ("interleaved", 2)])
def test_norm_rotation_backward_is_the_derivative(layout, rot):
    g = torch.Generator().manual_seed(1)
    tokens, heads_, dim, eps, h = 3, 2, 8, 1e-2, 1e-6
    x, w, gain = (torch.randn(*s, generator=g, dtype=torch.float64)
                  for s in ((tokens, heads_, dim), (tokens, heads_, dim), (dim,)))
    pos = torch.tensor([0, 7, -1])
    freq, scale = ref.frequencies(rot, scaling="parts", factor=4.0, original=32, fast=4.0, slow=1.0)

    def loss(x, gain):
        return (w * ref.rotate(ref.norm(x, gain, eps), pos, freq, scale, layout)).sum()

    dx, dg, _, _ = ref.norm_back(x, ref.rotate(w, pos, freq, scale, layout, True), gain, eps, pos >= 0)
    for t, grad in ((x, dx), (gain, dg)):
        flat = t.view(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss(x, gain)
            flat[i] = keep - h
            down = loss(x, gain)
            flat[i] = keep
            assert abs((up - down) / (2 * h) - grad.reshape(-1)[i]) < 1e-7
