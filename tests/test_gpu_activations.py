"""The activation operators on the GPU against their definitions in 64 bits.

Bounds count roundings: half a step of the output's type, plus the FP32
operations between (2^-24 each, CUDA's documented ulps for exp, rsqrt and
sincospi), relative to the sizes of the terms that are added.  Packing,
and sums of integers, have to be equal bit for bit.
"""
import numpy as np
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [F16, BF16, F32]


def rng(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, slack, dtype=None):
    """|got - want| <= half a step of the type + slack, everywhere; NaN only where wanted."""
    got, want = got.detach().cpu(), want.double()
    t = dtype or got.dtype
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs()
    tol = ref.HALF[t] * want.abs() + ref.TINY[t] + slack
    bad = ~(off <= tol) & ~torch.isnan(want)
    assert not bad.any(), (off[bad][:4], tol[bad][:4] if tol.dim() else tol, bad.nonzero()[:4])


# ----------------------------------------------------------------- checkpoints
def hard_values(rows, cols, dtype, seed):
    """Sizes from one end of the type to the other, exact ties, zeros, whole empty blocks."""
    g = rng(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    span = {F16: 12, BF16: 60, F32: 60}[dtype]
    x *= torch.exp2(torch.randint(-span, span, (rows, 1), generator=g).double())
    ties = torch.randint(-255, 256, (rows, cols), generator=g).double() / 2
    x = torch.where(torch.rand(rows, 1, generator=g) < 0.3, ties, x)
    x = torch.where(torch.rand(rows, cols, generator=g) < 0.1, torch.zeros_like(x), x)
    x = x.to(dtype)
    if rows > 3:
        x[1, : min(32, cols)] = 0
        x[2, 0] = torch.finfo(dtype).max
        x[3, -1] = torch.finfo(dtype).smallest_normal / 2
    return x


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (64, 128), (7, 129), (33, 768),
                                       (2, 2049), (700, 96)])
def test_pack_and_unpack(rows, cols, dtype, kind):
    x = hard_values(rows, cols, dtype, rows * 1000 + cols)
    c = ab.act8_pack(x.cuda(), kind)
    data, scale = ref.pack(x, kind)
    assert torch.equal(c.scale.cpu(), scale)
    assert torch.equal(c.data.cpu(), data)
    want = ref.values(data, scale, cols, kind)
    for out in TYPES:
        y = ab.act8_unpack(c, out).cpu()
        top = torch.finfo(out).max
        assert torch.equal(y, want.clamp(-top, top).to(out))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", TYPES)
def test_pack_nonfinite_blocks_read_as_nan(dtype, kind):
    x = torch.ones(4, 100)
    x[0, 3], x[1, 40], x[2, 99] = float("inf"), float("nan"), -float("inf")
    c = ab.act8_pack(x.to(dtype).cuda(), kind)
    y = ab.act8_unpack(c, F32).cpu()
    want = torch.ones(4, 100)
    want[0, :32] = want[1, 32:64] = want[2, 96:] = float("nan")
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_pack_strided_rows_and_offsets(dtype):
    base = hard_values(40, 300, dtype, 9).cuda()
    for x in (base[:, :128], base[:, 1:130], base[::3, 8:264], base[5:6].expand(7, 300)):
        c = ab.act8_pack(x, "int8")
        data, scale = ref.pack(x.cpu(), "int8")
        assert torch.equal(c.data.cpu(), data) and torch.equal(c.scale.cpu(), scale)
    keep = torch.full((40, 300), 7.0, dtype=dtype, device="cuda")
    ab.act8_unpack(ab.act8_pack(base[:, :129], "e4m3"), out=keep[:, 5:134])
    assert torch.equal(keep[:, 5:134].cpu().double(),
                       ref.through(base[:, :129].cpu(), "e4m3").clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype).double())
    assert (keep[:, :5] == 7).all() and (keep[:, 134:] == 7).all()


def test_pack_empty():
    for shape in ((0, 64), (5, 0)):
        c = ab.act8_pack(torch.empty(shape, dtype=F16, device="cuda"))
        assert ab.act8_unpack(c).shape == shape


# ----------------------------------------------------------------- SwiGLU
def near_exp(a):
    """Relative error of s = 1 / (1 + exp(-a)) in FP32: exp is off by 2 + 1.173 |a|
    ulps, which the sum passes on times (1 - s) <= 1, the division by 2, the sum by 1/2."""
    return (5 + 1.2 * a.abs()) * 2.0 ** -23


def small_end(a, factor):
    """For a below -87 s is among the subnormals, where exp(a), s and a * s are each rounded
    to a multiple of 2^-149, that is by 2^-150 whatever their size: s is then off by 2^-149,
    a * s by 2^-149 |a| + 2^-150, and the product with a factor f by (2^-149 (|a| + 1)) |f|,
    which for a sum of two such terms in the slope doubles."""
    return 2.0 ** -148 * (a.abs() + 1) * (1 + factor.abs())


SWIGLU_SHAPES = [(1, 1), (1, 2048), (3, 33), (17, 96), (64, 768), (5, 1025)]


def swiglu_inputs(rows, cols, dtype, seed):
    g = rng(seed)
    a = 4 * torch.randn(rows, cols, generator=g)
    a = torch.where(torch.rand(rows, cols, generator=g) < 0.05, 30 * a, a)
    return [t.to(dtype) for t in (a, torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g))]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SWIGLU_SHAPES)
def test_swiglu(rows, cols, dtype, kind):
    a, b, dy = swiglu_inputs(rows, cols, dtype, rows + cols)
    y, ca, cb = ab.swiglu(a.cuda(), b.cuda(), checkpoint=kind)
    assert torch.equal(ab.swiglu(a.cuda(), b.cuda()), y)
    A, B, G = a.double(), b.double(), dy.double()
    want = ref.silu_parts(A)[1] * B
    close(y, want, want.abs() * (near_exp(A) + 2 ** -23) + small_end(A, B))
    for c, x in ((ca, a), (cb, b)):
        data, scale = ref.pack(x, kind)
        assert torch.equal(c.data.cpu(), data) and torch.equal(c.scale.cpu(), scale)
    da, db = ab.swiglu_backward(dy.cuda(), ca, cb)
    A, B = ref.through(a, kind), ref.through(b, kind)
    s, t, slope = ref.silu_parts(A)
    close(db, G * t, (G * t).abs() * (near_exp(A) + 2 ** -23) + small_end(A, G))
    # slope = s (1 + a (1 - s)): the terms' sizes, not their sum, carry the error; 1 - s is
    # off by 2^-24 and by the error of s
    size = (G * B).abs() * s * (1 + A.abs() * (1 - s + s * near_exp(A) + 2 ** -23))
    loss = (G * B).abs() * s * A.abs() * (s * near_exp(A) + 2 ** -23)
    close(da, G * B * slope, size * (near_exp(A) + 2 ** -21) + loss + small_end(A, G * B))
    da2, db2, cy = ab.swiglu_backward(dy.cuda(), ca, cb, checkpoint=kind)
    assert torch.equal(da, da2) and torch.equal(db, db2)
    # the remade product is rounded to the type, then packed: one step of the type may
    # move it over a border of the 8-bit grid, that is by one step of the grid
    got = ab.act8_unpack(cy, F32).cpu().double()
    Y = (t * B).to(dtype)
    want = ref.through(Y, kind)
    step = torch.exp2(ref.pack(Y, kind)[1].double() - 127).repeat_interleave(32, 1)[:, :cols]
    grid = step if kind == "int8" else torch.maximum(want.abs() / 8, step * 2.0 ** -9)
    assert ((got - want).abs() <= 2 * grid).all()   # a block's scale may move with its largest
    assert (got != want).double().mean() < 0.01 or got.numel() < 1000


def test_swiglu_in_place_and_fused_buffer():
    ab_, dy = torch.randn(50, 2 * 136).half().cuda(), torch.randn(50, 136).half().cuda()
    a, b = ab_[:, :136], ab_[:, 136:]
    y, ca, cb = ab.swiglu(a, b, checkpoint="int8")
    da, db = ab.swiglu_backward(dy, ca, cb)
    g = torch.zeros(50, 2 * 136, dtype=F16, device="cuda")
    ab.swiglu_backward(dy, ca, cb, out=(g[:, :136], g[:, 136:]))
    assert torch.equal(g, torch.cat([da, db], 1))
    d2 = dy.clone()
    ab.swiglu_backward(d2, ca, cb, out=(d2, g[:, 136:]))
    assert torch.equal(d2, da)
    a2 = a.clone()
    assert ab.swiglu(a2, b, out=a2) is a2 and torch.equal(a2, y)


def test_swiglu_nonfinite_reaches_the_gradients():
    a, b = torch.ones(2, 64, dtype=F16), torch.ones(2, 64, dtype=F16)
    a[0, 5] = float("inf")
    y, ca, cb = ab.swiglu(a.cuda(), b.cuda(), checkpoint="e4m3")
    da, db = ab.swiglu_backward(torch.ones(2, 64, dtype=F16, device="cuda"), ca, cb)
    assert torch.isnan(da[0, :32]).all() and torch.isnan(db[0, :32]).all()
    assert torch.isfinite(da[0, 32:]).all() and torch.isfinite(da[1]).all()


# ----------------------------------------------------------------- rotation
SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
            dict(scaling="parts", factor=16.0, original=4096), dict(scaling="wave", factor=8.0, original=8192, fast=4.0)]


def rot_slack(x, freq, pos):
    """Four FP32 roundings and sincospi's 2 ulps on each product, and the angle's 2^-32 of
    a turn, relative to the pair; 64-bit angles themselves are off by pos * 2^-53."""
    size = x.abs().amax(-1, keepdim=True) * 2
    return size * (8 * 2.0 ** -24 + 2e-9 + pos.abs().double().view(-1, 1, 1) * 2.0 ** -52) * 1.5


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 64), (96, 32), (80, 80), (100, 50), (2, 2), (7, 4),
                                     (256, 256), (255, 254), (72, 8)])
def test_rope(dim, rot, dtype, layout):
    g = rng(dim * 7 + rot)
    tokens, hq, hk = 37, 5, 2
    q, k = torch.randn(tokens, hq, dim, generator=g).to(dtype), torch.randn(tokens, hk, dim, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g)
    pos[0], pos[1], pos[2], pos[3] = 0, 1, -1, (1 << 31) - 1
    for n, sc in enumerate(SCALINGS):
        if sc.get("scaling") == "base" and rot == 2:
            continue
        plan = ab.RopePlan(rot, layout=layout, **sc)
        freq, gain = ref.frequencies(rot, **sc)
        # a plan holds whole 2^-64 of a turn: 2 pi 2^-64 = 3.41e-19 radians per position
        assert np.allclose(plan.frequencies(), freq, rtol=1e-14, atol=3.42e-19) and abs(plan.gain - gain) < 1e-6
        inverse = n % 2 == 1
        p = pos.int() if n % 2 else pos
        yq, yk = ab.rope(q.cuda(), k.cuda(), plan, p.cuda(), inverse=inverse)
        for y, x in ((yq, q), (yk, k)):
            X = x.double()
            close(y, ref.rotate(X, pos, freq, gain, layout, inverse), rot_slack(X, freq, pos) * gain)


def test_rope_inverse_undoes_and_in_place():
    plan = ab.RopePlan(64, layout="interleaved")
    qkv = torch.randn(100, 24, 64, device="cuda")
    q, k = qkv[:, :12], qkv[:, 12:18]
    want = ab.rope(q, k, plan, seq_len=50)
    back = ab.rope(*want, plan, seq_len=50, inverse=True)
    assert torch.allclose(back[0], q, atol=1e-5) and torch.allclose(back[1], k, atol=1e-5)
    pos = (torch.arange(100, device="cuda") % 50)
    assert all(torch.equal(x, y) for x, y in zip(want, ab.rope(q, k, plan, pos)))
    rest = qkv[:, 18:].clone()
    ab.rope(q, k, plan, pos, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 18:], rest)


def test_rope_orders_strides_and_q_alone():
    plan = ab.RopePlan(32)
    x = torch.randn(6, 40, 48, device="cuda", dtype=BF16)          # [heads, tokens, dim]
    want, none = ab.rope(x.transpose(0, 1).contiguous(), None, plan)
    assert none is None
    got, _ = ab.rope(x.transpose(0, 1), None, plan)
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    ab.rope(x.transpose(0, 1), None, plan, out=(out.transpose(0, 1), None))
    assert torch.equal(out.transpose(0, 1), want)
    odd = torch.randn(40, 6 * 48 + 1, device="cuda", dtype=BF16)[:, 1:].view(40, 6, 48)
    assert torch.equal(ab.rope(odd, None, plan)[0], ab.rope(odd.contiguous(), None, plan)[0])
    one = torch.randn(40, 1, 48, device="cuda", dtype=BF16)
    a, b = ab.rope(one.expand(40, 6, 48), one, plan)
    assert torch.equal(a, b.expand(40, 6, 48))


def test_rope_padding_is_not_read():
    plan = ab.RopePlan(16)
    q = torch.randn(9, 3, 16, device="cuda")
    q[4:] = float("nan")
    pos = torch.tensor([3, 2, 1, 0] + [-1] * 5, device="cuda")
    y, _ = ab.rope(q, None, plan, pos)
    assert torch.isfinite(y).all() and (y[4:] == 0).all()


# ----------------------------------------------------------------- norm and rotation
QK = [(64, 64, "half"), (128, 128, "half"), (128, 64, "half"), (32, 32, "interleaved"), (64, 32, "interleaved"),
      (96, 96, "interleaved"), (80, 80, "half"), (100, 50, "half"), (256, 256, "half"), (33, 32, "interleaved"), (2, 2, "half")]


@pytest.mark.parametrize("kind", ["e4m3", "int8", None])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot,layout", QK)
def test_qk_norm_rope(dim, rot, layout, dtype, kind):
    g = rng(dim * 3 + rot)
    tokens, hq, hk, eps = 41, 6, 2, 1e-5
    mk = lambda h: (torch.randn(tokens, h, dim, generator=g) * torch.exp2(torch.randint(-6, 6, (tokens, h, 1), generator=g).float())).to(dtype)  # noqa: E731
    q, k, dq, dk = mk(hq), mk(hk), mk(hq), mk(hk)
    q[5] = 0                                            # a head of zeros: eps alone
    gt = dtype if dim % 3 else F32
    gq, gk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(gt) for _ in range(2))
    pos = torch.arange(tokens)
    pos[7], pos[30:33] = 123456, -1
    plan = ab.RopePlan(rot, layout=layout)
    freq, gain = ref.frequencies(rot)
    cu = lambda *t: [x.cuda() for x in t]  # noqa: E731
    res = ab.qk_norm_rope(*cu(q, k, gq, gk), plan, pos.cuda(), eps=eps, checkpoint=kind)
    live = pos >= 0
    # the mean of dim squares and rsqrt: (dim / 2 + 4) 2^-24 relative to each element
    rel = (dim / 2 + 8) * 2.0 ** -24
    for y, x, gn in ((res[0], q, gq), (res[1], k, gk)):
        n = ref.norm(x.double(), gn.double(), eps)
        close(y, ref.rotate(n, pos, freq, gain, layout), rot_slack(n, freq, pos) + n.abs().amax(-1, keepdim=True) * 2 * rel)
    if kind:
        for c, x in ((res[2], q), (res[3], k)):
            data, scale = ref.pack(x.flatten(1), kind)
            assert torch.equal(c.data.cpu()[live], data[live]) and torch.equal(c.scale.cpu()[live], scale[live])
    src = res[2:] if kind else cu(q, k)
    back = ab.qk_norm_rope_backward(*cu(dq, dk), *src, *cu(gq, gk), plan, pos.cuda(), eps=eps)
    for i, (d, x, gn) in enumerate(((dq, q, gq), (dk, k, gk))):
        X = ref.through(x.flatten(1), kind).view_as(x) if kind else x.double()
        u = ref.rotate(d.double(), pos, freq, gain, layout, True)
        slack_u = rot_slack(d.double(), freq, pos)
        dx, dg, size, gsize = ref.norm_back(X, u, gn.double(), eps, live)
        r = torch.rsqrt((X * X).mean(-1, keepdim=True) + eps)
        G = gn.double().abs().max()
        h = (X * r).abs().amax(-1, keepdim=True)
        close(back[i], dx, (size.amax(-1, keepdim=True) * 2 * (dim + 24) * 2.0 ** -24 + slack_u * G * r * (1 + h * h)) * live.view(-1, 1, 1))
        terms = tokens * d.shape[1]
        slack_g = gsize * (terms + dim + 24) * 2.0 ** -24 + (slack_u * (X * r).abs() * live.view(-1, 1, 1)).sum((0, 1))
        close(back[2 + i], dg, slack_g)


def test_qk_backward_in_place_accumulate_and_order():
    plan = ab.RopePlan(64)
    mk = lambda h: torch.randn(300, h, 64, device="cuda").half()  # noqa: E731
    q, k, dq, dk = mk(8), mk(2), mk(8), mk(2)
    gq, gk = torch.rand(64, device="cuda").half(), torch.rand(64, device="cuda").half()
    _, _, cq, ck = ab.qk_norm_rope(q, k, gq, gk, plan, checkpoint="e4m3")
    args = (cq, ck, gq, gk, plan)
    first = ab.qk_norm_rope_backward(dq, dk, *args)
    again = ab.qk_norm_rope_backward(dq, dk, *args)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    acc = torch.ones(64, device="cuda"), torch.full((64,), 2.0, device="cuda")
    full = ab.qk_norm_rope_backward(dq, dk, *args, out_gains=(torch.empty(64, device="cuda"), torch.empty(64, device="cuda")))
    ab.qk_norm_rope_backward(dq, dk, *args, out_gains=acc, accumulate=True)
    assert torch.equal(acc[0], full[2] + 1) and torch.equal(acc[1], full[3] + 2)
    d1, d2 = dq.clone(), dk.clone()
    ab.qk_norm_rope_backward(d1, d2, *args, out=(d1, d2))
    assert torch.equal(d1, first[0]) and torch.equal(d2, first[1])
    alone = ab.qk_norm_rope_backward(dq, None, cq, None, gq, None, plan)
    assert torch.equal(alone[0], first[0]) and alone[1] is None and alone[3] is None
    # the grid is another one, so the sum's order is: 2400 terms, FP32 tree
    assert torch.allclose(alone[2].float(), first[2].float(), rtol=2 ** -10, atol=1e-3)


def test_qk_no_tokens():
    plan = ab.RopePlan(32)
    e = torch.empty(0, 4, 32, device="cuda", dtype=F16)
    g = torch.ones(32, device="cuda", dtype=F16)
    y = ab.qk_norm_rope(e, e[:, :2], g, g, plan, checkpoint="int8")
    out = ab.qk_norm_rope_backward(e, e[:, :2], y[2], y[3], g, g, plan)
    assert (out[2] == 0).all() and (out[3] == 0).all()
    assert ab.rope(e, None, plan)[0].shape == (0, 4, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,extra,off", [(511, 0, 0), (700, 1, 1), (1000, 3, 2), (129, 0, 3), (513, 2, 5), (2000, 7, 7), (40, 1, 1),
                                            (24, 9, 1), (17, 0, 0), (600, 8, 8), (600, 8, 4)])
def test_rows_on_any_boundary(cols, extra, off, dtype):
    """Rows that start anywhere: every value right, and nothing written beside them."""
    rows, width = 37, cols + extra + off
    g = rng(cols)
    x = torch.randn(rows, width, generator=g).to(dtype).cuda()[:, off: off + cols]
    c = ab.act8_pack(x, "int8")
    data, scale = ref.pack(x.cpu(), "int8")
    assert torch.equal(c.data.cpu(), data) and torch.equal(c.scale.cpu(), scale)
    guard = torch.full((rows + 2, width), 9.0, dtype=dtype, device="cuda")
    out = guard[1: rows + 1, off: off + cols]
    ab.act8_unpack(c, out=out)
    assert torch.equal(out.cpu(), ref.values(data, scale, cols, "int8").to(dtype))
    aligned = [t.contiguous() for t in (x, x.flip(0))]
    y, ca, cb = ab.swiglu(*aligned, checkpoint="int8")
    z = torch.empty(rows, width, dtype=dtype, device="cuda")[:, off: off + cols]
    z.copy_(aligned[1])
    got, da, db = ab.swiglu(x, z, checkpoint="int8", out=out)
    assert torch.equal(out, y) and torch.equal(da.data, ca.data) and torch.equal(db.data, cb.data)
    ga, gb = ab.swiglu_backward(aligned[0], ca, cb)
    ab.swiglu_backward(x, ca, cb, out=(out, z))
    assert torch.equal(out, ga) and torch.equal(z, gb)
    ab.swiglu(x, aligned[1], out=x)                                  # in place
    assert torch.equal(x, y)
    out.fill_(9)
    assert (guard == 9).all()
