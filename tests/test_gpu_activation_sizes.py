"""Every way through the weight gradient, and sizes at which a thread of the
other kernels comes round again."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab
from test_gpu_activations import close, near_exp, rot_slack, small_end

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def way(c, dy):
    """(pairs of CTAs?, runs of tokens that are split) from the workspace that the call asks for: X
    in 16 bits and, of split tokens, FP32 sums; dY again where its rows do not start on 16 bytes."""
    import ctypes

    from ark_b200 import _lib
    x = _lib.Act8(c.data.data_ptr(), c.scale.data_ptr(), c.rows, c.cols, 0, 0)
    n = dy.shape[1]
    need = _lib.lib().ark_cuda_weight_grad_workspace(ctypes.byref(x), dy.data_ptr(), dy.stride(0), n)
    if dy.data_ptr() % 16 or dy.stride(0) % 8:
        need -= c.rows * (-(-n // 8) * 8) * 2
    if not need:
        return False, 1
    sums = need - c.rows * c.pitch * 2
    run = c.cols * (-(-n // 4) * 4) * 4
    assert sums >= 0 and sums % run == 0
    return True, max(1, sums // run)


def whole(tokens, nin, nout, dtype, seed):
    """As in the weight gradient's own tests: every sum is a whole number below 15 * 8 * tokens < 2^24,
    exact in FP32 in any order and however it is cut off."""
    assert 120 * tokens < 1 << 24
    g = gen(seed)
    x = torch.randint(-15, 16, (tokens, nin), generator=g, device="cuda").to(dtype)
    return x, torch.randint(-8, 9, (tokens, nout), generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("name,tokens,nin,nout,pairs,split", [
    ("few tiles, one accumulator", 500, 700, 700, False, False),
    ("few tiles, two accumulators", 2048, 768, 2048, False, False),
    ("few tiles, several accumulators of clusters", 8000, 1000, 1001, False, False),
    ("pairs, one run where FP32 has several", 4200, 2048, 5504, True, False),
    ("pairs, rows of any boundary", 4096, 2048, 5501, True, False),
    ("pairs, dY realigned, an odd height", 2100, 2049, 5503, True, False),
    ("pairs, runs of FP16", 8200, 2048, 2301, True, False),
    ("pairs, runs of BF16", 66000, 2048, 2301, True, False),
    ("split tokens", 8192, 768, 2048, True, True),
    ("split tokens, columns not in fours", 8192, 770, 2046, True, True),
    ("split tokens, runs in each", 130000, 500, 510, True, True),
])
@pytest.mark.parametrize("dtype,kind", [(F16, "e4m3"), (BF16, "int8")])
def test_every_way_of_the_weight_gradient(name, tokens, nin, nout, pairs, split, dtype, kind):
    x, dy = whole(tokens, nin, nout, dtype, tokens + nout)
    c = ab.act8_pack(x, kind)
    got = way(c, dy)
    assert got[0] is pairs and (got[1] > 1) is split
    want = x.double().T @ dy.double()
    assert torch.equal(ab.weight_grad(c, dy, dtype=F32).double(), want)
    assert torch.equal(ab.weight_grad(c, dy), want.to(dtype))
    # added to what is there, between guards, on rows of any boundary
    for out in (F32, dtype):
        big = torch.full((nin + 2, nout + 3), 5.0, device="cuda", dtype=out)
        for lo in (0, 1):                 # whole vectors only where nout + 3 allows
            view = big[1: nin + 1, lo: lo + nout]
            view.copy_(torch.arange(nout, device="cuda") % 7)
            ab.weight_grad(c, dy, out=view, accumulate=True)
            assert torch.equal(view, (want + torch.arange(nout, device="cuda") % 7).to(out))
            view.fill_(5)
            assert (big == 5).all()
        whole_rows = torch.full((nin + 1, -(-nout // 8) * 8), 2.0, device="cuda", dtype=out)
        view = whole_rows[:nin, :nout]
        ab.weight_grad(c, dy, out=view, accumulate=True)
        assert torch.equal(view, (want + 2).to(out))
        view.fill_(2)
        assert (whole_rows == 2).all()


@pytest.mark.parametrize("tokens,nin,nout", [(4000, 768, 300), (8000, 1000, 1001), (4096, 2048, 5501), (8192, 768, 2048)])
@pytest.mark.parametrize("dtype,kind", [(F16, "int8"), (BF16, "e4m3")])
def test_no_token_is_lost(tokens, nin, nout, dtype, kind):
    """Terms of one size and sign: a token is 1 / tokens of the sum.  What is cut off is at most 128
    (FP32) or 512 times 2^-23 of it, and the additions of a few partial sums 2^-24 each."""
    g = gen(tokens)
    x = (1 + torch.rand(tokens, nin, generator=g, device="cuda")).to(dtype)
    dy = (2.0 ** -10 * (1 + torch.rand(tokens, nout, generator=g, device="cuda"))).to(dtype)
    c = ab.act8_pack(x, kind)
    want = ab.act8_unpack(c, F32).double().T @ dy.double()
    for out, cut in ((F32, 128), (dtype, 512)):
        off = (ab.weight_grad(c, dy, dtype=out).double() - want).abs()
        tol = want * (ref.HALF[out] + cut * 2.0 ** -23 + 24 * 2.0 ** -24)
        assert (off <= tol).all()
        if out == F32:
            assert tol.max() / want.max() < 0.5 / tokens     # half a token shows


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,cols", [(5200, 1111), (700, 9001), (60000, 96)])
def test_checkpoints_and_swiglu_of_many_elements(rows, cols, dtype):
    """More than the 148 * 8 * 256 threads of a launch have in one round (16 columns each)."""
    kind = "int8" if dtype == F16 else "e4m3"
    g = torch.Generator().manual_seed(rows)
    a, b, dy = ((torch.randn(rows, cols, generator=g) * 2).to(dtype) for _ in range(3))
    y, ca, cb = ab.swiglu(a.cuda(), b.cuda(), checkpoint=kind)
    c = ab.act8_pack(a.cuda(), kind)
    data, scale = ref.pack(a, kind)
    assert torch.equal(c.data.cpu(), data) and torch.equal(c.scale.cpu(), scale)
    assert torch.equal(ca.data, c.data) and torch.equal(ca.scale, c.scale)
    A8 = ref.values(data, scale, cols, kind)
    assert torch.equal(ab.act8_unpack(c, dtype).cpu(), A8.to(dtype))
    A, B, G = a.double(), b.double(), dy.double()
    want = ref.silu_parts(A)[1] * B
    close(y, want, want.abs() * (near_exp(A) + 2 ** -23) + small_end(A, B))
    da, db, _ = ab.swiglu_backward(dy.cuda(), ca, cb, checkpoint=kind)
    B8 = ab.act8_unpack(cb, F32).cpu().double()
    s, t, _ = ref.silu_parts(A8)
    close(db, G * t, (G * t).abs() * (near_exp(A8) + 2 ** -23) + small_end(A8, G))
    size = (G * B8).abs() * s * (1 + A8.abs())
    slope = s * (1 + A8 * (1 - s))
    close(da, G * B8 * slope, size * (near_exp(A8) + 2 ** -21) + small_end(A8, G * B8))


@pytest.mark.parametrize("tokens,hq,hk,dim,layout", [(40000, 2, 1, 64, "half"), (30011, 3, 1, 128, "interleaved"), (25000, 1, 1, 40, "half")])
def test_heads_of_many_tokens(tokens, hq, hk, dim, layout):
    """More tokens than the groups of a launch take at once."""
    g, eps = torch.Generator().manual_seed(tokens), 1e-5
    q, k, dq, dk = (torch.randn(tokens, h, dim, generator=g).half() for h in (hq, hk, hq, hk))
    gq, gk = (1 + 0.2 * torch.randn(dim, generator=g) for _ in range(2))
    pos = torch.arange(tokens) % 5000
    pos[7::11] = -1
    live = pos >= 0
    plan = ab.RopePlan(dim, layout=layout)
    freq, gain = ref.frequencies(dim)
    cu = [t.cuda() for t in (q, k, gq, gk)]
    y = ab.qk_norm_rope(*cu, plan, pos.cuda(), eps=eps, checkpoint="int8")
    back = ab.qk_norm_rope_backward(dq.cuda(), dk.cuda(), y[2], y[3], *cu[2:], plan, pos.cuda(), eps=eps)
    rel = (dim / 2 + 8) * 2.0 ** -24
    for i, (x, d, gn) in enumerate(((q, dq, gq), (k, dk, gk))):
        n = ref.norm(x.double(), gn.double(), eps)
        close(y[i], ref.rotate(n, pos, freq, gain, layout), rot_slack(n, freq, pos) + n.abs().amax(-1, keepdim=True) * 2 * rel)
        X = ref.values(y[2 + i].data, y[2 + i].scale, x[0].numel(), "int8").view_as(x)
        assert (X - x.double())[live].abs().max() <= x.abs().max() / 127 * 1.01    # a scale is below 2 max / 127
        u = ref.rotate(d.double(), pos, freq, gain, layout, True)
        slack_u = rot_slack(d.double(), freq, pos)
        dx, dg, size, gsize = ref.norm_back(X, u, gn.double(), eps, live)
        r = torch.rsqrt((X * X).mean(-1, keepdim=True) + eps)
        h = (X * r).abs().amax(-1, keepdim=True)
        close(back[i], dx, (size.amax(-1, keepdim=True) * 2 * (dim + 24) * 2.0 ** -24
                            + slack_u * gn.abs().max() * r * (1 + h * h)) * live.view(-1, 1, 1))
        # a lane adds its tokens one by one (their number divided by a launch's groups, at most
        # tokens / 592 + heads), the lanes and blocks follow: far fewer than tokens / 8 additions
        slack_g = gsize * (tokens / 8 + dim + 24) * 2.0 ** -24 + (slack_u * (X * r).abs() * live.view(-1, 1, 1)).sum((0, 1))
        close(back[2 + i], dg, slack_g)
