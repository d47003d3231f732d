"""The weight gradient from 8-bit checkpoints against 64-bit sums."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def integers(tokens, nin, nout, kind, dtype, seed):
    """X whose checkpoint is X itself and small whole dY: every product and partial sum is a
    whole number below 2^24 (15 * 8 * 8192 tokens < 2^20), so FP32 sums in any order are exact."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-15, 16, (tokens, nin), generator=g).to(dtype)
    dy = torch.randint(-8, 9, (tokens, nout), generator=g).to(dtype)
    return x, dy


SHAPES = [(1, 1, 1), (1, 128, 128), (63, 128, 64), (64, 64, 256), (65, 129, 257), (130, 768, 768), (300, 96, 2048),
          (1000, 33, 40), (1024, 256, 8), (2049, 200, 100), (77, 1300, 5000), (513, 2048, 4800)]


@pytest.mark.parametrize("kind,dtype", [("e4m3", F16), ("int8", BF16), ("int8", F16), ("e4m3", BF16)])
@pytest.mark.parametrize("tokens,nin,nout", SHAPES)
def test_integer_sums_are_exact(tokens, nin, nout, kind, dtype):
    x, dy = integers(tokens, nin, nout, kind, dtype, tokens + nin)
    c = ab.act8_pack(x.cuda(), kind)
    want = (x.double().T @ dy.double())
    got = ab.weight_grad(c, dy.cuda(), dtype=F32)
    assert torch.equal(got.cpu().double(), want)
    assert torch.equal(ab.weight_grad(c, dy.cuda()).cpu(), want.to(dtype))
    acc = got.clone()
    ab.weight_grad(c, dy.cuda(), out=acc, accumulate=True)
    assert torch.equal(acc.cpu().double(), 2 * want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,nin,nout", [(500, 130, 264), (4000, 768, 300)])
def test_random(tokens, nin, nout, dtype, kind):
    g = torch.Generator().manual_seed(tokens)
    x = (torch.randn(tokens, nin, generator=g) * torch.exp2(torch.randint(-8, 8, (1, nin), generator=g).float())).to(dtype)
    dy = torch.randn(tokens, nout, generator=g).to(dtype)
    c = ab.act8_pack(x.cuda(), kind)
    X, D = ref.through(x, kind), dy.double()
    want, size = X.T @ D, X.abs().T @ D.abs()
    # products are exact in FP32 (8 + 11 significant bits); each of `tokens` additions is off
    # by at most one step, 2^-23 of what is summed so far
    for out in (F32, dtype):
        got = ab.weight_grad(c, dy.cuda(), dtype=out).cpu().double()
        tol = ref.HALF[out] * want.abs() + ref.TINY[out] + size * tokens * 2.0 ** -23
        assert ((got - want).abs() <= tol).all()
    assert torch.equal(ab.weight_grad(c, dy.cuda()), ab.weight_grad(c, dy.cuda()))


def test_scales_of_all_sizes_become_operands():
    """Every scale that FP16 activations give, down to subnormals and up to the largest."""
    for kind in ("e4m3", "int8"):
        x = torch.zeros(40, 40 * 32, dtype=F16)
        for i in range(40):
            x[i, 32 * i: 32 * i + 8] = torch.tensor([1, -1, 0.5, 0.75, 0.25, -0.875, 0.125, 0.9375]) * 2.0 ** (i - 24)
        x[39, 39 * 32] = 65504
        c = ab.act8_pack(x.cuda(), kind)
        eye = torch.eye(40, dtype=F16)
        got = ab.weight_grad(c, eye.cuda(), dtype=F32).cpu()
        want = ref.through(x, kind).clamp(-65504, 65504).to(F16)   # the operand is FP16
        assert torch.equal(got.T, want.float())


def test_strides_offsets_and_what_is_outside():
    for nout, off, extra in ((96, 0, 0), (96, 8, 16), (96, 1, 0), (95, 0, 1), (97, 3, 0), (256, 0, 8)):
        x, buf = integers(150, 200, nout + off + extra, "int8", F16, nout + off)
        dy = buf.cuda()[:, off: off + nout]
        c = ab.act8_pack(x.cuda(), "int8")
        want = x.double().T @ buf[:, off: off + nout].double()
        big = torch.full((202, nout + 5), 3.0, device="cuda", dtype=F16)
        ab.weight_grad(c, dy, out=big[1:201, 2: 2 + nout])
        assert torch.equal(big[1:201, 2: 2 + nout].cpu(), want.half())
        big[1:201, 2: 2 + nout] = 3
        assert (big == 3).all()
    x, dy = integers(150, 64, 64, "int8", F16, 1)
    row = dy[:1].cuda().expand(150, 64)                                # one gradient for all tokens
    got = ab.weight_grad(ab.act8_pack(x.cuda(), "int8"), row, dtype=F32)
    assert torch.equal(got.cpu().double(), x.double().T @ row.cpu().double())


def test_no_tokens_and_no_features():
    c = ab.act8_pack(torch.empty(0, 70, dtype=F16, device="cuda"))
    dy = torch.empty(0, 50, dtype=F16, device="cuda")
    assert (ab.weight_grad(c, dy, out=torch.ones(70, 50, device="cuda")) == 0).all()
    assert (ab.weight_grad(c, dy, out=torch.ones(70, 50, device="cuda"), accumulate=True) == 1).all()
    assert ab.weight_grad(ab.act8_pack(torch.empty(4, 0, dtype=F16, device="cuda")), torch.ones(4, 8, dtype=F16, device="cuda")).shape == (0, 8)


def test_nonfinite_and_overflow_reach_the_gradient():
    x = torch.ones(70, 64, dtype=F16)
    x[3, 40] = float("inf")
    dy = torch.ones(70, 24, dtype=F16)
    w = ab.weight_grad(ab.act8_pack(x.cuda(), "int8"), dy.cuda()).cpu()
    assert torch.isnan(w[32:]).all() and (w[:32] == 70).all()
    w = ab.weight_grad(ab.act8_pack(torch.full((70, 64), 1000.0, dtype=F16, device="cuda")), dy.cuda() * 10)
    assert torch.isinf(w).all()
