"""The FP32 forms are as exact as FP32 operations make them."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F32 = torch.float32
ULP = 2.0 ** -23


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_swiglu(kind):
    """exp is off by 1 ulp, 1 + exp by 1/2, its reciprocal by 1 and their product by 1/2: s by 3 and
    a s b by 4 ulps of 2^-23, whatever the size of a.  Below a = -87 s is among the subnormals, where
    exp, s and a s are each off by 2^-150, which the factors a and b then multiply."""
    g = torch.Generator().manual_seed(1)
    a = torch.cat([torch.linspace(-100, 40, 4096), 3 * torch.randn(12288, generator=g)]).view(8, 2048)
    b, dy = (torch.randn(8, 2048, generator=g) for _ in range(2))
    tiny = lambda x, f: 2.0 ** -148 * (x.abs() + 1) * (1 + f.abs())  # noqa: E731
    y, ca, cb = ab.swiglu(a.cuda(), b.cuda(), checkpoint=kind)
    A, B, G = a.double(), b.double(), dy.double()
    want = ref.silu_parts(A)[1] * B
    assert ((y.cpu().double() - want).abs() <= 4 * ULP * want.abs() + tiny(A, B)).all()
    da, db = ab.swiglu_backward(dy.cuda(), ca, cb)
    A, B = ref.through(a, kind), ref.through(b, kind)
    s, t, slope = ref.silu_parts(A)
    assert ((db.cpu().double() - G * t).abs() <= 4 * ULP * (G * t).abs() + tiny(A, G)).all()
    # slope = s (1 + a (1 - s)): s, the products and the sum by 5 ulps of the result, and the term
    # a (1 - s) by 3 of its own size
    size = (G * B).abs() * s * (5 * (1 + A * (1 - s)).abs() + 3 * (A * (1 - s)).abs())
    assert ((da.cpu().double() - G * B * slope).abs() <= ULP * size + tiny(A, G * B)).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles_near_quarter_turns(layout):
    """Pairs (1, 0) rotate into (cos, sin).  sincospi is off by 2 ulps, a turn by its 2^-32 (its
    lower bits are cut) and by a position's 2^-64 of a turn; small cosines and sines show it."""
    rot = 64
    plan = ab.RopePlan(rot, layout=layout, base=10000.0)
    freq, _ = ref.frequencies(rot)
    pos = torch.arange(0, 1 << 22, 37)
    q = torch.zeros(pos.numel(), 1, rot)
    i1, i2 = (slice(0, 32), slice(32, 64)) if layout == "half" else (slice(0, 64, 2), slice(1, 64, 2))
    q[..., i1] = 1
    y = ab.rope(q.cuda(), None, plan, pos.cuda())[0].cpu().double()[:, 0]
    angle = pos.double().view(-1, 1) * freq
    # in 64 bits the angle is off by 2^-53 of itself, and the plan by 3.41e-19 a position
    slack = 2 * 3.1416 * 2.0 ** -32 + angle * 2.0 ** -52 + pos.double().view(-1, 1) * 3.42e-19
    for got, want in ((y[:, i1], torch.cos(angle)), (y[:, i2], torch.sin(angle))):
        # two roundings after sincospi's: the turn on, and the product with 1
        assert ((got - want).abs() <= (2 * ULP + 2 * 2.0 ** -24) * want.abs() + slack).all()
