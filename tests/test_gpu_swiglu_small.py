"""The remade SwiGLU product where it is among FP16's subnormals."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def test_products_next_to_borders_of_subnormals():
    """Every a of 7 bits and every b of 7 bits, over the sizes that leave silu(a) b below 2^-14,
    where FP16's borders are odd multiples of 2^-25.  A product as near to one as FP32 is off is
    made in 64 bits, rounded to FP32, to FP16, and into 8 bits, where one step more or less shows."""
    c = torch.arange(64, 128).double()
    a = torch.cat([c * 2.0 ** e for e in range(-14, -1)])            # 2^-8 to 32
    a = torch.cat([a, -a]).view(-1, 1)
    b = torch.cat([c * 2.0 ** e for e in range(-24, 9)]).view(1, -1)
    a, b = (t.expand(a.shape[0], b.shape[1]).half() for t in (a, b))
    ca, cb = ab.act8_pack(a.cuda(), "int8"), ab.act8_pack(b.cuda(), "int8")
    A, B = a.double(), b.double()
    assert torch.equal(ref.through(a[:, :64], "int8"), A[:, :64]) and torch.equal(ref.through(b[:2], "int8"), B[:2])
    exact = A / (1 + torch.exp(-A)) * B
    y = exact.float().half()
    # as near as FP32 is off: 4 steps, and 2.4 |a| more for a negative a
    steps = exact.abs() * 2.0 ** 24
    ulps = 4 + 2.4 * (-A).clamp(min=0)
    near = ((steps - steps.floor() - 0.5).abs() < steps * ulps * 2.0 ** -24) & (steps < 1024)
    assert near.sum() > 100
    _, _, cy = ab.swiglu_backward(torch.ones_like(a, device="cuda"), ca, cb, checkpoint="int8")
    data, scale = ref.pack(y, "int8")
    assert torch.equal(cy.scale.cpu(), scale)
    got, want = ab.act8_unpack(cy, F32).cpu().double(), ref.values(data, scale, a.shape[1], "int8")
    bad = (got != want) & ~(got.isnan() & want.isnan())              # blocks beyond FP16 are NaN
    assert not bad.any(), (bad.sum().item(), steps[bad][:4].tolist())
