"""Calls at the edges of what the activation operators document."""
import pytest
import torch

import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_positions_of_no_tokens(itype):
    """A batch without tokens gives positions without elements."""
    plan, pos = ab.RopePlan(32), torch.empty(0, dtype=itype, device="cuda")
    q, g = torch.empty(0, 4, 32, dtype=F16, device="cuda"), torch.ones(32, dtype=F16, device="cuda")
    assert ab.rope(q, q[:, :2], plan, pos)[1].shape == (0, 2, 32)
    y = ab.qk_norm_rope(q, q[:, :2], g, g, plan, pos, checkpoint="int8")
    assert y[0].shape == q.shape and y[2].rows == 0
    back = ab.qk_norm_rope_backward(q, q[:, :2], y[2], y[3], g, g, plan, pos)
    assert (back[2] == 0).all() and (back[3] == 0).all()


@pytest.mark.parametrize("hq,hk", [(0, 2), (3, 0), (0, 0)])
def test_gains_of_no_heads_have_no_gradient(hq, hk):
    """A sum over no heads is zero, and stays what was there when it is added to."""
    plan, tokens, dim = ab.RopePlan(32), 5, 32
    q, k = (torch.randn(tokens, h, dim, device="cuda").half() for h in (hq, hk))
    g = torch.ones(dim, device="cuda")
    junk = [torch.full((dim,), 7.0, device="cuda") for _ in range(2)]
    kept = [t.clone() for t in junk]
    out = ab.qk_norm_rope_backward(q, k, q, k, g, g, plan, out_gains=tuple(junk))
    ab.qk_norm_rope_backward(q, k, q, k, g, g, plan, out_gains=tuple(kept), accumulate=True)
    for h, got, more in ((hq, out[2], kept[0]), (hk, out[3], kept[1])):
        if h:
            assert torch.equal(more, got + 7) and got.any()
        else:
            assert (got == 0).all() and (more == 7).all()


def test_pack_is_of_the_kind_that_was_asked_for():
    x = torch.randn(4, 64, device="cuda").half()
    room = ab.Act8.empty(4, 64, "int8")
    assert ab.act8_pack(x).kind == "e4m3" and ab.act8_pack(x, "int8").kind == "int8"
    assert ab.act8_pack(x, out=room).kind == "int8" and ab.act8_pack(x, "int8", room).kind == "int8"
    with pytest.raises(ValueError, match="int8"):
        ab.act8_pack(x, "e4m3", out=room)
    with pytest.raises(ValueError, match="kind"):
        ab.act8_pack(x, "int4", out=room)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, F16, torch.bfloat16])
def test_rotation_does_not_depend_on_the_rows_alignment(layout, dtype):
    """Chunks of 1, 2, 4 and 8 elements: the same products, rounded in the same order."""
    plan, g = ab.RopePlan(48, layout=layout), torch.Generator().manual_seed(9)
    x = torch.randn(300, 6, 48, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 100000, (300,), generator=g).cuda()
    for inverse in (False, True):
        want = ab.rope(x, None, plan, pos, inverse=inverse)[0]
        for off in (1, 2, 4):
            odd = torch.empty(300, 6 * 48 + off, dtype=dtype, device="cuda")[:, off:].view(300, 6, 48).copy_(x)
            assert odd.data_ptr() % (16 if dtype == F32 else 8) or off == 4
            assert torch.equal(ab.rope(odd, None, plan, pos, inverse=inverse)[0], want)
            assert torch.equal(ab.rope(odd, None, plan, pos, inverse=inverse, out=(odd, None))[0], want)
