"""Tensors whose offsets pass 32 bits: the last rows come out as they do alone."""
import pytest
import torch

import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
ROWS, COLS = 525_000, 8192          # 4.3e9 elements, above 2^32


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 70 GB")
    yield
    torch.cuda.empty_cache()


def big(seed, rows=ROWS, cols=COLS):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols, dtype=F16, device="cuda")
    for i in range(0, rows, 65536):
        x[i: i + 65536].normal_(generator=g)
    return x


def ends(t):
    """Rows at the start, around the 2^32nd element and at the end."""
    mid = (1 << 32) // COLS
    return torch.cat([t[:3], t[mid - 2: mid + 2], t[-3:]])


def test_checkpoints_and_swiglu():
    a, b = big(1), big(2)
    c = ab.act8_pack(a, "int8")
    few = ab.act8_pack(ends(a), "int8")
    assert torch.equal(ends(c.data), few.data) and torch.equal(ends(c.scale), few.scale)
    y = ab.act8_unpack(c)
    assert torch.equal(ends(y), ab.act8_unpack(few))
    y, ca, cb = ab.swiglu(a, b, checkpoint="e4m3", out=y)
    fy, fa, fb = ab.swiglu(ends(a), ends(b), checkpoint="e4m3")
    assert torch.equal(ends(y), fy) and torch.equal(ends(ca.data), fa.data) and torch.equal(ends(cb.scale), fb.scale)
    del c, y
    fda, fdb, fcy = ab.swiglu_backward(ends(a), fa, fb, checkpoint="e4m3")
    da, db, cy = ab.swiglu_backward(a, ca, cb, checkpoint="e4m3", out=(a, b))
    assert torch.equal(ends(da), fda) and torch.equal(ends(db), fdb)
    assert torch.equal(ends(cy.data), fcy.data) and torch.equal(ends(cy.scale), fcy.scale)


def test_heads():
    q = big(3).view(ROWS, 64, 128)
    plan, g = ab.RopePlan(128), torch.ones(128, dtype=F16, device="cuda")
    pos = torch.arange(ROWS, device="cuda")
    fq, fpos = ends(q.view(ROWS, -1)).view(-1, 64, 128), ends(pos)
    want = ab.rope(fq, None, plan, fpos)[0]
    want2, _, fc, _ = ab.qk_norm_rope(fq, None, g, None, plan, fpos, checkpoint="e4m3")
    y, _, c, _ = ab.qk_norm_rope(q, None, g, None, plan, pos, checkpoint="e4m3")
    assert torch.equal(ends(y.view(ROWS, -1)).view_as(fq), want2) and torch.equal(ends(c.data), fc.data)
    back = ab.qk_norm_rope_backward(y, None, c, None, g, None, plan, pos, out=(y, None))[0]
    few = ab.qk_norm_rope_backward(want2, None, fc, None, g, None, plan, fpos)[0]
    assert torch.equal(ends(back.view(ROWS, -1)).view_as(fq), few)
    ab.rope(q, None, plan, pos, out=(q, None))
    assert torch.equal(ends(q.view(ROWS, -1)).view_as(fq), want)


@pytest.mark.parametrize("nin,nout,dtype", [(4224, 64, F16), (64, 4224, F16), (64, 4221, torch.bfloat16)])
def test_weight_grad(nin, nout, dtype):
    """Ones and zeros with signs: a sum is a whole number below the 1.1 million tokens, exact in FP32."""
    tokens, part = 1_060_000, 100_000
    g = torch.Generator(device="cuda").manual_seed(nin)
    mk = lambda n: torch.randint(-1, 2, (tokens, n), generator=g, device="cuda", dtype=torch.int8).to(dtype)  # noqa: E731
    x, dy = mk(nin), mk(nout)
    got = ab.weight_grad(ab.act8_pack(x), dy, dtype=F32)
    want = torch.zeros(nin, nout, dtype=torch.float64, device="cuda")
    for i in range(0, tokens, part):
        want += x[i: i + part].double().T @ dy[i: i + part].double()
    assert torch.equal(got.double(), want)
