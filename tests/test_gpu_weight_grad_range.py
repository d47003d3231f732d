"""The weight gradient with FP16 dY from checkpoints of other types: values
that FP16 cannot hold keep their size, or show."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def inputs(tokens, nin, nout, seed):
    """Whole numbers whose checkpoint is exact, each 32 columns times a power of two far outside
    of FP16's range on both sides, and whole dY of FP16's 11 significant bits.  A sum is a whole
    number below 15 * 1023 * 1024 < 2^24 times that power: FP32 holds it exactly in any order."""
    assert tokens <= 1024
    g = torch.Generator().manual_seed(seed)
    size = torch.exp2(torch.randint(-60, 61, (-(-nin // 32),), generator=g).float()).repeat_interleave(32)[:nin]
    x = torch.randint(-15, 16, (tokens, nin), generator=g).float() * size
    return x, torch.randint(-1023, 1024, (tokens, nout), generator=g).to(F16)


# the last two are pairs of CTAs on a B200: whole tiles, and split tokens
@pytest.mark.parametrize("tokens,nin,nout", [(1, 1, 1), (65, 129, 257), (300, 96, 40), (513, 2048, 4800), (1000, 700, 100)])
@pytest.mark.parametrize("kind,dtype", [("e4m3", F32), ("int8", BF16), ("int8", F32), ("e4m3", BF16)])
def test_values_outside_of_fp16_keep_their_size(tokens, nin, nout, kind, dtype):
    x, dy = inputs(tokens, nin, nout, tokens + nin)
    c = ab.act8_pack(x.to(dtype).cuda(), kind)
    want = x.double().T @ dy.double()
    got = ab.weight_grad(c, dy.cuda(), dtype=F32)
    assert torch.equal(got.cpu().double(), want)
    acc = got.clone()
    ab.weight_grad(c, dy.cuda(), out=acc, accumulate=True)
    assert torch.equal(acc.cpu().double(), 2 * want)
    assert torch.equal(ab.weight_grad(c, dy.cuda(), dtype=BF16).cpu(), want.to(BF16))
    assert torch.equal(ab.weight_grad(c, dy.cuda()).cpu(), want.float().to(F16))     # beyond FP16: an infinity


def test_rows_of_any_lie_and_broadcast():
    x, buf = inputs(200, 160, 131, 3)
    c = ab.act8_pack(x.cuda(), "int8")
    dy = buf.cuda()[:, 1:130]
    want = x.double().T @ dy.cpu().double()
    big = torch.full((162, 134), 3.0, device="cuda")
    ab.weight_grad(c, dy, out=big[1:161, 2:131])
    assert torch.equal(big[1:161, 2:131].cpu().double(), want)
    big[1:161, 2:131] = 3
    assert (big == 3).all()
    row = dy[:1].expand(200, 129)
    assert torch.equal(ab.weight_grad(c, row, dtype=F32).cpu().double(), x.double().T @ row.cpu().double())
    none = ab.act8_pack(x[:0].cuda())
    assert (ab.weight_grad(none, dy[:0], out=torch.ones(160, 129, device="cuda")) == 0).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_large_and_small_activations(kind):
    """1e5 and 1e-8 beside ordinary values, as FP32 and BF16 activations have them."""
    x = torch.ones(64, 96)
    x[:, :32], x[:, 32:64] = 1e5, 1e-8
    dy = torch.full((64, 8), 16.0, dtype=F16, device="cuda")
    for dtype in (F32, BF16):
        X = ref.through(x.to(dtype), kind)
        got = ab.weight_grad(ab.act8_pack(x.to(dtype).cuda(), kind), dy, dtype=F32).cpu().double()
        want = X.sum(0)[:, None] * 16          # 64 equal terms: 14 significant bits
        assert torch.equal(got, want.expand(96, 8))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("tokens,nin,nout", [(70, 96, 24), (600, 2048, 4800)])   # few tiles, pairs
def test_what_fp16_cannot_hold_shows(tokens, nin, nout, kind):
    """A checkpoint that its holder calls FP16's and is not: an infinity, not a number of another size."""
    x = torch.ones(tokens, nin)
    x[3, 40], x[5, 70] = 1e5, 65504.0
    c = ab.act8_pack(x.cuda(), kind)
    assert c.wide
    c = ab.Act8(c.data, c.scale, c.cols, c.kind)
    assert not c.wide
    w = ab.weight_grad(c, torch.ones(tokens, nout, dtype=F16, device="cuda"), dtype=F32).cpu()
    assert torch.isinf(w[40]).all()
    # FP16's largest is not: it reads as 65536 and is taken for 65504
    X = ref.through(x, kind)
    assert X[5, 70] == 65536
    X[5, 70] = 65504
    rest = [i for i in range(nin) if i != 40]
    assert torch.equal(w[rest].double(), X[:, rest].sum(0)[:, None].expand(-1, nout))
    ok = ab.act8_pack(x.clamp(max=65504).half().cuda(), kind)
    assert not ok.wide and torch.isfinite(ab.weight_grad(ok, torch.ones(tokens, nout, dtype=F16, device="cuda"), dtype=F32)).all()


def test_who_is_wide():
    x = torch.ones(8, 64, device="cuda")
    for dtype, wide in ((F16, False), (BF16, True), (F32, True)):
        t = x.to(dtype)
        room = ab.Act8.empty(8, 64)
        assert not room.wide
        assert ab.act8_pack(t, out=room).wide is wide and room.wide is wide and ab.act8_pack(t).wide is wide
        _, a, b = ab.swiglu(t, t, checkpoint="int8")
        cy = ab.swiglu_backward(t, a, b, checkpoint="int8")[2]
        q, _, cq, ck = ab.qk_norm_rope(t.view(8, 2, 32), t.view(8, 2, 32), t[0, :32], t[0, :32], ab.RopePlan(32), checkpoint="e4m3")
        assert [c.wide for c in (a, b, cy, cq, ck)] == [wide] * 5
    ab.act8_pack(x.half(), out=room)
    assert not room.wide and ab.Act8(room.data, room.scale, 64, "e4m3", wide=True).wide


def test_captured_replayed_and_on_two_streams():
    sets = [[t.cuda() for t in inputs(500, 300, 200, s)] for s in (11, 12)]
    want = [x.double().T @ dy.double() for x, dy in sets]

    def call(x, dy):
        return ab.weight_grad(ab.act8_pack(x, "int8"), dy, dtype=F32)

    x, dy = (t.clone() for t in sets[0])
    call(x, dy)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(x, dy)
        graphs.append((graph, out))
    for (a, b), w in ((sets[1], want[1]), (sets[0], want[0])):
        x.copy_(a), dy.copy_(b)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out.double(), w) for _, out in graphs)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        got = []
        for st, s in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(call(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(g.double(), w) for g, w in zip(got, want))
