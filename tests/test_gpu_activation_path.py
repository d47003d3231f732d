"""The activation operators together, as a backward that fills the gradient
buffer uses them, and the step on what they left there."""
import numpy as np
import pytest
import torch

import act_ref as ref
import ark_b200 as ab
from ark_b200 import layout
from gpu_util import host

pytestmark = pytest.mark.gpu
F16 = torch.float16
T, D, H, HQ, HK, HD = 160, 128, 320, 4, 2, 32
SCALE = 1024.0
HP = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, grad_clip=1.0)


def model():
    S = layout.TensorSpec
    return layout.Layout("layer", [S("wq", D * HQ * HD, True), S("wk", D * HK * HD, True), S("w1", D * H, True),
                                   S("w3", D * H, True), S("w2", H * D, True), S("gq", HD, False), S("gk", HD, False)])


def weights(L, seed):
    g = torch.Generator().manual_seed(seed)
    w = (0.05 * torch.randn(L.n, generator=g)).half()
    w[L.offsets["gq"]:] = 1
    return w.cuda()


def at(L, buf, name, *shape):
    lo = L.offsets[name]
    return buf[lo: lo + int(np.prod(shape))].view(*shape)


def forward(L, w, x, plan, kind):
    """What the forward keeps: checkpoints alone."""
    cx = ab.act8_pack(x, kind)
    q = (x @ at(L, w, "wq", D, HQ * HD)).view(T, HQ, HD)
    k = (x @ at(L, w, "wk", D, HK * HD)).view(T, HK, HD)
    q, k, cq, ck = ab.qk_norm_rope(q, k, at(L, w, "gq", HD), at(L, w, "gk", HD), plan, seq_len=T // 2, checkpoint=kind)
    y, ca, cb = ab.swiglu(x @ at(L, w, "w1", D, H), x @ at(L, w, "w3", D, H), checkpoint=kind)
    return (q, k, y @ at(L, w, "w2", H, D)), (cx, cq, ck, ca, cb)


def backward(L, w, opt, kept, plan, dq, dk, dout):
    """Gradients of all tensors into the gradient buffer; what each product read."""
    cx, cq, ck, ca, cb = kept
    dy = dout @ at(L, w, "w2", H, D).t()
    da, db, cy = ab.swiglu_backward(dy, ca, cb, checkpoint=ca.kind)
    opt.weight_grad("w2", cy, dout)
    opt.weight_grad("w1", cx, da)
    opt.weight_grad("w3", cx, db)
    gains = opt.grad_view("gq", HD), opt.grad_view("gk", HD)
    dq, dk, _, _ = ab.qk_norm_rope_backward(dq, dk, cq, ck, at(L, w, "gq", HD), at(L, w, "gk", HD), plan, seq_len=T // 2,
                                            out_gains=gains, accumulate=True)
    opt.weight_grad("wq", cx, dq.flatten(1))
    opt.weight_grad("wk", cx, dk.flatten(1))
    return {"w2": (cy, dout), "w1": (cx, da), "w3": (cx, db), "wq": (cx, dq.flatten(1)), "wk": (cx, dk.flatten(1))}


def gradients(seed):
    g = torch.Generator().manual_seed(seed)
    return [(0.02 * torch.randn(*s, generator=g)).half().cuda() for s in ((T, HQ, HD), (T, HK, HD), (T, D))]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_backward_and_step(oracle, kind):
    L = model()
    sc = ab.LossScaleConfig(init=SCALE, every=50, max=2.0 ** 24)
    opt = ab.Optimizer(L, ab.AdamConfig(**HP), sc, constant_lr=True, initial_step=3)
    w, m, v = weights(L, 1), torch.zeros(L.n, device="cuda"), torch.zeros(L.n, device="cuda")
    full, shard = opt.grad_buffer(), torch.empty(L.n, dtype=F16, device="cuda")
    plan = ab.RopePlan(HD, layout="interleaved", scaling="linear", factor=2.0)
    cfg = oracle.make_cfg(lr_table=(3e-4,), n_decay=L.n_decay, scale_every=50, scale_max=2.0 ** 24)
    st = oracle.make_state(SCALE, opt_step=3)
    w_h, m_h, v_h = host(w).copy(), host(m).copy(), host(v).copy()
    for step in range(2):
        opt.zero_grads()
        want, size, first = {}, {}, {}
        for micro in range(2):                                   # gradients add up over micro-batches
            g = torch.Generator().manual_seed(10 * step + micro)
            x = torch.randn(T, D, generator=g).half().cuda()
            _, kept = forward(L, w, x, plan, kind)
            read = backward(L, w, opt, kept, plan, *gradients(100 + 10 * step + micro))
            for name, (c, dy) in read.items():
                X, G = ref.values(c.data, c.scale, c.cols, kind), dy.cpu().double()
                want[name] = want.get(name, 0) + X.T @ G
                size[name] = size.get(name, 0) + X.abs().T @ G.abs()
                first.setdefault(name, want[name])
        torch.cuda.synchronize()
        for name in want:
            got = opt.grad_view(name, *want[name].shape).cpu().double()
            # T FP32 additions a batch, and a rounding to FP16 after each
            sums = 2 * T * 2.0 ** -23 * size[name]
            tol = ref.HALF[F16] * (first[name].abs() + want[name].abs() + 2 * sums) + 2 * ref.TINY[F16] + sums
            assert ((got - want[name]).abs() <= tol).all(), name
        g_h = host(full).copy()
        opt.step_reduce(w, shard, m, v)
        assert oracle.step_flat_f16(cfg, st, w_h, g_h, m_h, v_h) == 0
        s = opt.status()
        assert s["last_overflow"] == 0 and s["opt_step"] == 4 + step
        assert np.array_equal(host(w), w_h) and np.array_equal(host(m).view(np.uint32), m_h.view(np.uint32))
    # an infinity in an activation makes the next step a skipped one
    opt.zero_grads()
    x[5, 7] = float("inf")
    out, kept = forward(L, w, x, plan, kind)
    backward(L, w, opt, kept, plan, *gradients(7))
    before = w.clone()
    opt.step_reduce(w, shard, m, v)
    s = opt.status()
    assert s["last_overflow"] == 1 and s["loss_scale"] == SCALE / 2 and torch.equal(w, before)
    opt.close()


def chain(x, y, plan, pos, g, dy):
    """Every operator once, on given tensors."""
    c = ab.act8_pack(x)
    a, ca, cb = ab.swiglu(x, y, checkpoint="int8")
    da, db, cy = ab.swiglu_backward(dy, ca, cb, checkpoint="int8")
    q = x.view(x.shape[0], -1, 64)
    r = ab.qk_norm_rope(q, q[:, :2], g, g, plan, pos, checkpoint="e4m3")
    b = ab.qk_norm_rope_backward(r[0], r[1], r[2], r[3], g, g, plan, pos)
    big = ab.weight_grad(ab.act8_pack(dy.repeat(1, 8)), dy.repeat(1, 8))
    split = ab.weight_grad(c, dy[:, 1:], dtype=torch.float32)
    return [ab.act8_unpack(c), a, da, db, ab.act8_unpack(cy), *r[:2], *b, ab.weight_grad(c, da), big, split,
            *ab.rope(q, None, plan, pos, inverse=True)[:1]]


def inputs(seed, t=600, d=256):
    g = torch.Generator().manual_seed(seed)
    mk = lambda: torch.randn(t, d, generator=g).half().cuda()  # noqa: E731
    return mk(), mk(), mk()


def test_captured_and_replayed():
    plan, g = ab.RopePlan(64), torch.ones(64, dtype=F16, device="cuda")
    pos = torch.arange(600, device="cuda", dtype=torch.int32) % 100
    x, y, dy = inputs(1)
    other = inputs(2)
    want = [t.clone() for t in chain(*other[:2], plan, pos, g, other[2])]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                           # two graphs of the same calls alive at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain(x, y, plan, pos, g, dy)
        graphs.append((graph, out))
    for t, o in zip((x, y, dy), other):
        t.copy_(o)
    pos.add_(0)
    for graph, _ in graphs:
        graph.replay()
    for graph, out in graphs:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_calls_on_two_streams():
    plan, g = ab.RopePlan(64), torch.ones(64, dtype=F16, device="cuda")
    pos = torch.arange(600, device="cuda") % 100
    sets = [inputs(3), inputs(4)]
    want = [[t.clone() for t in chain(s[0], s[1], plan, pos, g, s[2])] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        got = []
        for st, s in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(chain(s[0], s[1], plan, pos, g, s[2]))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_optimizer_weight_grad_runs_on_the_steps_stream():
    L = layout.Layout("one", [layout.TensorSpec("w", 64 * 96, True)])
    side = torch.cuda.Stream()
    opt = ab.Optimizer(L, ab.AdamConfig(**HP), ab.LossScaleConfig(init=1.0), constant_lr=True, stream=side)
    opt.grad_buffer()
    opt.zero_grads()
    x = torch.randint(-8, 9, (200, 64)).half().cuda()
    dy = torch.randint(-4, 5, (200, 96)).half().cuda()
    c = ab.act8_pack(x, "int8")
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        opt.weight_grad("w", c, dy)
    side.synchronize()
    want = 3 * (x.double().T @ dy.double())
    assert want.abs().max() < 2048 * 8 and torch.equal(opt.grad_view("w", 64, 96).double(), want.half().double())
    opt.weight_grad("w", c, dy, accumulate=False)
    side.synchronize()
    assert torch.equal(opt.grad_view("w", 64, 96).double(), want / 3)
    opt.close()


def test_tensors_without_the_right_shape_are_refused():
    x = torch.zeros(8, 128, dtype=F16, device="cuda")
    c, p = ab.act8_pack(x), ab.RopePlan(64)
    q, g = x.view(8, 2, 64), torch.ones(64, dtype=F16, device="cuda")
    for call in (lambda: ab.act8_pack(x.t()), lambda: ab.act8_pack(x, out=ab.Act8.empty(8, 127)),
                 lambda: ab.act8_pack(x, "fp8"), lambda: ab.act8_unpack(c, out=x[:7]),
                 lambda: ab.act8_unpack(c, out=x[:1].expand(8, 128)),
                 lambda: ab.weight_grad(c, x[:7]), lambda: ab.weight_grad(c, x, out=x), lambda: ab.weight_grad(c, x, accumulate=True),
                 lambda: ab.weight_grad(c, x, out=torch.zeros(128, 128, device="cuda"), dtype=F16),
                 lambda: ab.swiglu(x, x.bfloat16()), lambda: ab.swiglu(x, x[:, 1:]), lambda: ab.swiglu(x, x, out=x.float()),
                 lambda: ab.swiglu_backward(x, c, ab.act8_pack(x, "int8")), lambda: ab.swiglu_backward(x[1:], c, c),
                 lambda: ab.swiglu_backward(x, c, c, checkpoint="int8"),
                 lambda: ab.rope(q.transpose(1, 2), None, p), lambda: ab.rope(q, q[:7], p), lambda: ab.rope(q, q.float(), p),
                 lambda: ab.rope(q[..., :32], None, p), lambda: ab.rope(q, None, p, positions=torch.zeros(7, device="cuda", dtype=torch.int32)),
                 lambda: ab.rope(q, None, p, positions=torch.zeros(8, dtype=torch.int32)),
                 lambda: ab.rope(q, None, p, out=(q, q)), lambda: ab.rope(q, q, p, out=(q, None)),
                 lambda: ab.rope(q, None, p, seq_len=0), lambda: ab.rope(q, None, p, torch.zeros(8, device="cuda", dtype=torch.int32), 8),
                 lambda: ab.qk_norm_rope(q, None, g[:32], None, p), lambda: ab.qk_norm_rope(q, q, g, g.float(), p),
                 lambda: ab.qk_norm_rope_backward(q, None, ab.act8_pack(x[:7]), None, g, None, p),
                 lambda: ab.qk_norm_rope_backward(q, q, c, q, g, g, p),
                 lambda: ab.qk_norm_rope_backward(q, None, q, None, g, None, p, accumulate=True),
                 lambda: ab.rope(torch.zeros(2, 1, 300, device="cuda"), None, p)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ab.act8_unpack(c, torch.float64), lambda: ab.weight_grad(c, x.float()), lambda: ab.weight_grad(x, x),
                 lambda: ab.rope(q, None, None), lambda: ab.rope(q, None, p, positions=torch.zeros(8, device="cuda")),
                 lambda: ab.swiglu(x.double(), x.double())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ab.ArkError):
        ab.rope(q, None, p, out=(x[:1].view(1, 2, 64).expand(8, 2, 64), None))
