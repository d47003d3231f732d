"""Cases of the activation operators beside the optimizer step: 8-bit
activation checkpoints and the backward that reads them, and the norm and
rotation of queries and keys.

An 8-bit checkpoint holds a [rows, cols] activation as one byte per element
and one power-of-two scale per 32 columns of a row: the scale 2^k is the
smallest with max|x| <= top * 2^k (top: 448 for e4m3, 127 for int8, k at
least -126), the byte is x * 2^-k rounded to nearest even, and the scale byte
is k + 127, or 255 (the block reads back as NaN) when the block holds an
infinity or a NaN.  Rows are padded to 128 columns.

Five operators, by a case's "op":
  checkpoint  pack, then unpack (a finite value saturates at the type's largest)
  weight_grad dW = X^T dY with X read from its checkpoint
  swiglu      y = silu(a) * b, a and b checkpointed; and the backward from them
  qk_norm     RMS norm of each head of q and k with gains, then the rotation,
              q and k checkpointed; and the backward from the checkpoints
  rope        the rotation alone, forward or inverse (its backward)
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK, PITCH = 32, 128


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decoding step's worth of rows of the 768-wide model: latency
        dict(name="checkpoint_small", op="checkpoint", rows=64, cols=768, kind="e4m3", dtype="fp16"),
        # the FFN activation of the 4096-wide model over 8192 tokens
        dict(name="checkpoint_ffn", op="checkpoint", rows=8192, cols=11008, kind="int8", dtype="fp16"),
        # wq of the 768-wide model: two micro-batches of 512 tokens, the second added to the first
        dict(name="weight_grad_768", op="weight_grad", tokens=1024, micro=2, nin=768, nout=768, kind="e4m3",
             dtype="fp16", out="fp16"),
        # w1 of the 2048-wide model over a batch cut to an odd number of tokens, FP32 gradients
        dict(name="weight_grad_ragged", op="weight_grad", tokens=4001, micro=1, nin=2048, nout=5504, kind="int8",
             dtype="bf16", out="fp32"),
        # w1 of the 4096-wide model over 8192 tokens: the largest
        dict(name="weight_grad_4096", op="weight_grad", tokens=8192, micro=1, nin=4096, nout=11008, kind="e4m3",
             dtype="fp16", out="fp16"),
        # the FFN of the 768-wide model, one sequence of 1024, forward and backward
        dict(name="swiglu_2048", op="swiglu", part="train", rows=1024, cols=2048, kind="e4m3", dtype="fp16", fused=False),
        # backward alone on an odd number of rows and columns, gate and up in one buffer, and
        # the product remade as a checkpoint for the down projection's weight gradient
        dict(name="swiglu_ragged", op="swiglu", part="back", rows=777, cols=5501, kind="int8", dtype="bf16", fused=True),
        # the FFN of the 4096-wide model over 8192 tokens, forward and backward
        dict(name="swiglu_11008", op="swiglu", part="train", rows=8192, cols=11008, kind="e4m3", dtype="fp16", fused=False),
        # 12 heads of 64, one sequence of 1024, forward and backward
        dict(name="qk_norm_12x64", op="qk_norm", tokens=1024, seq=1024, hq=12, hk=12, dim=64, rot=64, kind="e4m3",
             dtype="fp16", gains="fp16", layout="half", scaling="none"),
        # 32 query and 8 key heads of 128, four sequences of 2048 with padding at their ends
        dict(name="qk_norm_32x128", op="qk_norm", tokens=8192, seq=2048, hq=32, hk=8, dim=128, rot=128, kind="e4m3",
             dtype="bf16", gains="fp32", layout="half", scaling="none"),
        # single tokens of 64 requests at far positions, q and k inside one qkv buffer
        dict(name="rope_tokens", op="rope", tokens=64, seq=0, hq=12, hk=12, dim=64, rot=32, dtype="fp16",
             layout="interleaved", scaling="linear", inverse=False),
        # one long sequence, positions scaled by parts, the backward's rotation
        dict(name="rope_long", op="rope", tokens=131072, seq=131072, hq=8, hk=2, dim=128, rot=128, dtype="bf16",
             layout="half", scaling="parts", inverse=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["checkpoint", "weight_grad", "swiglu", "qk_norm", "rope"])
    kind, dtype = rng.choice(["e4m3", "int8"]), rng.choice(["fp16", "bf16"])
    if op == "checkpoint":
        return dict(op=op, rows=_spread(rng, 1, 8192), cols=_spread(rng, 48, 11008), kind=kind,
                    dtype=rng.choice(["fp16", "bf16", "fp32"]))
    if op == "weight_grad":
        micro = rng.choice([1, 1, 2])
        return dict(op=op, tokens=micro * _spread(rng, 1, 4096), micro=micro, nin=_spread(rng, 48, 4096),
                    nout=_spread(rng, 48, 11008), kind=kind, dtype=dtype, out=rng.choice([dtype, "fp32"]))
    if op == "swiglu":
        return dict(op=op, part=rng.choice(["train", "back"]), rows=_spread(rng, 1, 8192), cols=_spread(rng, 48, 11008),
                    kind=kind, dtype=dtype, fused=rng.random() < 0.5)
    dim = rng.choice([32, 64, 72, 80, 96, 100, 128, 192, 256])
    rot = rng.choice([dim, dim, dim // 4 * 2, rng.randrange(4, dim + 1, 2)])
    hk = rng.choice([1, 2, 4, 8])
    c = dict(op=op, hq=hk * rng.choice([1, 2, 3, 4]), hk=hk, dim=dim, rot=rot, dtype=dtype,
             layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "base", "parts", "wave"]))
    if op == "qk_norm":
        seq = _spread(rng, 1, 2048)
        return dict(c, tokens=seq * rng.choice([1, 2, 4]), seq=seq, kind=kind, gains=rng.choice([dtype, "fp32"]))
    tokens = _spread(rng, 1, 32768)
    return dict(c, tokens=tokens, seq=rng.choice([0, tokens]), inverse=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _activation(g, rows, cols, dtype, device):
    """Activations as layers leave them: columns of unlike size, one in 256 eight times larger."""
    col = torch.exp(0.5 * torch.randn(cols, generator=g, device=device))
    col = torch.where(torch.rand(cols, generator=g, device=device) < 1 / 256, 8 * col, col)
    return (torch.randn(rows, cols, generator=g, device=device) * col).to(dtype)


def _scaling(name):
    """Arguments of the position scaling, as a model's configuration has them."""
    return {
        "none": dict(base=10000.0),
        "linear": dict(base=10000.0, scaling="linear", factor=4.0),
        "base": dict(base=10000.0, scaling="base", factor=8.0),
        "parts": dict(base=10000.0, scaling="parts", factor=16.0, original=8192, fast=32.0, slow=1.0),
        "wave": dict(base=500000.0, scaling="wave", factor=8.0, original=8192, fast=4.0, slow=1.0),
    }[name]


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    op, dt = c["op"], TYPES[c["dtype"]]
    s = {"case": c}
    if op == "checkpoint":
        s["x"] = _activation(g, c["rows"], c["cols"], dt, dev)
    elif op == "weight_grad":
        n = c["tokens"] // c["micro"]
        s["x"] = [_pack(_activation(g, n, c["nin"], dt, dev), c["kind"]) for _ in range(c["micro"])]
        s["dy"] = [(0.05 * torch.randn(n, c["nout"], generator=g, device=dev)).to(dt) for _ in range(c["micro"])]
    elif op == "swiglu":
        ab = _activation(g, c["rows"], 2 * c["cols"], dt, dev)
        a, b = ab[:, : c["cols"]], ab[:, c["cols"]:]
        s["a"], s["b"] = (a, b) if c["fused"] else (a.contiguous(), b.contiguous())
        s["dy"] = (0.05 * torch.randn(c["rows"], c["cols"], generator=g, device=dev)).to(dt)
        if c["part"] == "back":
            s["ca"], s["cb"] = _pack(s["a"], c["kind"]), _pack(s["b"], c["kind"])
    else:
        t, hq, hk, d = c["tokens"], c["hq"], c["hk"], c["dim"]
        qkv = _activation(g, t, (hq + 2 * hk) * d, dt, dev).view(t, hq + 2 * hk, d)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq: hq + hk]
        if c["seq"]:
            pos = torch.arange(t, device=dev, dtype=torch.int32) % c["seq"]
        else:
            pos = torch.randint(0, 1 << 17, (t,), generator=g, device=dev, dtype=torch.int32)
        if op == "qk_norm":
            # the last sequence ends early: padding
            pos = torch.where(torch.arange(t, device=dev) < t - c["seq"] // 16, pos, torch.full_like(pos, -1))
            s["gq"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(TYPES[c["gains"]])
            s["gk"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(TYPES[c["gains"]])
            s["dq"] = (0.05 * torch.randn(t, hq, d, generator=g, device=dev)).to(dt)
            s["dk"] = (0.05 * torch.randn(t, hk, d, generator=g, device=dev)).to(dt)
        s["pos"] = pos
        if own:  # the rotation's plan, which a program makes once from its configuration
            import ark_b200 as ab
            s["plan"] = ab.RopePlan(c["rot"], layout=c["layout"], **_scaling(c["scaling"]))
        else:
            s["freq"], s["gain"] = _freqs(c, dev)
    return s


# ---------------------------------------------------------------- plain forms
def _pad(x, to):
    n = -x.shape[1] % to
    return torch.cat([x, x.new_zeros(x.shape[0], n)], 1) if n else x


def _pack(x, kind):
    """(bytes [rows, cols padded to 128], scale bytes [rows, padded cols / 32])."""
    blocks = _pad(x.float(), PITCH).unflatten(1, (-1, BLOCK))
    top, m0, e0 = (448.0, 448.0 / 512, 9) if kind == "e4m3" else (127.0, 127.0 / 128, 7)
    amax = blocks.abs().amax(2)
    bad = ~torch.isfinite(amax)
    m, e = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))
    k = torch.where(m > m0, e - e0 + 1, e - e0)
    k = torch.where(amax == 0, torch.full_like(k, -126), k).clamp(min=-126)
    v = torch.ldexp(blocks, -k.unsqueeze(2))
    v = torch.where(bad.unsqueeze(2), torch.zeros_like(v), v)
    q = v.to(torch.float8_e4m3fn).view(torch.uint8) if kind == "e4m3" else torch.round(v).to(torch.int8).view(torch.uint8)
    return q.flatten(1), torch.where(bad, torch.full_like(k, 255), k + 127).to(torch.uint8)


def _values(packed, kind, cols):
    """The FP32 values that a checkpoint stands for."""
    q, scale = packed
    v = q.view(torch.float8_e4m3fn).float() if kind == "e4m3" else q.view(torch.int8).float()
    s = torch.ldexp(torch.ones_like(scale, dtype=torch.float32), scale.int() - 127)
    s = torch.where(scale == 255, torch.full_like(s, math.nan), s)
    return (v.unflatten(1, (-1, BLOCK)) * s.unsqueeze(2)).flatten(1)[:, :cols]


def _round(x, dt):
    """Finite values saturate at the type's largest."""
    return x.clamp(-torch.finfo(dt).max, torch.finfo(dt).max).to(dt)


def _freqs(c, dev):
    """Radians a position of each pair, in 64 bits, and the factor on cos and sin."""
    a = _scaling(c["scaling"])
    half = c["rot"] // 2
    i = torch.arange(half, device=dev, dtype=torch.float64)
    base, f = a["base"], a.get("factor", 1.0)
    kind = a.get("scaling", "none")
    if kind == "base":
        base = base * f ** (c["rot"] / (c["rot"] - 2))
    w = base ** (-2 * i / c["rot"])
    if kind == "linear":
        return w / f, 1.0
    if kind == "parts":
        at = lambda turns: c["rot"] * math.log(a["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(a["fast"])), 0), min(math.ceil(at(a["slow"])), c["rot"] - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1
    if kind == "wave":
        turns = a["original"] * w / (2 * math.pi)
        keep = ((turns - a["slow"]) / (a["fast"] - a["slow"])).clamp(0, 1)
        return w * keep + w / f * (1 - keep), 1.0
    return w, 1.0


def _turn(n, s, sign):
    """The rotation of the first `rot` of each head's values, in FP32."""
    c = s["case"]
    angle = s["pos"].double().unsqueeze(1) * s["freq"]
    co, si = (torch.cos(angle) * s["gain"]).float().unsqueeze(1), (sign * torch.sin(angle) * s["gain"]).float().unsqueeze(1)
    r, rest = n[..., : c["rot"]], n[..., c["rot"]:]
    if c["layout"] == "half":
        x, y = r.chunk(2, 2)
        r = torch.cat([x * co - y * si, y * co + x * si], 2)
    else:
        x, y = r[..., 0::2], r[..., 1::2]
        r = torch.stack([x * co - y * si, y * co + x * si], 3).flatten(2)
    return torch.cat([r, rest], 2) * (s["pos"] >= 0).view(-1, 1, 1)


EPS = 1e-6


def _norm_back(x, dn, gain, live):
    """(dx, dgain) of n = x * rsqrt(mean x^2 + eps) * gain; rows that are not live have no part in it."""
    x = torch.where(live, x, torch.zeros_like(x))
    r = torch.rsqrt(x.square().mean(2, keepdim=True) + EPS)
    h, gd = x * r, dn * gain.float()
    return (gd - h * (h * gd).mean(2, keepdim=True)) * r * live, (dn * h).sum((0, 1))


def _plain(s):
    c = s["case"]
    op, dt = c["op"], TYPES[c["dtype"]]
    if op == "checkpoint":
        p = _pack(s["x"], c["kind"])
        return {"x": _round(_values(p, c["kind"], c["cols"]), dt), "scale": p[1]}
    if op == "weight_grad":
        out = TYPES[c["out"]]
        dw = [_values(x, c["kind"], c["nin"]).t() @ dy.float() for x, dy in zip(s["x"], s["dy"])]
        return {"dw": (dw[0].to(out).float() + dw[1]).to(out) if c["micro"] == 2 else dw[0].to(out)}
    if op == "swiglu":
        res = {}
        if c["part"] == "train":
            a, b = s["a"].float(), s["b"].float()
            res["y"] = (a * torch.sigmoid(a) * b).to(dt)
            ca, cb = _pack(s["a"], c["kind"]), _pack(s["b"], c["kind"])
        else:
            ca, cb = s["ca"], s["cb"]
        a, b, dy = _values(ca, c["kind"], c["cols"]), _values(cb, c["kind"], c["cols"]), s["dy"].float()
        sg = torch.sigmoid(a)
        res["da"], res["db"] = (dy * b * sg * (1 + a * (1 - sg))).to(dt), (dy * a * sg).to(dt)
        if c["part"] == "back":
            # remade in 64 bits and rounded to its type, as the forward's was: most products of
            # two 8-bit values lie next to a border of the 8-bit grid
            y = (a.double() * torch.sigmoid(a.double()) * b.double()).to(dt)
            res["y"] = _round(_values(_pack(y, c["kind"]), c["kind"], c["cols"]), dt)
        return res
    if op == "rope":
        sign = -1.0 if c["inverse"] else 1.0
        return {"q": _turn(s["q"].float(), s, sign).to(dt), "k": _turn(s["k"].float(), s, sign).to(dt)}
    q, k = s["q"].float(), s["k"].float()
    nq = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * s["gq"].float()
    nk = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * s["gk"].float()
    live = (s["pos"] >= 0).view(-1, 1, 1)
    xq = _values(_pack(s["q"].flatten(1), c["kind"]), c["kind"], q[0].numel()).view_as(q)
    xk = _values(_pack(s["k"].flatten(1), c["kind"]), c["kind"], k[0].numel()).view_as(k)
    dq, dgq = _norm_back(xq, _turn(s["dq"].float(), s, -1.0), s["gq"], live)
    dk, dgk = _norm_back(xk, _turn(s["dk"].float(), s, -1.0), s["gk"], live)
    return {"q": _turn(nq, s, 1.0).to(dt), "k": _turn(nk, s, 1.0).to(dt), "dq": dq.to(dt), "dk": dk.to(dt),
            "dgq": dgq.to(TYPES[c["gains"]]), "dgk": dgk.to(TYPES[c["gains"]])}


# ---------------------------------------------------------------- the framework's calls
def _kernels(s):
    import ark_b200 as ab
    c = s["case"]
    op, dt = c["op"], TYPES[c["dtype"]]
    if op == "checkpoint":
        p = ab.act8_pack(s["x"], c["kind"])
        return {"x": ab.act8_unpack(p, dt), "scale": p.scale}
    if op == "weight_grad":
        dw = ab.weight_grad(ab.Act8(*s["x"][0], c["nin"], c["kind"]), s["dy"][0], dtype=TYPES[c["out"]])
        if c["micro"] == 2:
            ab.weight_grad(ab.Act8(*s["x"][1], c["nin"], c["kind"]), s["dy"][1], out=dw, accumulate=True)
        return {"dw": dw}
    if op == "swiglu":
        if c["part"] == "train":
            y, ca, cb = ab.swiglu(s["a"], s["b"], checkpoint=c["kind"])
            da, db = ab.swiglu_backward(s["dy"], ca, cb)
            return {"y": y, "da": da, "db": db}
        ca, cb = ab.Act8(*s["ca"], c["cols"], c["kind"]), ab.Act8(*s["cb"], c["cols"], c["kind"])
        da, db, cy = ab.swiglu_backward(s["dy"], ca, cb, checkpoint=c["kind"])
        return {"y": ab.act8_unpack(cy, dt), "da": da, "db": db}
    if op == "rope":
        q, k = ab.rope(s["q"], s["k"], s["plan"], s["pos"], inverse=c["inverse"])
        return {"q": q, "k": k}
    q, k, cq, ck = ab.qk_norm_rope(s["q"], s["k"], s["gq"], s["gk"], s["plan"], s["pos"], eps=EPS, checkpoint=c["kind"])
    dq, dk, dgq, dgk = ab.qk_norm_rope_backward(s["dq"], s["dk"], cq, ck, s["gq"], s["gk"], s["plan"], s["pos"], eps=EPS)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dgq": dgq, "dgk": dgk}


def run(state):
    return _kernels(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    e = size[c["dtype"]]
    held = 1 + 1 / BLOCK
    if c["op"] == "checkpoint":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (2 * e + 2 * held), "flops": 4 * n}
    if c["op"] == "weight_grad":
        t, i, o = c["tokens"], c["nin"], c["nout"]
        return {"bytes": t * i * held + t * o * e + i * o * size[c["out"]] * (2 * c["micro"] - 1), "flops": 2 * t * i * o}
    if c["op"] == "swiglu":
        n = c["rows"] * c["cols"]
        fore, back = 3 * e + 2 * held, 3 * e + 2 * held
        if c["part"] == "train":
            return {"bytes": n * (fore + back), "flops": 30 * n}
        return {"bytes": n * (back + 2 * held + e), "flops": 25 * n}
    n = c["tokens"] * (c["hq"] + c["hk"]) * c["dim"]
    if c["op"] == "rope":
        return {"bytes": 2 * n * e + 4 * c["tokens"], "flops": 3 * n}
    return {"bytes": n * (4 * e + 2 * held) + 8 * c["tokens"], "flops": 30 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _e64(x, kind):
    """x in 64 bits -> the values of its checkpoint, from the definition."""
    rows, cols = x.shape
    full = torch.zeros(rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :cols] = x
    v = full.reshape(rows, -1, BLOCK)
    top = 448.0 if kind == "e4m3" else 127.0
    amax = v.abs().max(dim=2, keepdim=True).values
    k = torch.floor(torch.log2(amax.clamp(min=2.0 ** -126))) - 9
    for _ in range(5):  # up to the first power of two that holds the largest
        k = torch.where(amax > top * torch.exp2(k), k + 1, k)
    k = k.clamp(min=-126)
    u = v / torch.exp2(k)
    if kind == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
        u = torch.round(u / step) * step
    else:
        u = torch.round(u)
    return (u * torch.exp2(k)).reshape(rows, -1)[:, :cols]


def _held64(packed, kind, cols):
    """The 64-bit values of stored bytes, by their bit fields."""
    q, scale = packed
    b = q.to(torch.int64)
    if kind == "e4m3":
        ex, man = (b >> 3) & 15, (b & 7).double()
        mag = torch.where(ex == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * torch.exp2(ex.double() - 7))
        v = torch.where(b >= 128, -mag, mag)
    else:
        v = torch.where(b >= 128, b - 256, b).double()
    return (v * torch.repeat_interleave(torch.exp2(scale.double() - 127), BLOCK, dim=1))[:, :cols]


def _angles64(c, pos):
    a, r = _scaling(c["scaling"]), c["rot"]
    f = a.get("factor", 1.0)
    kind = a.get("scaling", "none")
    base = a["base"] * (f ** (r / (r - 2)) if kind == "base" else 1.0)
    w = np.array([base ** (-2.0 * j / r) for j in range(r // 2)])
    gain = 1.0
    if kind == "linear":
        w = w / f
    elif kind == "parts":
        gain = 1 + math.log(f) / 10
        edge = [r * math.log(a["original"] / (2 * math.pi * a[n])) / (2 * math.log(base)) for n in ("fast", "slow")]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
        part = np.clip((np.arange(r // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        w = w * (1 - part + part / f)
    elif kind == "wave":
        share = np.clip((a["original"] * w / (2 * math.pi) - a["slow"]) / (a["fast"] - a["slow"]), 0, 1)
        w = w * (share + (1 - share) / f)
    th = pos.to(torch.float64)[:, None, None] * torch.tensor(w, device=pos.device)
    return th, gain


def _rotate64(c, x, pos, back):
    th, gain = _angles64(c, pos)
    half = c["rot"] // 2
    j = torch.arange(half, device=x.device)
    i1, i2 = (j, j + half) if c["layout"] == "half" else (2 * j, 2 * j + 1)
    z = torch.complex(x[..., i1], x[..., i2]) * torch.polar(torch.full_like(th, gain), -th if back else th)
    y = x.clone()
    y[..., i1], y[..., i2] = z.real, z.imag
    y[pos < 0] = 0
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    d = lambda t: t.to(torch.float64)  # noqa: E731
    if op == "checkpoint":
        return {"x": _e64(d(s["x"]), c["kind"]), "scale": None}
    if op == "weight_grad":
        return {"dw": sum(_held64(x, c["kind"], c["nin"]).T.matmul(d(dy)) for x, dy in zip(s["x"], s["dy"]))}
    if op == "swiglu":
        a, b = (d(s["a"]), d(s["b"])) if c["part"] == "train" else (_held64(s["ca"], c["kind"], c["cols"]), _held64(s["cb"], c["kind"], c["cols"]))
        y = a / (1 + torch.exp(-a)) * b
        if c["part"] == "train":
            a, b = _e64(a, c["kind"]), _e64(b, c["kind"])
        else:
            y = _e64(d(y.to(TYPES[c["dtype"]])), c["kind"])
        e = torch.exp(-a)
        slope = 1 / (1 + e) + a * e / (1 + e) ** 2
        return {"y": y, "da": d(s["dy"]) * b * slope, "db": d(s["dy"]) * a / (1 + e)}
    if op == "rope":
        return {n: _rotate64(c, d(s[n]), s["pos"], c["inverse"]) for n in ("q", "k")}
    out = {}
    on = s["pos"] >= 0
    for n, gn in (("q", "gq"), ("k", "gk")):
        x, gain = d(s[n]), d(s[gn])
        out[n] = _rotate64(c, x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gain, s["pos"], False)
        x = _e64(x.reshape(x.shape[0], -1), c["kind"]).reshape(x.shape)
        u = _rotate64(c, d(s["d" + n]), s["pos"], True)
        rms = torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        dx = gain * u / rms - x * (gain * u * x).mean(-1, keepdim=True) / rms ** 3
        dx[~on] = 0
        out["d" + n] = dx
        out["dg" + n] = (u * x / rms).sum((0, 1))
    return out
