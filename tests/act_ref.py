"""The activation operators in 64 bits, on the CPU, from their definitions."""
import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half a step among the type's subnormals
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def e4m3_values():
    """The 256 values of the format by byte (NaN at 0x7f and 0xff)."""
    out = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = math.nan if (b & 127) == 127 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out.append(-v if b >= 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def pack(x, kind):
    """x [rows, cols] -> (bytes [rows, pitch], scale [rows, pitch / 32]) by definition."""
    rows, cols = x.shape
    pitch = -(-cols // 128) * 128
    v = torch.zeros(rows, pitch, dtype=torch.float64)
    v[:, :cols] = x.double()
    v = v.view(rows, pitch // 32, 32)
    amax = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    k = torch.full(amax.shape, -126, dtype=torch.int64)
    for e in range(-126, 122):   # the smallest power of two that holds the largest
        k = torch.where((amax > TOP[kind] * 2.0 ** e) & ~bad, torch.full_like(k, e + 1), k)
    u = v / torch.exp2(k.double()).unsqueeze(2)
    u = torch.where(bad.unsqueeze(2), torch.zeros_like(u), u)
    if kind == "int8":
        q = torch.round(u).to(torch.int64) & 255
    else:
        table = e4m3_values()
        pos = table[:127]
        hi = torch.searchsorted(pos, u.abs()).clamp(max=126)   # first value >= |u|
        lo = (hi - 1).clamp(min=0)
        up, dn = pos[hi] - u.abs(), u.abs() - pos[lo]
        code = torch.where((up < dn) | ((up == dn) & (hi % 2 == 0)), hi, lo)
        q = code + 128 * torch.signbit(u).long()
    s = torch.where(bad, torch.full_like(k, 255), k + 127)
    return q.reshape(rows, pitch).to(torch.uint8), s.to(torch.uint8)


def values(data, scale, cols, kind):
    """What stored bytes stand for."""
    b = data.cpu().long()
    v = e4m3_values()[b] if kind == "e4m3" else torch.where(b > 127, b - 256, b).double()
    s = torch.exp2(scale.cpu().double() - 127)
    s = torch.where(scale.cpu() == 255, torch.full_like(s, math.nan), s)
    return (v * s.repeat_interleave(32, 1))[:, :cols]


def through(x, kind):
    return values(*pack(x, kind), x.shape[1], kind)


def silu_parts(a):
    s = 1 / (1 + torch.exp(-a))
    return s, a * s, s * (1 + a * (1 - s))


def frequencies(rot, base=10000.0, scaling=None, factor=1.0, original=0.0, fast=32.0, slow=1.0):
    """(radians per position, factor on cos and sin)."""
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    w = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    gain = 1.0
    if scaling == "linear":
        w = [x / factor for x in w]
    if scaling == "parts":
        gain = 0.1 * math.log(factor) + 1
        at = [rot * math.log(original / (2 * math.pi * t)) / (2 * math.log(base)) for t in (fast, slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        w = [x * (1 - r) + x / factor * r for x, r in zip(w, ramp)]
    if scaling == "wave":
        keep = [min(max((original * x / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0) for x in w]
        w = [x * k + x / factor * (1 - k) for x, k in zip(w, keep)]
    return torch.tensor(w, dtype=torch.float64), gain


def rotate(x, pos, freq, gain, layout, inverse=False):
    """x [tokens, heads, dim] in 64 bits; padding tokens become zero."""
    half = freq.numel()
    th = pos.double().view(-1, 1, 1) * freq
    c, s = torch.cos(th) * gain, torch.sin(th) * gain * (-1 if inverse else 1)
    j = torch.arange(half)
    i1, i2 = (j, j + half) if layout == "half" else (2 * j, 2 * j + 1)
    y = x.clone()
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    return torch.where((pos >= 0).view(-1, 1, 1), y, torch.zeros_like(y))


def norm(x, gain, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * gain


def norm_back(x, u, gain, eps, live):
    """(dx, dgain, magnitude of dx's terms, magnitude of dgain's terms)."""
    x = torch.where(live.view(-1, 1, 1), x, torch.zeros_like(x))
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    h, gu = x * r, u * gain
    dx = r * (gu - h * (gu * h).mean(-1, keepdim=True))
    size = r * (gu.abs() + h.abs() * (gu * h).abs().mean(-1, keepdim=True))
    return dx * live.view(-1, 1, 1), (u * h).sum((0, 1)), size, (u * h).abs().sum((0, 1))
