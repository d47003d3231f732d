"""Activation operators beside the optimizer step: 8-bit activation
checkpoints and the backward that reads them, and the norm and rotary
positions of queries and keys.

They produce what the step consumes: `weight_grad` writes (or adds) a
projection's gradient straight into its range of the FP16 gradient buffer
(`Optimizer.weight_grad` finds the range by the tensor's name), and the gains'
gradients of `qk_norm_rope_backward` go the same way.

Every function is asynchronous on torch's current stream of the tensors'
device, allocates what it returns (and workspaces) from torch's allocator, and
may be captured into a CUDA graph.  A tensor made on another stream has to be
ordered before the call, as for torch's own operators.  Everything goes
through libark_cuda.so; there is no autograd node and no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2, torch.int32: 3, torch.int64: 4}
KINDS = {"e4m3": 0, "int8": 1}
SCALINGS = {None: 0, "none": 0, "linear": 1, "base": 2, "parts": 3, "wave": 4}
PITCH, BLOCK = 128, 32


# ----------------------------------------------------------------- arguments
FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _float(t, what, types=FLOATS):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a CUDA torch.Tensor")
    if t.dtype not in types:
        raise TypeError(f"{what}: unsupported type {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what}: buffers must be CUDA tensors (device memory)")
    return t


def _rows(t, what, rows=None, cols=None, written=False, like=None):
    """(pointer, row stride) of a [rows, cols] tensor with contiguous rows."""
    _float(t, what)
    if t.dim() != 2:
        raise ValueError(f"{what}: expected [rows, cols], got {tuple(t.shape)}")
    if (rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{what}: expected [{rows}, {cols}], got {tuple(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{what}: expected {like.dtype} on {like.device}, got {t.dtype} on "
                         f"{t.device}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}: rows must be contiguous")
    ld = t.stride(0)
    if written and t.shape[0] > 1 and ld < t.shape[1]:
        raise ValueError(f"{what}: rows of an output may not overlap")
    return t.data_ptr(), ld


def _heads(t, what, like=None, shape=None):
    """ark_heads of a [tokens, heads, dim] tensor."""
    _float(t, what)
    if t.dim() != 3:
        raise ValueError(f"{what}: expected [tokens, heads, dim], got {tuple(t.shape)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected {tuple(shape)}, got {tuple(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{what}: expected {like.dtype} on {like.device}, got {t.dtype} on "
                         f"{t.device}")
    ts, hs, ds = t.stride()
    if t.shape[2] > 1 and ds != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    return _lib.Heads(t.data_ptr(), t.shape[1], ts, hs)


def _device(first, *others):
    """The tensors' one device."""
    d = first.device
    for t in others:
        if t is not None and t.device != d:
            raise ValueError(f"buffers on {d} and {t.device}")
    return d


class _on:
    """Makes a device the current one for a call, and gives the handle of
    torch's current stream there (without making a Stream object: 3 us)."""
    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _call(fn, *args):
    _lib.check(fn, getattr(_lib.lib(), fn)(*args))


# ----------------------------------------------------------------- 8-bit checkpoints
class Act8:
    """An 8-bit checkpoint of a [rows, cols] activation.

    data:  uint8 [rows, cols rounded up to 128], one byte per element;
    scale: uint8 [rows, data.shape[1] / 32], the power-of-two scale of 32
           columns as its exponent + 127 (255: the block held an infinity or
           a NaN and reads back as NaN).
    kind:  "e4m3" (4 significant bits at every size) or "int8" (a fixed step
           of 1/127 to 1/64 of the block's largest).
    """
    __slots__ = ("_data", "_scale", "_whole", "device", "rows", "cols", "kind", "c")

    def __init__(self, data, scale, cols, kind="e4m3"):
        cols = int(cols)
        pitch = -(-cols // PITCH) * PITCH
        if kind not in KINDS:
            raise ValueError(f"kind: expected one of {sorted(KINDS)}, got {kind!r}")
        for t, w, n in ((data, pitch, "data"), (scale, pitch // BLOCK, "scale")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8:
                raise TypeError(f"{n}: expected a uint8 CUDA tensor")
            if not t.is_cuda:
                raise ValueError(f"{n}: buffers must be CUDA tensors (device memory)")
            if t.dim() != 2 or t.shape[1] != w or t.shape[0] != data.shape[0] or not t.is_contiguous():
                raise ValueError(f"{n}: expected contiguous [rows, {w}], got {tuple(t.shape)}")
        if data.device != scale.device:
            raise ValueError("data and scale on different devices")
        self._data, self._scale, self._whole, self.device = data, scale, None, data.device
        self.rows, self.cols, self.kind = data.shape[0], cols, kind
        self.c = _lib.Act8(data.data_ptr(), scale.data_ptr(), self.rows, cols, KINDS[kind], 0)

    @classmethod
    def empty(cls, rows, cols, kind="e4m3", device="cuda"):
        """Room for a checkpoint (its contents are whatever was there), in one
        allocation; `data` and `scale` are views of it."""
        if kind not in KINDS:
            raise ValueError(f"kind: expected one of {sorted(KINDS)}, got {kind!r}")
        pitch = -(-cols // PITCH) * PITCH
        self = cls.__new__(cls)
        self._whole = torch.empty(rows * (pitch + pitch // BLOCK), dtype=torch.uint8, device=device)
        if not self._whole.is_cuda:
            raise ValueError("buffers must be CUDA tensors (device memory)")
        self._data = self._scale = None
        self.device = self._whole.device
        self.rows, self.cols, self.kind = rows, cols, kind
        p = self._whole.data_ptr()
        self.c = _lib.Act8(p, p + rows * pitch, rows, cols, KINDS[kind], 0)
        return self

    @property
    def pitch(self):
        return -(-self.cols // PITCH) * PITCH

    @property
    def data(self):
        if self._data is None:
            self._data = self._whole[: self.rows * self.pitch].view(self.rows, self.pitch)
        return self._data

    @property
    def scale(self):
        if self._scale is None:
            self._scale = self._whole[self.rows * self.pitch:].view(self.rows, self.pitch // BLOCK)
        return self._scale

    @property
    def nbytes(self):
        return self.rows * (self.pitch + self.pitch // BLOCK)


def _held(c, what, rows=None, cols=None):
    if not isinstance(c, Act8):
        raise TypeError(f"{what}: expected an Act8")
    if (rows is not None and c.rows != rows) or (cols is not None and c.cols != cols):
        raise ValueError(f"{what}: expected a checkpoint of [{rows}, {cols}], got "
                         f"[{c.rows}, {c.cols}]")
    return ctypes.byref(c.c)


def act8_pack(x, kind="e4m3", out=None) -> Act8:
    """Checkpoint x [rows, cols] (FP16, BF16 or FP32) in 8 bits."""
    p, ld = _rows(x, "x")
    with _on(x.device) as s:
        if out is None:
            out = Act8.empty(x.shape[0], x.shape[1], kind, x.device)
        else:
            _held(out, "out", *x.shape)
            _device(x, out)
        _call("ark_cuda_act8_pack", p, TYPES[x.dtype], ld, ctypes.byref(out.c), s)
    return out


def act8_unpack(c, dtype=torch.float16, out=None):
    """The activation that a checkpoint stands for; a finite value that the
    type cannot hold saturates at its largest."""
    h = _held(c, "checkpoint")
    with _on(c.device) as s:
        if out is None:
            if dtype not in FLOATS:
                raise TypeError(f"unsupported type {dtype}")
            out = torch.empty((c.rows, c.cols), dtype=dtype, device=c.device)
            p, ld = out.data_ptr(), c.cols
        else:
            p, ld = _rows(out, "out", c.rows, c.cols, written=True)
            _device(c, out)
        _call("ark_cuda_act8_unpack", h, p, TYPES[out.dtype], ld, s)
    return out


def weight_grad(x, dy, out=None, accumulate=False, dtype=None):
    """dW [in, out_features] = X^T dY of y = x W, X [tokens, in] read from its
    checkpoint, dY [tokens, out_features] FP16 or BF16.

    out: where to write (FP16, BF16 or FP32; for example a range of the
         gradient buffer viewed as [in, out_features]); default: a new tensor
         of `dtype` (default: dY's).
    accumulate: add to what is in `out`.
    """
    hx = _held(x, "x")
    _float(dy, "dy", (torch.float16, torch.bfloat16))
    p, ld = _rows(dy, "dy", rows=x.rows)
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    n = dy.shape[1]
    with _on(_device(x, dy, out)) as s:
        if out is None:
            if dtype is not None and dtype not in FLOATS:
                raise TypeError(f"unsupported type {dtype}")
            out = torch.empty((x.cols, n), dtype=dtype or dy.dtype, device=dy.device)
            po, ldo = out.data_ptr(), n
        else:
            if dtype is not None and out.dtype != dtype:
                raise ValueError(f"out: expected {dtype}, got {out.dtype}")
            po, ldo = _rows(out, "out", x.cols, n, written=True)
        need = _lib.lib().ark_cuda_weight_grad_workspace(hx, p, ld, n, po, TYPES[out.dtype],
                                                                  ldo)
        ws = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
        _call("ark_cuda_weight_grad", hx, p, TYPES[dy.dtype], ld, n, po, TYPES[out.dtype], ldo,
              1 if accumulate else 0, ws.data_ptr() if need else None, need, s)
    return out


# ----------------------------------------------------------------- SwiGLU
def swiglu(a, b, checkpoint=None, out=None):
    """y = silu(a) * b for a, b [rows, cols].  With checkpoint ("e4m3" or
    "int8") returns (y, Act8 of a, Act8 of b), made in the same pass.  out may
    be a or b."""
    pa, la = _rows(a, "a")
    pb, lb = _rows(b, "b", a.shape[0], a.shape[1], like=a)
    with _on(a.device) as s:
        if out is None:
            out = torch.empty(a.shape, dtype=a.dtype, device=a.device)
            py, ly = out.data_ptr(), a.shape[1]
        else:
            py, ly = _rows(out, "out", a.shape[0], a.shape[1], written=True, like=a)
        ca = cb = ha = hb = None
        if checkpoint is not None:
            ca, cb = (Act8.empty(a.shape[0], a.shape[1], checkpoint, a.device) for _ in range(2))
            ha, hb = ctypes.byref(ca.c), ctypes.byref(cb.c)
        _call("ark_cuda_swiglu", pa, la, pb, lb, TYPES[a.dtype], a.shape[0], a.shape[1], py, ly, ha,
              hb, s)
    return out if checkpoint is None else (out, ca, cb)


def swiglu_backward(dy, ca, cb, checkpoint=None, out=None):
    """(da, db) of swiglu from the checkpoints of a and b.  With checkpoint,
    returns (da, db, Act8 of the remade product) for the weight gradient of
    the projection that reads it; its kind is that of ca.  out: (da, db)."""
    ha = _held(ca, "ca")
    hb = _held(cb, "cb", ca.rows, ca.cols)
    if cb.kind != ca.kind or (checkpoint is not None and checkpoint != ca.kind):
        raise ValueError("checkpoints of one call are of one kind")
    pg, lg = _rows(dy, "dy", ca.rows, ca.cols)
    with _on(_device(dy, ca, cb)) as s:
        if out is None:
            da = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
            db = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
            pa, pb, la = da.data_ptr(), db.data_ptr(), ca.cols
            lb = la
        else:
            da, db = out
            pa, la = _rows(da, "da", ca.rows, ca.cols, written=True, like=dy)
            pb, lb = _rows(db, "db", ca.rows, ca.cols, written=True, like=dy)
        cy = Act8.empty(ca.rows, ca.cols, ca.kind, dy.device) if checkpoint is not None else None
        _call("ark_cuda_swiglu_backward", pg, lg, TYPES[dy.dtype], ha, hb, pa, la, pb, lb,
              ctypes.byref(cy.c) if cy is not None else None, s)
    return (da, db) if checkpoint is None else (da, db, cy)


# ----------------------------------------------------------------- rotary positions
class RopePlan:
    """The rotation of the first rotary_dim elements of each head.

    layout:  "half" (pairs i, i + rotary_dim/2) or "interleaved" (2i, 2i + 1).
    base:    pair i turns base^(-2i/rotary_dim) radians per position.
    scaling: for contexts longer than the trained one: None; "linear" (every
             frequency / factor); "base" (base * factor^(d/(d-2))); "parts"
             (frequencies above `fast` turns over the `original` length kept,
             below `slow` divided by factor, a ramp over the pairs between, and
             cos and sin times 0.1 ln(factor) + 1); "wave" (the same ends, a
             ramp over the number of turns).
    Host memory only: made once, usable on every device and in graphs.
    """
    __slots__ = ("c", "rotary_dim", "layout")

    def __init__(self, rotary_dim, base=10000.0, layout="half", scaling=None, factor=1.0,
                 original=0.0, fast=32.0, slow=1.0):
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout: expected 'half' or 'interleaved', got {layout!r}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling: expected one of {[k for k in SCALINGS if k]}, got {scaling!r}")
        self.rotary_dim, self.layout = int(rotary_dim), layout
        if not 2 <= self.rotary_dim <= _lib.ARK_ROPE_MAX_DIM or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim: expected an even number from 2 to "
                             f"{_lib.ARK_ROPE_MAX_DIM}, got {rotary_dim}")
        self.c = _lib.RopePlan()
        _call("ark_cuda_rope_plan", ctypes.byref(self.c), self.rotary_dim,
              1 if layout == "interleaved" else 0, base, SCALINGS[scaling], factor, original, fast,
              slow)

    @property
    def gain(self):
        return self.c.gain

    def frequencies(self):
        """Radians per position of each pair."""
        return [t * (6.283185307179586 / 2.0 ** 64) for t in self.c.turns[: self.rotary_dim // 2]]


def _positions(positions, tokens, seq_len, device):
    """(pointer, type, seq_len)."""
    if positions is None:
        n = tokens if seq_len is None else int(seq_len)
        if n < 0 or (n == 0 and tokens):
            raise ValueError("seq_len: expected a positive length")
        return None, 0, max(n, 1)
    if seq_len is not None:
        raise ValueError("positions or seq_len, not both")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions: expected an int32 or int64 CUDA tensor")
    if positions.device != device:
        raise ValueError(f"positions: expected on {device}, got {positions.device}")
    if positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"positions: expected contiguous [{tokens}], got {tuple(positions.shape)}")
    return positions.data_ptr(), TYPES[positions.dtype], 0


def _qk(q, k, plan, out, names=("q", "k")):
    """The four ark_heads of a call and its outputs."""
    if not isinstance(plan, RopePlan):
        raise TypeError("plan: expected a RopePlan")
    hq = _heads(q, names[0])
    t, h, d = q.shape
    if d < plan.rotary_dim:
        raise ValueError(f"{names[0]}: heads of {d} are shorter than the rotated {plan.rotary_dim}")
    if d > _lib.ARK_ROPE_MAX_DIM:
        raise ValueError(f"{names[0]}: heads of {d}: at most {_lib.ARK_ROPE_MAX_DIM} are supported")
    hk = hp = ok = None
    if k is not None:
        hk = _heads(k, names[1], like=q)
        if k.shape[0] != t or k.shape[2] != d:
            raise ValueError(f"{names[1]}: expected [{t}, heads, {d}], got {tuple(k.shape)}")
    if out is None:
        oq = torch.empty((t, h, d), dtype=q.dtype, device=q.device)
        ho = _lib.Heads(oq.data_ptr(), h, h * d, d)
        if k is not None:
            h = k.shape[1]
            ok = torch.empty((t, h, d), dtype=q.dtype, device=q.device)
            hp = _lib.Heads(ok.data_ptr(), h, h * d, d)
    else:
        oq, ok = out
        ho = _heads(oq, "out " + names[0], like=q, shape=q.shape)
        if k is not None:
            hp = _heads(ok, "out " + names[1], like=q, shape=k.shape)
        elif ok is not None:
            raise ValueError(f"out {names[1]}: there is no {names[1]}")
    byref = ctypes.byref
    return (byref(hq), hk and byref(hk), byref(ho), hp and byref(hp)), oq, ok


def rope(q, k, plan, positions=None, seq_len=None, inverse=False, out=None):
    """Rotate q [tokens, heads, dim] and k [tokens, kv heads, dim] (or None).

    positions: int32 / int64 [tokens], any non-negative value; a negative one
               marks a padding token, whose outputs are zero.  None: token
               index modulo seq_len (default: one sequence).
    inverse:   the opposite rotation, which is the backward.
    out:       (q, k) to write to, for example q and k themselves.
    Any strides with contiguous heads' elements.  Returns (q, k).
    """
    with _on(_float(q, "q").device) as s:
        ref, oq, ok = _qk(q, k, plan, out)
        pos = _positions(positions, q.shape[0], seq_len, q.device)
        _call("ark_cuda_rope", ctypes.byref(plan.c), *ref, TYPES[q.dtype], q.shape[0], q.shape[2],
              *pos, 1 if inverse else 0, s)
    return oq, ok


def _gain(g, what, dim, device):
    _float(g, what)
    if g.shape != (dim,) or not g.is_contiguous() or g.device != device:
        raise ValueError(f"{what}: expected contiguous [{dim}] on {device}, got {tuple(g.shape)} on "
                         f"{g.device}")
    return g.data_ptr()


def _gains(q, k, gain_q, gain_k):
    pq = _gain(gain_q, "gain_q", q.shape[2], q.device)
    if k is None:
        return pq, None, TYPES[gain_q.dtype]
    pk = _gain(gain_k, "gain_k", q.shape[2], q.device)
    if gain_k.dtype != gain_q.dtype:
        raise ValueError("gain_q and gain_k are of different types")
    return pq, pk, TYPES[gain_q.dtype]


def qk_norm_rope(q, k, gain_q, gain_k, plan, positions=None, seq_len=None, eps=1e-6,
                 checkpoint=None, out=None):
    """RMS norm of each head of q and k (k may be None) with its gain [dim],
    then the rotation, in one pass.  With checkpoint ("e4m3" or "int8") q and k
    as they come in are checkpointed too: returns (q, k, Act8 of q, Act8 of k),
    each of [tokens, heads * dim], else (q, k)."""
    with _on(_float(q, "q").device) as s:
        ref, oq, ok = _qk(q, k, plan, out)
        g = _gains(q, k, gain_q, gain_k)
        pos = _positions(positions, q.shape[0], seq_len, q.device)
        cq = ck = None
        if checkpoint is not None:
            cq = Act8.empty(q.shape[0], q.shape[1] * q.shape[2], checkpoint, q.device)
            if k is not None:
                ck = Act8.empty(k.shape[0], k.shape[1] * k.shape[2], checkpoint, q.device)
        _call("ark_cuda_qk_norm_rope", ctypes.byref(plan.c), *ref, TYPES[q.dtype], q.shape[0],
              q.shape[2], *g, eps, *pos, ctypes.byref(cq.c) if cq is not None else None,
              ctypes.byref(ck.c) if ck is not None else None, s)
    return (oq, ok) if checkpoint is None else (oq, ok, cq, ck)


def qk_norm_rope_backward(dq, dk, q, k, gain_q, gain_k, plan, positions=None, seq_len=None,
                          eps=1e-6, out=None, out_gains=None, accumulate=False):
    """Backward of qk_norm_rope: (dq, dk, dgain_q, dgain_k).

    dq, dk:  gradients of the outputs (dk may be None).
    q, k:    the inputs' checkpoints (Act8), or the inputs themselves.
    out:     (dq, dk) to write to, for example dq and dk themselves.
    out_gains: (dgain_q, dgain_k) [dim] to write to, for example ranges of the
             gradient buffer; default: new tensors of the gains' type.
    accumulate: add the gains' gradients to what is in out_gains.
    """
    if accumulate and out_gains is None:
        raise ValueError("accumulate needs out_gains")
    with _on(_float(dq, "dq").device) as s:
        ref, oq, ok = _qk(dq, dk, plan, out, ("dq", "dk"))
        g = _gains(dq, dk, gain_q, gain_k)
        t, dim = dq.shape[0], dq.shape[2]
        pos = _positions(positions, t, seq_len, dq.device)
        src = [None] * 4
        for i, (d, x, n) in enumerate(((dq, q, "q"), (dk, k, "k"))):
            if d is None:
                continue
            if isinstance(x, Act8):
                _device(d, x)
                src[i] = _held(x, n, t, d.shape[1] * dim)
            else:
                src[2 + i] = ctypes.byref(_heads(x, n, like=dq, shape=d.shape))
        if dk is not None and ((src[0] is None) != (src[1] is None)
                               or (src[0] is not None and q.kind != k.kind)):
            raise ValueError("q and k: both checkpoints of one kind, or both tensors")
        if out_gains is None:
            out_gains = (torch.empty_like(gain_q), torch.empty_like(gain_k) if dk is not None else None)
        gq, gk = out_gains
        pq = _gain(gq, "dgain_q", dim, dq.device)
        pk = _gain(gk, "dgain_k", dim, dq.device) if dk is not None else None
        if dk is not None and gk.dtype != gq.dtype:
            raise ValueError("dgain_q and dgain_k are of different types")
        need = _lib.lib().ark_cuda_qk_norm_rope_workspace(dim)
        ws = torch.empty(need // 4, dtype=torch.float32, device=dq.device)
        _call("ark_cuda_qk_norm_rope_backward", ctypes.byref(plan.c), *ref, TYPES[dq.dtype], t, dim,
              *src, *g, eps, *pos, pq, pk, TYPES[gq.dtype], 1 if accumulate else 0, ws.data_ptr(),
              need, s)
    return oq, ok, gq, gk
