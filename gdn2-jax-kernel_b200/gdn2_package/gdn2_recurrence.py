"""Gated linear recurrence (no counterpart in the reference): the diagonal
member of the family GDN-2 belongs to, on its layouts and gates,

    h_t = e^{g_t} h_{t-1} + w_t v_t   per channel,   o_t = h_t.

``gdn2_linear_recurrence(v, w, g, h0=None)`` takes (B, T, H, D) float32 or
bfloat16 tensors (T from one token up, D 64, 128 or 256) and a state (B, H, D),
and returns (o, h_final), both float32.  One call with T = 1 is a decode step.
``gdn2_linear_recurrence_trainable`` is differentiable w.r.t. v, w, g and h0;
``checkpoint="int8"`` keeps v and w in 8 bits for the backward.
``gdn2_linear_recurrence_with_residuals`` / ``_backward`` are the same two
passes without autograd, e.g. to capture a step into a CUDA graph.

``gdn2_fwd.GATES`` applies: with "raw", w and g are pre-activations.  The gates
may be any value up to 0, -inf included (the state restarts there).  No
sanitiser acts: a clip inside the recurrence would make it serial.
"""
from __future__ import annotations

import torch

from . import _lib
from . import gdn2_fwd as _fwd
from .gdn2_checkpoint import GROUP, _aligned

INTERVAL = 64   # tokens between the states kept for the backward (GDN2_RECUR_INTERVAL)


class _Call:
    """Checked, device-resident operands of one call."""

    __slots__ = ("B", "T", "H", "D", "dev", "on_host", "code", "v", "w", "g", "h0", "dtypes",
                 "h0_dtype")

    def __init__(self, v, w, g, h0):
        ts = (v, w, g)
        if not all(isinstance(t, torch.Tensor) for t in ts):
            ts = tuple(torch.as_tensor(t) for t in ts)
        shape = tuple(ts[0].shape)
        if len(shape) != 4 or any(tuple(t.shape) != shape for t in ts):
            raise _fwd.Gdn2ShapeError(f"inputs must share one (B, T, H, D) shape; got {shape}")
        self.B, self.T, self.H, self.D = B, T, H, D = shape
        if D not in (64, 128, 256):
            raise _fwd.Gdn2ShapeError(f"head dim D={D} unsupported (64, 128 or 256)")
        if B * T * H == 0:
            raise _fwd.Gdn2ShapeError("empty problem")
        self.dtypes = tuple(t.dtype for t in ts)
        if any(not dt.is_floating_point for dt in self.dtypes):
            raise _fwd.Gdn2ShapeError("inputs must be floating point")
        if _fwd.GATES not in ("activated", "raw"):
            raise _fwd.Gdn2ShapeError(f"GATES={_fwd.GATES!r}: 'activated' or 'raw'")
        self.on_host = ts[0].device.type != "cuda"
        self.dev = dev = (torch.device("cuda", torch.cuda.current_device()) if self.on_host
                          else ts[0].device)
        bf16 = all(dt == torch.bfloat16 for dt in self.dtypes)
        cdt = torch.bfloat16 if bf16 else torch.float32
        self.code = (_lib.BF16 if bf16 else _lib.F32) | (_lib.GATES_RAW if _fwd.GATES == "raw" else 0)
        self.v, self.w, self.g = (_aligned(t.to(device=dev, dtype=cdt, non_blocking=True))
                                  for t in ts)
        self.h0 = self.h0_dtype = None
        if h0 is not None:
            h0 = torch.as_tensor(h0)
            if tuple(h0.shape) != (B, H, D):
                raise _fwd.Gdn2ShapeError(f"h0 must be {(B, H, D)}; got {tuple(h0.shape)}")
            self.h0_dtype = h0.dtype
            self.h0 = _aligned(h0.to(device=dev, dtype=torch.float32, non_blocking=True))


class Gdn2RecurrenceResiduals:
    """What the backward of one forward needs: g, v and w or their int8 form,
    and the state before every 64th token."""

    __slots__ = ("B", "T", "H", "D", "dev", "on_host", "code", "dtypes", "h0_dtype", "g", "v", "w",
                 "int8", "kept")

    def __init__(self, c, int8, kept):
        for n in ("B", "T", "H", "D", "dev", "on_host", "code", "dtypes", "h0_dtype", "g"):
            setattr(self, n, getattr(c, n))
        self.v, self.w = (None, None) if int8 else (c.v, c.w)
        self.int8, self.kept = int8, kept   # int8: (v codes, v scales, w codes, w scales)

    @property
    def nbytes(self):
        ts = [self.g, self.kept, *(self.int8 if self.int8 else (self.v, self.w))]
        return sum(t.numel() * t.element_size() for t in ts)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _workspace(lib, c):
    """Scratch of one call; none where the sequence is one tile."""
    if c.T <= INTERVAL:
        return None, 0
    n = lib.gdn2_recur_workspace_bytes(c.B, c.T, c.H, c.D)
    if n == 0:
        raise _fwd.Gdn2ShapeError("invalid sizes for the workspace")
    return torch.empty(n, dtype=torch.uint8, device=c.dev), n


def _forward(c, keep, int8):
    lib = _lib.load()
    B, T, H, D, dev = c.B, c.T, c.H, c.D, c.dev
    o = torch.empty((B, T, H, D), dtype=torch.float32, device=dev)
    hf = torch.empty((B, H, D), dtype=torch.float32, device=dev)
    kept = packed = None
    if keep:
        kept = torch.empty((B, -(-T // INTERVAL), H, D), dtype=torch.float32, device=dev)
        if int8:
            packed = tuple(torch.empty(s, dtype=dt, device=dev) for _ in range(2)
                           for s, dt in (((B, T, H, D), torch.int8),
                                         ((B, T, H, D // GROUP), torch.float32)))
    ws, n = _workspace(lib, c)
    with torch.cuda.device(dev):
        stream = _fwd._stream(dev)
        rc = lib.gdn2_recur_fwd(c.code, c.v.data_ptr(), c.w.data_ptr(), c.g.data_ptr(), _ptr(c.h0),
                                o.data_ptr(), hf.data_ptr(), _ptr(kept),
                                *(map(_ptr, packed) if packed else (None,) * 4), _ptr(ws), n,
                                B, T, H, D, stream)
        _lib.check(rc, "gdn2_linear_recurrence")
        if ws is not None:
            _lib.check_status(ws, stream, "gdn2_linear_recurrence", synced=c.on_host)
    return o, hf, (Gdn2RecurrenceResiduals(c, packed, kept) if keep else None)


def _int8(checkpoint):
    if checkpoint not in (None, "int8"):
        raise _fwd.Gdn2ShapeError(f"checkpoint={checkpoint!r}: None or 'int8'")
    return checkpoint == "int8"


def gdn2_linear_recurrence(v, w, g, h0=None):
    """o (B, T, H, D) and h_final (B, H, D), float32."""
    c = _Call(v, w, g, h0)
    o, hf, _ = _forward(c, False, False)
    return (o.cpu(), hf.cpu()) if c.on_host else (o, hf)


def gdn2_linear_recurrence_with_residuals(v, w, g, h0=None, checkpoint=None):
    """(o, h_final, residuals); ``gdn2_linear_recurrence_backward`` takes the
    residuals.  They share v, w and g with the caller where those need no copy
    (with checkpoint="int8" only g)."""
    c = _Call(v, w, g, h0)
    o, hf, res = _forward(c, True, _int8(checkpoint))
    return (o.cpu(), hf.cpu(), res) if c.on_host else (o, hf, res)


def gdn2_linear_recurrence_backward(residuals, dout, dh_final=None):
    """(dv, dw, dg, dh0) for cotangents of (o, h_final), each in its input's
    type (dh0 float32 where h0 was not given).  With int8 residuals these are the
    gradients at the restored v and w, from the forward's states every 64
    tokens."""
    r = residuals
    shape = (r.B, r.T, r.H, r.D)
    f32 = dict(device=r.dev, dtype=torch.float32, non_blocking=True)
    dout = torch.as_tensor(dout)
    if tuple(dout.shape) != shape:
        raise _fwd.Gdn2ShapeError(f"dout must be {shape}; got {tuple(dout.shape)}")
    do = _aligned(dout.to(**f32))
    dh = None
    if dh_final is not None:
        dh_final = torch.as_tensor(dh_final)
        if tuple(dh_final.shape) != (r.B, r.H, r.D):
            raise _fwd.Gdn2ShapeError(f"dh_final must be {(r.B, r.H, r.D)}")
        dh = _aligned(dh_final.to(**f32))
    lib = _lib.load()
    dv, dw, dg = (torch.empty(shape, dtype=r.g.dtype, device=r.dev) for _ in range(3))
    dh0 = torch.empty((r.B, r.H, r.D), dtype=torch.float32, device=r.dev)
    ws, n = _workspace(lib, r)
    with torch.cuda.device(r.dev):
        stream = _fwd._stream(r.dev)
        rc = lib.gdn2_recur_bwd(r.code, _ptr(r.v), _ptr(r.w), r.g.data_ptr(),
                                *(map(_ptr, r.int8) if r.int8 else (None,) * 4),
                                r.kept.data_ptr(), do.data_ptr(), _ptr(dh), dv.data_ptr(),
                                dw.data_ptr(), dg.data_ptr(), dh0.data_ptr(), _ptr(ws), n,
                                r.B, r.T, r.H, r.D, stream)
        _lib.check(rc, "gdn2_linear_recurrence_backward")
        if ws is not None:
            _lib.check_status(ws, stream, "gdn2_linear_recurrence_backward", synced=r.on_host)
    out = [t.to(dt) for t, dt in zip((dv, dw, dg), r.dtypes)]
    out.append(dh0 if r.h0_dtype is None else dh0.to(r.h0_dtype))
    return tuple(t.cpu() for t in out) if r.on_host else tuple(out)


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, v, w, g, h0, int8):
        ctx.set_materialize_grads(False)
        c = _Call(v, w, g, h0)
        o, hf, res = _forward(c, True, int8)
        # through save_for_backward, which notices inputs that change in place
        ctx.save_for_backward(res.g, res.kept, *(res.int8 if int8 else (res.v, res.w)))
        res.g = res.kept = res.int8 = res.v = res.w = None
        ctx.res, ctx.int8 = res, int8
        return (o.cpu(), hf.cpu()) if c.on_host else (o, hf)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dh):
        if do is None and dh is None:
            return (None,) * 5
        saved = ctx.saved_tensors
        c, r = ctx.res, Gdn2RecurrenceResiduals.__new__(Gdn2RecurrenceResiduals)
        for n in ("B", "T", "H", "D", "dev", "on_host", "code", "dtypes", "h0_dtype"):
            setattr(r, n, getattr(c, n))
        r.g, r.kept = saved[:2]
        r.int8 = tuple(saved[2:]) if ctx.int8 else None
        r.v, r.w = (None, None) if ctx.int8 else saved[2:]
        if do is None:
            do = torch.zeros((r.B, r.T, r.H, r.D), dtype=torch.float32, device=r.dev)
        dv, dw, dg, dh0 = gdn2_linear_recurrence_backward(r, do, dh)
        return dv, dw, dg, None if r.h0_dtype is None else dh0, None


def gdn2_linear_recurrence_trainable(v, w, g, h0=None, checkpoint=None):
    """``gdn2_linear_recurrence`` with gradients for v, w, g and h0.

    The backward needs v, w, g and the states before every 64th token, not o.
    checkpoint="int8" keeps v and w in 8 bits (6.2 bytes a value with g in
    float32, against 12.1): the gradients are then those at the restored
    values."""
    return _Recurrence.apply(v, w, g, h0, _int8(checkpoint))
