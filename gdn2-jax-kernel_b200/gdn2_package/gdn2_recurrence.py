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

import functools

import torch

from . import _lib
from . import gdn2_fwd as _fwd
from .gdn2_checkpoint import GROUP, _operand

INTERVAL = 64   # tokens between the states kept for the backward (GDN2_RECUR_INTERVAL)


class _Call:
    """Checked, device-resident operands of one call."""

    __slots__ = ("B", "T", "H", "D", "dev", "on_host", "code", "v", "w", "g", "h0", "dtypes",
                 "h0_dtype")

    def __init__(self, v, w, g, h0):
        if not (isinstance(v, torch.Tensor) and isinstance(w, torch.Tensor)
                and isinstance(g, torch.Tensor)):
            v, w, g = torch.as_tensor(v), torch.as_tensor(w), torch.as_tensor(g)
        shape = v.shape
        if len(shape) != 4 or w.shape != shape or g.shape != shape:
            raise _fwd.Gdn2ShapeError(
                f"inputs must share one (B, T, H, D) shape; got {tuple(shape)}")
        self.B, self.T, self.H, self.D = B, T, H, D = shape
        if D not in (64, 128, 256):
            raise _fwd.Gdn2ShapeError(f"head dim D={D} unsupported (64, 128 or 256)")
        if B * T * H == 0:
            raise _fwd.Gdn2ShapeError("empty problem")
        vt, wt, gt = self.dtypes = (v.dtype, w.dtype, g.dtype)
        if not (vt.is_floating_point and wt.is_floating_point and gt.is_floating_point):
            raise _fwd.Gdn2ShapeError("inputs must be floating point")
        gates = _fwd.GATES
        if gates not in ("activated", "raw"):
            raise _fwd.Gdn2ShapeError(f"GATES={gates!r}: 'activated' or 'raw'")
        self.on_host = not v.is_cuda
        self.dev = dev = (torch.device("cuda", torch.cuda.current_device()) if self.on_host
                          else v.device)
        bf16 = vt is wt is gt is torch.bfloat16
        cdt = torch.bfloat16 if bf16 else torch.float32
        self.code = (_lib.BF16 if bf16 else _lib.F32) | (_lib.GATES_RAW if gates == "raw" else 0)
        host = self.on_host
        self.v, self.w = _operand(v, dev, cdt, host), _operand(w, dev, cdt, host)
        self.g = _operand(g, dev, cdt, host)
        self.h0 = self.h0_dtype = None
        if h0 is not None:
            if not isinstance(h0, torch.Tensor):
                h0 = torch.as_tensor(h0)
            if h0.shape != (B, H, D):
                raise _fwd.Gdn2ShapeError(f"h0 must be {(B, H, D)}; got {tuple(h0.shape)}")
            self.h0_dtype = h0.dtype
            self.h0 = _operand(h0, dev, torch.float32, host)


class Gdn2RecurrenceResiduals:
    """What the backward of one forward needs: g, v and w or their int8 form
    (codes (2, B, T, H, D) and scales (2, B, T, H, D / 64)), and ``kept``, the
    state before every 64th token."""

    __slots__ = ("shape", "dev", "on_host", "code", "dtypes", "h0_dtype", "g", "v", "w", "int8",
                 "kept")

    def __init__(self, c, int8, kept):
        self.shape, self.dev, self.on_host = (c.B, c.T, c.H, c.D), c.dev, c.on_host
        self.code, self.dtypes, self.h0_dtype = c.code, c.dtypes, c.h0_dtype
        self.g, self.v, self.w = c.g, None if int8 else c.v, None if int8 else c.w
        self.int8, self.kept = int8, kept

    def without_tensors(self):
        """The sizes and types alone, for a copy that ``with_tensors`` completes."""
        return (self.shape, self.dev, self.on_host, self.code, self.dtypes, self.h0_dtype,
                self.int8 is not None)

    @classmethod
    def with_tensors(cls, rest, g, kept, *pair):
        self = cls.__new__(cls)
        (self.shape, self.dev, self.on_host, self.code, self.dtypes, self.h0_dtype, int8) = rest
        self.g, self.kept = g, kept
        self.int8 = pair if int8 else None
        self.v, self.w = (None, None) if int8 else pair
        return self

    @property
    def nbytes(self):
        ts = [self.g, self.kept, *(self.int8 or (self.v, self.w))]
        return sum(t.numel() * t.element_size() for t in ts)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _int8_pointers(packed):
    """Codes and scales of v, then of w."""
    if packed is None:
        return None, None, None, None
    codes, scales = packed
    c, s, n = codes.data_ptr(), scales.data_ptr(), codes.numel() // 2
    return c, s, c + n, s + n // GROUP * 4


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B, T, H, D):
    n = _lib.load().gdn2_recur_workspace_bytes(B, T, H, D)
    if n == 0:
        raise _fwd.Gdn2ShapeError("invalid sizes for the workspace")
    return n


def _workspace(shape, dev):
    """Scratch of one call; none where the sequence is one tile."""
    if shape[1] <= INTERVAL:
        return None, 0
    n = _workspace_bytes(*shape)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def _forward(c, keep, int8):
    lib = _lib.load()
    B, T, H, D, dev = c.B, c.T, c.H, c.D, c.dev
    o = torch.empty_like(c.v, dtype=torch.float32)
    hf = o.new_empty((B, H, D))
    kept = packed = None
    if keep:
        kept = o.new_empty((B, -(-T // INTERVAL), H, D))
        if int8:
            packed = (torch.empty((2, B, T, H, D), dtype=torch.int8, device=dev),
                      o.new_empty((2, B, T, H, D // GROUP)))
    ws, n = _workspace((B, T, H, D), dev)
    stream = _lib.raw_stream(dev.index)
    rc = _lib.on_device(dev.index, lib.gdn2_recur_fwd, c.code, c.v.data_ptr(), c.w.data_ptr(),
                        c.g.data_ptr(), _ptr(c.h0), o.data_ptr(), hf.data_ptr(), _ptr(kept),
                        *_int8_pointers(packed), _ptr(ws), n, B, T, H, D, stream)
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
    r, dev = residuals, residuals.dev
    B, T, H, D = r.shape
    if not isinstance(dout, torch.Tensor):
        dout = torch.as_tensor(dout)
    if dout.shape != r.shape:
        raise _fwd.Gdn2ShapeError(f"dout must be {r.shape}; got {tuple(dout.shape)}")
    do, dh = _operand(dout, dev, torch.float32, r.on_host), None
    if dh_final is not None:
        if not isinstance(dh_final, torch.Tensor):
            dh_final = torch.as_tensor(dh_final)
        if dh_final.shape != (B, H, D):
            raise _fwd.Gdn2ShapeError(f"dh_final must be {(B, H, D)}")
        dh = _operand(dh_final, dev, torch.float32, r.on_host)
    lib = _lib.load()
    dv, dw, dg = torch.empty_like(r.g), torch.empty_like(r.g), torch.empty_like(r.g)
    dh0 = do.new_empty((B, H, D))
    ws, n = _workspace(r.shape, dev)
    stream = _lib.raw_stream(dev.index)
    rc = _lib.on_device(dev.index, lib.gdn2_recur_bwd, r.code, _ptr(r.v), _ptr(r.w),
                        r.g.data_ptr(), *_int8_pointers(r.int8), r.kept.data_ptr(), do.data_ptr(),
                        _ptr(dh), dv.data_ptr(), dw.data_ptr(), dg.data_ptr(), dh0.data_ptr(),
                        _ptr(ws), n, B, T, H, D, stream)
    _lib.check(rc, "gdn2_linear_recurrence_backward")
    if ws is not None:
        _lib.check_status(ws, stream, "gdn2_linear_recurrence_backward", synced=r.on_host)
    out = [t if t.dtype is dt else t.to(dt)
           for t, dt in zip((dv, dw, dg, dh0), (*r.dtypes, r.h0_dtype or torch.float32))]
    return tuple(t.cpu() for t in out) if r.on_host else tuple(out)


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, v, w, g, h0, int8):
        ctx.set_materialize_grads(False)
        c = _Call(v, w, g, h0)
        o, hf, res = _forward(c, True, int8)
        # through save_for_backward, which notices inputs that change in place
        ctx.save_for_backward(res.g, res.kept, *(res.int8 or (res.v, res.w)))
        ctx.rest = res.without_tensors()
        return (o.cpu(), hf.cpu()) if c.on_host else (o, hf)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dh):
        if do is None and dh is None:
            return (None,) * 5
        r = Gdn2RecurrenceResiduals.with_tensors(ctx.rest, *ctx.saved_tensors)
        if do is None:
            do = torch.zeros(r.shape, dtype=torch.float32, device=r.dev)
        dv, dw, dg, dh0 = gdn2_linear_recurrence_backward(r, do, dh)
        return dv, dw, dg, None if r.h0_dtype is None else dh0, None


def gdn2_linear_recurrence_trainable(v, w, g, h0=None, checkpoint=None):
    """``gdn2_linear_recurrence`` with gradients for v, w, g and h0.

    The backward needs v, w, g and the states before every 64th token, not o.
    checkpoint="int8" keeps v and w in 8 bits (6.2 bytes a value with g in
    float32, against 12.1): the gradients are then those at the restored
    values."""
    return _Recurrence.apply(v, w, g, h0, _int8(checkpoint))
