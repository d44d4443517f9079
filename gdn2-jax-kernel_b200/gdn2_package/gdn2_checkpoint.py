"""int8 activation checkpoints (no counterpart in the reference, whose
custom_vjp keeps its inputs as they are, gdn2_pipeline.py:64-67).

``gdn2_checkpoint_pack(*tensors)`` keeps tensors in 8 bits and
``gdn2_checkpoint_unpack(kept)`` restores them.  Groups of 64 values along the
last axis share one float32 scale: code = rint(127 x / max|x|) with ties to
even, value = code * max|x| / 127, off by at most max|x| / 254.  A group with a
NaN or an infinity reads back as NaN throughout.

``gdn2_pallas_forward_trainable(..., checkpoint="int8")`` and
``gdn2_linear_recurrence_trainable(..., checkpoint="int8")`` use this form for
what their backward needs.  Log-decay gates are not kept in it: the rounding
of a log decay compounds over the sequence, that of the other inputs does not.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from . import gdn2_fwd as _fwd

GROUP = 64         # values that share a scale
_MAX_TENSORS = 8   # of one launch (GDN2_INT8_MAX_TENSORS)


def _aligned(t):
    """``t`` contiguous and on a 16-byte boundary."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class Gdn2Checkpoint:
    """Tensors in the int8 form: per tensor ``codes`` (its shape, int8) and
    ``scales`` (its shape with the last axis divided by 64, float32)."""

    __slots__ = ("codes", "scales", "dtypes", "on_host")

    def __init__(self, codes, scales, dtypes, on_host):
        self.codes, self.scales, self.dtypes, self.on_host = codes, scales, dtypes, on_host

    @property
    def nbytes(self):
        return sum(c.numel() for c in self.codes) + 4 * sum(s.numel() for s in self.scales)


def _pointers(ts):
    return (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


def _launches(dtypes, counts):
    """Indexes of the tensors of each launch: one type and size, at most eight."""
    sets = {}
    for i, key in enumerate(zip(dtypes, counts)):
        sets.setdefault(key, []).append(i)
    return [(key, at[i:i + _MAX_TENSORS]) for key, at in sets.items()
            for i in range(0, len(at), _MAX_TENSORS)]


def gdn2_checkpoint_pack(*tensors):
    """The int8 form of ``tensors`` (floating point, last axis a multiple of
    64) as a ``Gdn2Checkpoint``.  Not differentiable."""
    ts = [torch.as_tensor(t).detach() for t in tensors]
    if not ts:
        raise _fwd.Gdn2ShapeError("no tensors to pack")
    for t in ts:
        if not t.dtype.is_floating_point:
            raise _fwd.Gdn2ShapeError("inputs must be floating point")
        if t.dim() == 0 or t.shape[-1] % GROUP or t.numel() == 0:
            raise _fwd.Gdn2ShapeError(
                f"the last axis must be a positive multiple of {GROUP}; got {tuple(t.shape)}")
    on_host = ts[0].device.type != "cuda"
    dev = torch.device("cuda", torch.cuda.current_device()) if on_host else ts[0].device
    x = [_aligned(t.to(device=dev, dtype=t.dtype if t.dtype == torch.bfloat16 else torch.float32,
                       non_blocking=True)) for t in ts]
    codes = [torch.empty(t.shape, dtype=torch.int8, device=dev) for t in x]
    scales = [torch.empty((*t.shape[:-1], t.shape[-1] // GROUP), dtype=torch.float32, device=dev)
              for t in x]
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _fwd._stream(dev)
        for (dt, n), at in _launches([t.dtype for t in x], [t.numel() for t in x]):
            rc = lib.gdn2_int8_pack(_lib.BF16 if dt == torch.bfloat16 else _lib.F32, len(at),
                                    _pointers([x[i] for i in at]),
                                    _pointers([codes[i] for i in at]),
                                    _pointers([scales[i] for i in at]), n, stream)
            _lib.check(rc, "gdn2_checkpoint_pack")
    return Gdn2Checkpoint(codes, scales, [t.dtype for t in ts], on_host)


def gdn2_checkpoint_unpack(kept):
    """The tensors that ``kept`` holds, each in the type it was packed from."""
    dev = kept.codes[0].device
    out = [torch.empty(c.shape, dtype=dt if dt == torch.bfloat16 else torch.float32, device=dev)
           for c, dt in zip(kept.codes, kept.dtypes)]
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _fwd._stream(dev)
        for (dt, n), at in _launches([t.dtype for t in out], [t.numel() for t in out]):
            rc = lib.gdn2_int8_unpack(_lib.BF16 if dt == torch.bfloat16 else _lib.F32, len(at),
                                      _pointers([out[i] for i in at]),
                                      _pointers([kept.codes[i] for i in at]),
                                      _pointers([kept.scales[i] for i in at]), n, stream)
            _lib.check(rc, "gdn2_checkpoint_unpack")
    out = [t.to(dt) for t, dt in zip(out, kept.dtypes)]
    return tuple(t.cpu() for t in out) if kept.on_host else tuple(out)
