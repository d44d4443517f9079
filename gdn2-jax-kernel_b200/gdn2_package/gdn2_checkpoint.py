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


def _operand(t, dev, dtype, waits=False):
    """``t`` on ``dev`` in ``dtype``, contiguous and on a 16-byte boundary.

    A copy from pinned host memory is waited for, so that the caller may refill it
    after the call, unless the call ``waits`` for its stream anyway (it returns
    results on the host) or is being captured (its replays read the memory)."""
    if t.dtype is not dtype or t.device != dev:
        t = t.to(device=dev, dtype=dtype, non_blocking=waits or t.is_cuda
                 or torch.cuda.is_current_stream_capturing())
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class Gdn2Checkpoint:
    """Tensors in the int8 form.  ``codes[i]`` (the tensor's shape, int8) and
    ``scales[i]`` (its shape with the last axis divided by 64, float32) are views
    of one buffer each per launch (``buffers``: (indexes, codes, scales))."""

    __slots__ = ("buffers", "shapes", "dtypes", "on_host")

    def __init__(self, buffers, shapes, dtypes, on_host):
        self.buffers, self.shapes, self.dtypes, self.on_host = buffers, shapes, dtypes, on_host

    def _views(self, which, last):
        out = [None] * len(self.shapes)
        for entry in self.buffers:
            for j, i in enumerate(entry[0]):
                s = self.shapes[i]
                out[i] = entry[which][j].view((*s[:-1], s[-1] // last))
        return out

    codes = property(lambda self: self._views(1, 1))
    scales = property(lambda self: self._views(2, GROUP))

    @property
    def nbytes(self):
        return sum(c.numel() + 4 * s.numel() for _, c, s in self.buffers)


_ARRAYS = [ctypes.c_void_p * n for n in range(_MAX_TENSORS + 1)]


def _launches(dtypes, counts):
    """Indexes of the tensors of each launch: one type and size, at most eight."""
    if len(dtypes) <= _MAX_TENSORS and len(set(dtypes)) == 1 and len(set(counts)) == 1:
        return [((dtypes[0], counts[0]), list(range(len(dtypes))))]
    sets = {}
    for i, key in enumerate(zip(dtypes, counts)):
        sets.setdefault(key, []).append(i)
    return [(key, at[i:i + _MAX_TENSORS]) for key, at in sets.items()
            for i in range(0, len(at), _MAX_TENSORS)]


def gdn2_checkpoint_pack(*tensors):
    """The int8 form of ``tensors`` (floating point, last axis a multiple of
    64) as a ``Gdn2Checkpoint``.  Not differentiable."""
    ts = [t if isinstance(t, torch.Tensor) else torch.as_tensor(t) for t in tensors]
    if not ts:
        raise _fwd.Gdn2ShapeError("no tensors to pack")
    shapes, dtypes, sizes = [t.shape for t in ts], [t.dtype for t in ts], [t.numel() for t in ts]
    for shape, dt, n in zip(shapes, dtypes, sizes):
        if not dt.is_floating_point:
            raise _fwd.Gdn2ShapeError("inputs must be floating point")
        if not n or not shape or shape[-1] % GROUP:
            raise _fwd.Gdn2ShapeError(
                f"the last axis must be a positive multiple of {GROUP}; got {tuple(shape)}")
    on_host = not ts[0].is_cuda
    dev = torch.device("cuda", torch.cuda.current_device()) if on_host else ts[0].device
    kinds = [torch.bfloat16 if dt is torch.bfloat16 else torch.float32 for dt in dtypes]
    x = [_operand(t, dev, dt) for t, dt in zip(ts, kinds)]
    pack, stream = _lib.load().gdn2_int8_pack, _lib.raw_stream(dev.index)
    buffers = []
    for (dt, n), at in _launches(kinds, sizes):
        codes = torch.empty((len(at), n), dtype=torch.int8, device=dev)
        scales = torch.empty((len(at), n // GROUP), dtype=torch.float32, device=dev)
        rc = _lib.on_device(dev.index, pack, _lib.BF16 if dt is torch.bfloat16 else _lib.F32,
                            len(at), _ARRAYS[len(at)](*[x[i].data_ptr() for i in at]),
                            codes.data_ptr(), scales.data_ptr(), n, stream)
        _lib.check(rc, "gdn2_checkpoint_pack")
        buffers.append((at, codes, scales))
    return Gdn2Checkpoint(buffers, shapes, dtypes, on_host)


def gdn2_checkpoint_unpack(kept):
    """The tensors that ``kept`` holds, each in the type it was packed from."""
    dev = kept.buffers[0][1].device
    unpack, stream = _lib.load().gdn2_int8_unpack, _lib.raw_stream(dev.index)
    out = [None] * len(kept.shapes)
    for at, codes, scales in kept.buffers:
        bf16 = kept.dtypes[at[0]] is torch.bfloat16
        kind = torch.bfloat16 if bf16 else torch.float32
        for i in at:
            out[i] = scales.new_empty(kept.shapes[i], dtype=kind)
        rc = _lib.on_device(dev.index, unpack, _lib.BF16 if bf16 else _lib.F32, len(at),
                            _ARRAYS[len(at)](*[out[i].data_ptr() for i in at]),
                            codes.data_ptr(), scales.data_ptr(), codes.shape[1], stream)
        _lib.check(rc, "gdn2_checkpoint_unpack")
    out = [t if t.dtype is dt else t.to(dt) for t, dt in zip(out, kept.dtypes)]
    return tuple(t.cpu() for t in out) if kept.on_host else tuple(out)
