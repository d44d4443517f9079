"""int8 cache of recurrent states and the decode that runs on it (no
counterpart in the reference, whose states are float32, gdn2_fwd.py:400-404).

A ``Gdn2StateCache`` holds one (H, D, D) state per slot in the int8 form of
``gdn2_checkpoint`` (groups of 64 value columns of a key row), a quarter of the
float32 bytes.  ``gdn2_state_write`` parks states, ``gdn2_state_read`` fetches
them, ``gdn2_decode_cached`` runs tokens from one slot into another.

Slots are int32 or int64 tensors (B,), or lists.  -1 reads as the zero state
and drops what is written to it, so it pads a batch.  Slots given on the host
are checked there; slots on the device are checked by the kernels, which give
NaN for a row they refuse.

Each store rounds a state value by at most 1/254 of the largest of its group
(``gdn2_decode_cached`` by 3e-5 of a step more: it takes the nearest code by
float32 arithmetic, where ``gdn2_state_write`` decides it exactly).
``gdn2_decode_cached`` rounds once a call, whatever T is: the state is float32
between the call's tokens.  A decay or an update below half a step of its group
is lost in that rounding, so sequences that must remember over very many single
steps keep float32 states (``gdn2_decode``).
"""
from __future__ import annotations

import torch

from . import _lib
from . import gdn2_fwd as _fwd
from .gdn2_checkpoint import GROUP, _operand


class Gdn2StateCache:
    """int8 states of ``slots`` sequences; every slot starts as the zero state."""

    def __init__(self, slots, H, D, device=None):
        if slots <= 0 or H <= 0:
            raise _fwd.Gdn2ShapeError("empty cache")
        if D not in (64, 128, 256):
            raise _fwd.Gdn2ShapeError(f"head dim D={D} unsupported (64, 128 or 256)")
        device = torch.device("cuda" if device is None else device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.codes = torch.zeros((slots, H, D, D), dtype=torch.int8, device=device)
        self.scales = torch.zeros((slots, H, D, D // GROUP), dtype=torch.float32, device=device)

    @classmethod
    def from_tensors(cls, codes, scales):
        """A cache on existing tensors (S, H, D, D) int8 and (S, H, D, D / 64)
        float32, which it shares."""
        if codes.dim() != 4 or codes.dtype != torch.int8 or codes.shape[2] != codes.shape[3] \
                or codes.shape[3] not in (64, 128, 256) or codes.numel() == 0:
            raise _fwd.Gdn2ShapeError(f"codes must be (S, H, D, D) int8; got {tuple(codes.shape)}")
        want = (*codes.shape[:3], codes.shape[3] // GROUP)
        if tuple(scales.shape) != want or scales.dtype != torch.float32 \
                or scales.device != codes.device:
            raise _fwd.Gdn2ShapeError(f"scales must be {want} float32 on the codes' device")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16 \
                or scales.data_ptr() % 16:
            raise _fwd.Gdn2ShapeError("codes and scales must be contiguous and 16-byte aligned")
        self = cls.__new__(cls)
        self.codes, self.scales = codes, scales
        return self

    slots = property(lambda self: self.codes.shape[0])
    H = property(lambda self: self.codes.shape[1])
    D = property(lambda self: self.codes.shape[3])
    device = property(lambda self: self.codes.device)
    nbytes = property(lambda self: self.codes.numel() + 4 * self.scales.numel())


def _on_gpu(cache):
    if not cache.codes.is_cuda:
        raise _fwd.Gdn2ShapeError("the cache must be on a CUDA device")
    return cache.codes.device


def _host_slots(slots, B, S, what, distinct):
    """Checks of a slot list given on the host; the list."""
    at = [int(i) for i in slots]
    if any(i < -1 or i >= S for i in at):
        raise _fwd.Gdn2ShapeError(f"{what} must lie in [-1, {S})")
    used = [i for i in at if i >= 0]
    if distinct and len(set(used)) < len(used):
        raise _fwd.Gdn2ShapeError(f"{what} name a slot twice")
    return at


def _slots(slots, B, S, dev, what, distinct):
    """(device int32 tensor or None, host list or None) of a slot argument."""
    if slots is None:
        if B > S:
            raise _fwd.Gdn2ShapeError(f"{B} rows for {S} slots: give {what}")
        return None, None
    on_gpu = isinstance(slots, torch.Tensor) and slots.is_cuda
    if on_gpu and slots.dtype is torch.int32 and slots.shape == (B,) and slots.device == dev:
        return slots.contiguous(), None
    t = slots if isinstance(slots, torch.Tensor) else torch.as_tensor(slots)
    if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (B,):
        raise _fwd.Gdn2ShapeError(f"{what} must be {B} int32 or int64 values; "
                                  f"got {tuple(t.shape)} {t.dtype}")
    host = None if on_gpu else _host_slots(t.tolist(), B, S, what, distinct)
    if t.dtype == torch.int64 and on_gpu:
        # beyond int32 means outside every cache, whatever the low bits say
        t = t.clamp(-2, 0x7fffffff)
    return t.to(device=dev, dtype=torch.int32).contiguous(), host


def _ptr(t):
    return t.data_ptr() if t is not None else None


def gdn2_state_write(cache, h, slots=None):
    """Store states h (B, H, D, D) in ``slots`` of the cache (slot b for row b
    by default), through the CLIP sanitiser.  Of several rows that name one slot
    the last is kept (slots on the host must be distinct)."""
    dev = _on_gpu(cache)
    if not isinstance(h, torch.Tensor):
        h = torch.as_tensor(h)
    if h.dim() != 4 or h.shape[1:] != cache.codes.shape[1:] or h.shape[0] == 0:
        raise _fwd.Gdn2ShapeError(
            f"h must be (B, {cache.H}, {cache.D}, {cache.D}); got {tuple(h.shape)}")
    B, S = h.shape[0], cache.slots
    at, _ = _slots(slots, B, S, dev, "slots", True)
    hs = _operand(h, dev, torch.float32)
    _, H, D, _ = h.shape
    rc = _lib.on_device(dev.index, _lib.load().gdn2_state_write, hs.data_ptr(), _ptr(at),
                        cache.codes.data_ptr(), cache.scales.data_ptr(), B, S, H, D,
                        float(_fwd.CLIP), _lib.raw_stream(dev.index))
    _lib.check(rc, "gdn2_state_write")


def gdn2_state_read(cache, slots=None, dtype=torch.float32):
    """The states (B, H, D, D) of ``slots`` (all slots by default) in float32 or
    bfloat16.  A slot may be named several times; -1 reads as the zero state."""
    dev = _on_gpu(cache)
    if dtype not in (torch.float32, torch.bfloat16):
        raise _fwd.Gdn2ShapeError(f"dtype must be float32 or bfloat16; got {dtype}")
    S, H, D, _ = cache.codes.shape
    B = S
    if slots is not None:
        if not isinstance(slots, torch.Tensor):
            slots = torch.as_tensor(slots)
        B = slots.numel()
        if B == 0:
            raise _fwd.Gdn2ShapeError("empty problem")
    at, _ = _slots(slots, B, S, dev, "slots", False)
    h = cache.scales.new_empty((B, H, D, D), dtype=dtype)
    rc = _lib.on_device(dev.index, _lib.load().gdn2_state_read,
                        _lib.F32 if dtype is torch.float32 else _lib.BF16, cache.codes.data_ptr(),
                        cache.scales.data_ptr(), _ptr(at), h.data_ptr(), B, S, H, D,
                        _lib.raw_stream(dev.index))
    _lib.check(rc, "gdn2_state_read")
    return h


def gdn2_decode_cached(q, k, v, w, b, g, scale, cache, slots=None, out_slots=None):
    """``gdn2_decode`` from the states in ``slots`` into ``out_slots`` of the
    cache (the same slots by default; slot b for row b where neither is given).

    q..g (B, T, H, D) with T as small as 1 and D 64 or 128 (states of 256
    are read for ``gdn2_pallas_forward``); returns o (B, T, H, D) float32.
    Several rows may start from one slot, each with a destination of its own (a
    shared prefix).  A destination must not be another row's source or
    destination: the host refuses such slots where it has them, the kernel gives
    NaN for the row and stores nothing."""
    dev = _on_gpu(cache)
    ts = (q, k, v, w, b, g)
    if not all(isinstance(t, torch.Tensor) for t in ts):
        ts = tuple(torch.as_tensor(t) for t in ts)
    shape = ts[0].shape
    if len(shape) != 4 or any(t.shape != shape for t in ts):
        raise _fwd.Gdn2ShapeError(f"inputs must share one (B, T, H, D) shape; got {tuple(shape)}")
    B, T, H, D = shape
    if D not in (64, 128):
        raise _fwd.Gdn2ShapeError(f"head dim D={D} unsupported (64 or 128)")
    if B * T * H == 0:
        raise _fwd.Gdn2ShapeError("empty problem")
    dtypes = [t.dtype for t in ts]
    for dt in dtypes:
        if not dt.is_floating_point:
            raise _fwd.Gdn2ShapeError("inputs must be floating point")
    if cache.codes.shape[1:3] != (H, D):
        raise _fwd.Gdn2ShapeError(f"the cache holds states of H={cache.H}, D={cache.D}; "
                                  f"got H={H}, D={D}")
    S = cache.codes.shape[0]
    if slots is None and out_slots is not None:
        raise _fwd.Gdn2ShapeError("out_slots need slots")
    src, src_host = _slots(slots, B, S, dev, "slots", out_slots is None)
    dst = src
    if out_slots is not None:
        dst, dst_host = _slots(out_slots, B, S, dev, "out_slots", True)
        if src_host is not None and dst_host is not None:
            readers = {}
            for i, s in enumerate(src_host):
                readers.setdefault(s, []).append(i)
            if any(d >= 0 and any(j != i for j in readers.get(d, ())) for i, d in enumerate(dst_host)):
                raise _fwd.Gdn2ShapeError("a slot of out_slots is another row's slot")
    bf16 = dtypes.count(torch.bfloat16) == 6
    cdt = torch.bfloat16 if bf16 else torch.float32
    on_host = not ts[0].is_cuda
    x = [_operand(t, dev, cdt, on_host) for t in ts]   # copies live until the launch
    o = cache.scales.new_empty(shape)
    code = _lib.BF16 if bf16 else _lib.F32
    if _fwd.GATES == "raw":
        code |= _lib.GATES_RAW
    rc = _lib.on_device(dev.index, _lib.load().gdn2_decode_cached, code,
                        *[t.data_ptr() for t in x], cache.codes.data_ptr(),
                        cache.scales.data_ptr(), _ptr(src), _ptr(dst), o.data_ptr(), B, T, H, D, S,
                        float(scale), float(_fwd.CLIP), _lib.raw_stream(dev.index))
    _lib.check(rc, "gdn2_decode_cached")
    return o.cpu() if on_host else o
