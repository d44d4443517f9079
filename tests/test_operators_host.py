"""The recurrence, the int8 checkpoints and the state cache on a machine without
a GPU: refusals before any launch, sizes, and launch sets."""
import ctypes

import pytest
import torch

from gdn2_package import (Gdn2StateCache, _lib, gdn2_checkpoint, gdn2_checkpoint_pack, gdn2_fwd,
                          gdn2_linear_recurrence, gdn2_linear_recurrence_trainable,
                          gdn2_pallas_forward_trainable, gdn2_state_cache)

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4100)


def arr(*p):
    return (ctypes.c_void_p * len(p))(*[x.value if x is not None else None for x in p])


def test_int8_entry_points_refuse():
    lib = _lib.load()
    bad = _lib.ERR_INVALID
    for fn in (lib.gdn2_int8_pack, lib.gdn2_int8_unpack):
        assert fn(7, 1, arr(P), P, P, 64, None) == bad            # dtype
        assert fn(0, 0, arr(P), P, P, 64, None) == bad            # no tensors
        assert fn(0, 9, arr(*[P] * 9), P, P, 64, None) == bad
        assert fn(0, 1, arr(P), P, P, 0, None) == bad
        assert fn(0, 1, arr(P), P, P, 65, None) == bad            # not a multiple of 64
        assert fn(0, 1, None, P, P, 64, None) == bad
        assert fn(0, 1, arr(P), None, P, 64, None) == bad
        assert fn(0, 1, arr(P), P, None, 64, None) == bad
        assert fn(0, 2, arr(P, None), P, P, 64, None) == bad
        assert fn(0, 1, arr(ODD), P, P, 64, None) == bad          # alignment
        assert fn(0, 1, arr(P), ODD, P, 64, None) == bad
        assert b"aligned" in lib.gdn2_last_error()


def test_state_entry_points_refuse():
    lib = _lib.load()
    bad = _lib.ERR_INVALID

    def write(h=P, slots=P, codes=P, scales=P, B=1, S=2, H=1, D=64, clip=1e4):
        return lib.gdn2_state_write(h, slots, codes, scales, B, S, H, D, clip, None)

    def read(dtype=0, codes=P, scales=P, slots=P, h=P, B=1, S=2, H=1, D=64):
        return lib.gdn2_state_read(dtype, codes, scales, slots, h, B, S, H, D, None)

    for fn in (write, read):
        for kw in (dict(B=0), dict(S=0), dict(H=0), dict(D=96), dict(h=None), dict(codes=None),
                   dict(scales=None), dict(h=ODD), dict(codes=ODD), dict(B=3, slots=None),
                   dict(B=65536, S=70000)):
            assert fn(**kw) == bad, kw
    assert write(clip=0.0) == bad and read(dtype=5) == bad

    def decode(dtype=0, q=P, codes=P, scales=P, src=P, dst=P, o=P, B=1, T=1, H=1, D=64, S=2,
               scale=0.1, clip=1e4):
        return lib.gdn2_decode_cached(dtype, q, P, P, P, P, P, codes, scales, src, dst, o, B, T, H,
                                      D, S, scale, clip, None)

    for kw in (dict(dtype=3), dict(q=None), dict(codes=None), dict(scales=None), dict(o=None),
               dict(B=0), dict(T=0), dict(H=0), dict(S=0), dict(D=256), dict(clip=-1.0),
               dict(scale=float("nan")), dict(codes=ODD), dict(scales=ODD), dict(src=None), dict(dst=None),
               dict(src=None, dst=None, B=3), dict(B=65536)):
        assert decode(**kw) == bad, kw


def test_recurrence_entry_points_refuse():
    lib = _lib.load()
    bad = _lib.ERR_INVALID

    def fwd(dtype=0, v=P, h0=None, o=P, hf=P, kept=P, v8=None, vs=None, w8=None, ws8=None, ws=P,
            n=1 << 30, B=1, T=100, H=1, D=64):
        return lib.gdn2_recur_fwd(dtype, v, P, P, h0, o, hf, kept, v8, vs, w8, ws8, ws, n, B, T, H,
                                  D, None)

    for kw in (dict(dtype=9), dict(v=None), dict(o=None), dict(hf=None), dict(v8=P), dict(vs=P),
               dict(B=0), dict(T=0), dict(H=0), dict(D=96), dict(v=ODD), dict(h0=ODD),
               dict(kept=ODD), dict(T=(1 << 30) + 1), dict(H=1 << 20)):
        assert fwd(**kw) == bad, kw
    assert fwd(n=16) == _lib.ERR_WORKSPACE and fwd(ws=None) == _lib.ERR_WORKSPACE

    def bwd(dtype=0, v=P, g=P, v8=None, vs=None, w8=None, ws8=None, kept=P, dout=P, dhf=None, dv=P,
            dh0=P, ws=P, n=1 << 30, B=1, T=100, H=1, D=64):
        return lib.gdn2_recur_bwd(dtype, v, P, g, v8, vs, w8, ws8, kept, dout, dhf, dv, P, P, dh0,
                                  ws, n, B, T, H, D, None)

    for kw in (dict(dtype=9), dict(v=None), dict(g=None), dict(v8=P), dict(kept=None),
               dict(dout=None), dict(dv=None), dict(dh0=None), dict(T=0), dict(D=32),
               dict(dout=ODD), dict(dhf=ODD)):
        assert bwd(**kw) == bad, kw
    assert bwd(n=16) == _lib.ERR_WORKSPACE


def test_timeout_selftest_refuses():
    lib = _lib.load()
    for ws, n, polls in ((None, 4096, 8), (P, 512, 8), (P, 4096, 0)):
        assert lib.gdn2_selftest_recur_timeout(ws, n, polls, None) == _lib.ERR_INVALID


def test_recurrence_sizes():
    lib = _lib.load()
    assert lib.gdn2_recur_kept_floats(2, 65, 3, 64) == 2 * 2 * 3 * 64
    assert lib.gdn2_recur_kept_floats(2, 64, 3, 64) == 2 * 3 * 64
    assert lib.gdn2_recur_kept_floats(0, 64, 3, 64) == 0
    assert lib.gdn2_recur_workspace_bytes(1, 100, 1, 96) == 0
    assert lib.gdn2_recur_workspace_bytes(1, 100, 1, 64) >= 512


def test_python_refusals():
    bad = gdn2_fwd.Gdn2ShapeError
    x = torch.zeros(1, 4, 2, 64)
    for v, w, g in ((x, x, x[:, :3]), (x[0], x[0], x[0]), (x[..., :32],) * 3, (x[:, :0],) * 3,
                    (x.long(), x, x)):
        with pytest.raises(bad):
            gdn2_linear_recurrence(v, w, g)
    with pytest.raises(bad, match="checkpoint"):
        gdn2_linear_recurrence_trainable(x, x, x, checkpoint="fp8")
    with pytest.raises(bad, match="checkpoint"):
        gdn2_pallas_forward_trainable(x, x, x, x, x, x, 0.1, checkpoint="fp8")
    for ts in ((), (x[..., :63],), (x[:0],), (x.long(),), (torch.zeros(()),)):
        with pytest.raises(bad):
            gdn2_checkpoint_pack(*ts)
    for S, H, D in ((0, 1, 64), (1, 0, 64), (1, 1, 96)):
        with pytest.raises(bad):
            Gdn2StateCache(S, H, D, device="cpu")
    cache = Gdn2StateCache(2, 1, 64, device="cpu")
    with pytest.raises(bad, match="CUDA"):
        gdn2_state_cache.gdn2_state_write(cache, torch.zeros(1, 1, 64, 64))


def test_launch_sets():
    """One launch per type and size, eight tensors at most."""
    f, b = torch.float32, torch.bfloat16
    sets = gdn2_checkpoint._launches([f] * 9 + [b, f], [64] * 9 + [64, 128])
    assert [(k, at) for k, at in sets] == [((f, 64), list(range(8))), ((f, 64), [8]),
                                           ((b, 64), [9]), ((f, 128), [10])]


def test_host_slot_checks():
    at = gdn2_state_cache._host_slots
    bad = gdn2_fwd.Gdn2ShapeError
    assert at([1, -1, 0, -1], 4, 2, "slots", True) == [1, -1, 0, -1]
    assert at([1, 1], 2, 2, "slots", False) == [1, 1]
    for s in ([2], [-2]):
        with pytest.raises(bad):
            at(s, 1, 2, "slots", False)
    with pytest.raises(bad):
        at([1, 1], 2, 2, "slots", True)


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """The device is switched for a call, and back, only where another is current."""
    seen = []

    class Switch:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            seen.append(self.index)

        def __exit__(self, *exc):
            seen.append("back")

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Switch)
    assert _lib.on_device(0, lambda a, b: a + b, 1, 2) == 3 and seen == []
    assert _lib.on_device(1, lambda: 7) == 7 and seen == [1, "back"]


def test_slot_arguments():
    slots = gdn2_state_cache._slots
    bad = gdn2_fwd.Gdn2ShapeError
    dev = torch.device("cpu")
    assert slots(None, 2, 2, dev, "slots", True) == (None, None)
    t, host = slots([1, -1], 2, 2, dev, "slots", True)
    assert t.dtype == torch.int32 and t.tolist() == host == [1, -1]
    for s in (torch.tensor(0), torch.tensor([0.0, 1.0]), torch.tensor([True, False]), [0], [[0, 1]]):
        with pytest.raises(bad):
            slots(s, 2, 2, dev, "slots", True)
    with pytest.raises(bad, match="give slots"):
        slots(None, 3, 2, dev, "slots", True)


def test_settings_come_back_after_a_call(monkeypatch):
    from gdn2_package import gdn2_pipeline
    saved = gdn2_pipeline._settings()
    monkeypatch.setattr(gdn2_fwd, "GATES", "raw")
    monkeypatch.setattr(gdn2_fwd, "CLIP", 7.0)
    with pytest.raises(ZeroDivisionError):
        with gdn2_pipeline._with_settings(saved):
            assert gdn2_fwd.GATES == "activated" and gdn2_fwd.CLIP == 1e4
            1 / 0
    assert gdn2_fwd.GATES == "raw" and gdn2_fwd.CLIP == 7.0


def test_bytes_that_the_recurrence_keeps():
    """g, the states before every 64th token, and v and w or their 8-bit form."""
    from gdn2_package.gdn2_recurrence import Gdn2RecurrenceResiduals
    shape, n = (2, 130, 3, 64), 2 * 130 * 3 * 64
    rest = (shape, None, False, 0, (torch.float32,) * 3, None)
    g, kept = torch.zeros(shape), torch.zeros(2, 3, 3, 64)
    full = Gdn2RecurrenceResiduals.with_tensors((*rest, False), g, kept, g.clone(), g.clone())
    assert full.nbytes == 12 * n + 4 * kept.numel() and full.int8 is None
    codes, scales = torch.zeros((2, *shape), dtype=torch.int8), torch.zeros(2, n // 64)
    small = Gdn2RecurrenceResiduals.with_tensors((*rest, True), g, kept, codes, scales)
    assert small.nbytes == 4 * n + 2 * n + 8 * (n // 64) + 4 * kept.numel() and small.v is None
