"""int8 checkpoints, the int8 state cache and the decode that runs on it."""
import numpy as np
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

import gdn2_oracle as O  # noqa: E402
from int8_ref import pack64, values64  # noqa: E402
from gdn2_package import (Gdn2StateCache, gdn2_backward, gdn2_checkpoint_pack,  # noqa: E402
                          gdn2_checkpoint_unpack, gdn2_decode, gdn2_decode_cached, gdn2_fwd,
                          gdn2_pallas_forward, gdn2_pallas_forward_trainable, gdn2_state_read,
                          gdn2_state_write)
from gdn2_package.synthetic import make_inputs  # noqa: E402

NAMES = ("q", "k", "v", "w", "b", "g")


@pytest.fixture(autouse=True)
def _gates():
    saved = gdn2_fwd.GATES
    yield
    gdn2_fwd.GATES = saved


def rel(a, b):
    a = a.double().cpu().numpy() if isinstance(a, torch.Tensor) else np.asarray(a, np.float64)
    b = b.double().cpu().numpy() if isinstance(b, torch.Tensor) else np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


def same(a, b):
    """Equal, NaN in the same places."""
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


# ---------------------------------------------------------------- checkpoints

@pytest.mark.parametrize("shape", [(64,), (1, 64), (3, 5, 64), (2, 7, 3, 128), (1, 1031, 1, 256),
                                   (4, 100, 3, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_are_the_correctly_rounded_ones(shape, dtype):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).mul_(
        torch.randn(shape, generator=torch.Generator().manual_seed(2)).exp()).to(dtype).cuda()
    kept = gdn2_checkpoint_pack(x)
    codes, scales = pack64(x)
    assert torch.equal(kept.codes[0].long(), codes) and torch.equal(kept.scales[0], scales)
    (y,) = gdn2_checkpoint_unpack(kept)
    assert y.dtype == dtype and torch.equal(y, values64(x).to(dtype))


def test_ties_and_their_neighbours():
    """Values on a half step, and one float32 step to either side of it."""
    rows = []
    for top in (127.0, 1.0, 0.37, 254.0, 1e-20, 3e37, 2.0 ** -99):
        half = (torch.arange(-63, 63) + 0.5).mul(2) * 0.5 * (top / 127.0)
        for x in (half, torch.nextafter(half, torch.full_like(half, 1e38)),
                  torch.nextafter(half, torch.full_like(half, -1e38))):
            for part in x.split(63):
                rows.append(torch.cat([part, torch.tensor([top])]))
    x = torch.stack(rows).cuda()
    kept = gdn2_checkpoint_pack(x)
    codes, scales = pack64(x)
    assert torch.equal(kept.codes[0].long(), codes) and torch.equal(kept.scales[0], scales)
    exact_half = (torch.arange(63) + 0.5).cuda()   # of max 127: ties, to even
    c = gdn2_checkpoint_pack(torch.cat([exact_half, torch.tensor([127.0]).cuda()])).codes[0]
    assert c[:4].tolist() == [0, 2, 2, 4]


@pytest.mark.parametrize("power", [-90, 0, 119])
def test_every_bf16_quotient_next_to_a_half(power):
    """All pairs of 8-bit mantissas, sizes down to 2^-9 of the largest: the codes
    of a bf16 group are the correctly rounded ones, ties (one pair in a few
    hundred) included."""
    top = torch.arange(128, 256).view(-1, 1, 1)
    x = torch.arange(128, 256).view(1, -1, 1) * 0.5 ** torch.arange(0, 10).view(1, 1, -1)
    x = x.reshape(1, -1).expand(128, -1).clone()
    x[x > top[:, 0]] *= 0.5
    x[:, ::2] *= -1
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 63)).view(128, -1, 63)
    x = torch.cat([x, top.expand(-1, x.shape[1], 1)], 2) * 2.0 ** power
    x = x.to(torch.bfloat16).cuda()
    assert torch.isfinite(x).all()
    kept = gdn2_checkpoint_pack(x)
    codes, scales = pack64(x)
    assert torch.equal(kept.codes[0].long(), codes) and torch.equal(kept.scales[0], scales)


def test_zero_tiny_and_non_finite_groups():
    x = torch.randn(7, 64, generator=torch.Generator().manual_seed(3)).cuda()
    x[1] = 0
    x[2] *= 2.0 ** -120
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    x[5, 7] = -float("inf")
    (y,) = gdn2_checkpoint_unpack(gdn2_checkpoint_pack(x))
    assert same(y, values64(x))
    assert (y[1] == 0).all() and (y[2] == 0).all() and torch.isnan(y[3:6]).all()
    assert torch.isfinite(y[[0, 6]]).all()


def test_many_tensors_types_and_places():
    """More tensors than one launch takes, mixed types and sizes, strides, an
    unaligned view, float64 and half, host tensors; each comes back as it was."""
    gen = torch.Generator().manual_seed(4)
    ts = [torch.randn(3, 5, 64, generator=gen).cuda() for _ in range(9)]
    ts += [torch.randn(2, 64, generator=gen).to(dt).cuda()
           for dt in (torch.bfloat16, torch.float64, torch.float16)]
    ts.append(torch.randn(64, 6, generator=gen).cuda().t())
    ts.append(torch.randn(129, generator=gen).cuda()[1:])
    out = gdn2_checkpoint_unpack(gdn2_checkpoint_pack(*ts))
    for x, y in zip(ts, out):
        f = x if x.dtype == torch.bfloat16 else x.float()
        assert y.dtype == x.dtype and torch.equal(y, values64(f).to(x.dtype))
    host = torch.randn(2, 128, generator=gen)
    (y,) = gdn2_checkpoint_unpack(gdn2_checkpoint_pack(host))
    assert y.device.type == "cpu" and torch.equal(y, values64(host))
    kept = gdn2_checkpoint_pack(*ts[:9])
    assert kept.nbytes == 9 * (960 + 960 // 16)


@pytest.mark.parametrize("D,bt,bc,dtype", [(64, 64, 16, torch.float32), (128, 128, 64, torch.float32),
                                           (128, 64, 32, torch.bfloat16), (256, 64, 32, torch.float32)])
def test_gdn2_training_from_int8_checkpoints(D, bt, bc, dtype):
    """Outputs of the inputs, gradients of the backward at the restored inputs."""
    gdn2_fwd.BT, gdn2_fwd.BC = bt, bc
    inp = make_inputs(2, 256, 2, D, seed=41, h0_std=0.1)
    args = [torch.as_tensor(inp[n]).cuda().to(dtype) for n in NAMES]
    h0, do, dh = (torch.as_tensor(inp[n]).cuda() for n in ("h0", "dout", "dh_final"))
    leaves = [t.clone().requires_grad_(True) for t in (*args, h0)]
    o, h = gdn2_pallas_forward_trainable(*leaves[:6], inp["scale"], leaves[6], checkpoint="int8")
    o_r, h_r = gdn2_pallas_forward(*args, inp["scale"], h0)
    assert torch.equal(o, o_r) and torch.equal(h, h_r)
    got = torch.autograd.grad((o, h), leaves, (do, dh))
    restored = [values64(t).to(dtype) for t in args[:5]]
    want = gdn2_backward(*restored, args[5], inp["scale"], h0, do, dh)
    for n, a, b in zip((*NAMES, "h0"), got, want):
        assert a.dtype == b.dtype and torch.equal(a, b), n
    full = gdn2_backward(*args, inp["scale"], h0, do, dh)
    for n, a, b in zip((*NAMES, "h0"), got, full):
        assert rel(a, b) < 0.05, (n, rel(a, b))   # half a step is 1/254 of a group's largest


@pytest.mark.parametrize("host", [False, True])
def test_gdn2_int8_training_with_raw_gates_and_a_tail(host):
    """Pre-activations are packed as they are given; T that BT does not divide;
    leaves on the GPU or on the host."""
    gdn2_fwd.BT, gdn2_fwd.BC, gdn2_fwd.GATES, gdn2_fwd.MASKED_TAIL = 64, 16, "raw", True
    inp = make_inputs(1, 100, 2, 64, seed=42, h0_std=0.1)
    gen = torch.Generator().manual_seed(43)
    dev = "cpu" if host else "cuda"
    args = [torch.as_tensor(inp[n]).to(dev) for n in ("q", "k", "v")]
    args += [torch.randn(1, 100, 2, 64, generator=gen).to(dev) for _ in range(3)]
    h0, do, dh = (torch.as_tensor(inp[n]).to(dev) for n in ("h0", "dout", "dh_final"))
    leaves = [t.clone().requires_grad_(True) for t in (*args, h0)]
    o, h = gdn2_pallas_forward_trainable(*leaves[:6], inp["scale"], leaves[6], checkpoint="int8")
    got = torch.autograd.grad((o, h), leaves, (do, dh))
    restored = [values64(t) for t in args[:5]]
    want = gdn2_backward(*restored, args[5], inp["scale"], h0, do, dh)
    for n, a, b in zip((*NAMES, "h0"), got, want):
        assert a.device.type == dev and torch.equal(a, b), n


# ---------------------------------------------------------------- state cache

def states(B, H, D, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (0.1 * torch.randn(B, H, D, D, generator=gen)
            * torch.randn(B, H, D, 1, generator=gen).exp()).cuda()


@pytest.mark.parametrize("B,S,H,D", [(1, 1, 1, 64), (3, 7, 5, 64), (4, 4, 3, 128), (2, 9, 1, 256)])
@pytest.mark.parametrize("kind", ["none", "int32", "int64", "list"])
def test_write_and_read(B, S, H, D, kind):
    h = states(B, H, D)
    cache = Gdn2StateCache(S, H, D)
    at = torch.randperm(S, generator=torch.Generator().manual_seed(5))[:B]
    slots = {"none": None, "int32": at.cuda().int(), "int64": at.cuda(), "list": at.tolist()}[kind]
    gdn2_state_write(cache, h, slots)
    where = at if slots is not None else torch.arange(B)
    want = torch.zeros(S, H, D, D, device="cuda")
    want[where.cuda()] = values64(h)
    assert torch.equal(gdn2_state_read(cache), want)
    assert torch.equal(gdn2_state_read(cache, where.cuda()), values64(h))
    assert torch.equal(gdn2_state_read(cache, where.tolist(), dtype=torch.bfloat16),
                       values64(h).to(torch.bfloat16))


def test_padding_repeated_and_foreign_slots():
    h = states(6, 2, 64)
    cache = Gdn2StateCache(4, 2, 64)
    gdn2_state_write(cache, states(4, 2, 64, seed=9))
    old = gdn2_state_read(cache)
    slots = torch.tensor([2, -1, 0, 2, 4, -7], device="cuda")
    gdn2_state_write(cache, h, slots)   # the later row of slot 2 stays; -1, 4, -7 are dropped
    now = gdn2_state_read(cache)
    assert torch.equal(now[[1, 3]], old[[1, 3]])
    assert torch.equal(now[0], values64(h)[2]) and torch.equal(now[2], values64(h)[3])
    got = gdn2_state_read(cache, torch.tensor([0, -1, 0, 4, 2 ** 32], device="cuda"))
    assert torch.equal(got[0], now[0]) and torch.equal(got[2], now[0])
    assert (got[1] == 0).all() and torch.isnan(got[3:]).all()


def test_states_are_sanitised_as_they_are_written():
    gdn2_fwd.CLIP = 2.0
    h = states(1, 1, 64)
    h[0, 0, 0, 0], h[0, 0, 1, 1], h[0, 0, 2, 2], h[0, 0, 3, 3] = float("nan"), float("inf"), -float("inf"), 7.0
    cache = Gdn2StateCache(1, 1, 64)
    gdn2_state_write(cache, h)
    want = torch.nan_to_num(h, nan=0.0, posinf=2.0, neginf=-2.0).clamp(-2, 2)
    assert torch.equal(gdn2_state_read(cache), values64(want))


def test_cache_on_given_tensors():
    codes = torch.zeros((3, 2, 64, 64), dtype=torch.int8, device="cuda")
    scales = torch.zeros((3, 2, 64, 1), device="cuda")
    cache = Gdn2StateCache.from_tensors(codes, scales)
    gdn2_state_write(cache, states(3, 2, 64))
    assert int(codes.abs().max()) == 127 and cache.nbytes == 3 * 2 * 64 * 68
    for c, s in ((codes.float(), scales), (codes, scales[:2]), (codes[:, :, :32], scales),
                 (codes.transpose(2, 3), scales), (codes, scales.cpu())):
        with pytest.raises(ValueError):
            Gdn2StateCache.from_tensors(c, s)


# ---------------------------------------------------------------- decode on the cache

def tokens(B, T, H, D, dtype=torch.float32, seed=0):
    inp = make_inputs(B, T, H, D, seed=seed, grads=False)
    return [torch.as_tensor(inp[n]).cuda().to(dtype) for n in NAMES], inp["scale"]


def oracle(args, scale, h0, clip=1e4):
    """Chunks of one token, every sanitiser in place, in float64."""
    ref = [t.double().cpu().numpy() for t in args]
    return O.forward(*ref, scale, h0.double().cpu().numpy(), 1, 1, clip)


def check_state(got, want):
    """Within half a step of the exact state's group, and float32 arithmetic's
    error (1e-5 of the group's largest, as the float32 decode is held to)."""
    want = torch.as_tensor(want).cuda().unflatten(-1, (-1, 64))
    top = want.abs().amax(-1, keepdim=True)
    err = (got.double().unflatten(-1, (-1, 64)) - want).abs()
    assert bool((err <= top * (0.5 / 127 + 2e-5)).all()), float((err / top).max())


@pytest.mark.parametrize("B,T,H,D", [(1, 1, 1, 64), (3, 1, 5, 128), (2, 6, 3, 64), (2, 9, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_from_and_into_the_cache(B, T, H, D, dtype):
    args, scale = tokens(B, T, H, D, dtype, seed=51)
    cache = Gdn2StateCache(2 * B + 1, H, D)
    order = torch.randperm(2 * B + 1, generator=torch.Generator().manual_seed(6)).cuda()
    src, dst = order[:B], order[B:2 * B].int()
    gdn2_state_write(cache, states(B, H, D, seed=7), src)
    h0 = gdn2_state_read(cache, src)
    before = gdn2_state_read(cache)
    o = gdn2_decode_cached(*args, scale, cache, src, dst)
    o_r, h_r = oracle(args, scale, h0)
    assert rel(o, o_r) < 1e-5
    check_state(gdn2_state_read(cache, dst), h_r)
    kept = torch.ones(2 * B + 1, dtype=torch.bool, device="cuda")
    kept[dst.long()] = False
    assert torch.equal(gdn2_state_read(cache)[kept], before[kept])
    # in place gives the same outputs and states
    o2 = gdn2_decode_cached(*args, scale, cache, src)
    assert torch.equal(o, o2)
    assert torch.equal(gdn2_state_read(cache, src), gdn2_state_read(cache, dst))


def test_decode_of_all_slots_in_place():
    args, scale = tokens(3, 2, 2, 64, seed=52)
    cache = Gdn2StateCache(4, 2, 64)
    gdn2_state_write(cache, states(4, 2, 64, seed=8))
    h = gdn2_state_read(cache)
    o = gdn2_decode_cached(*args, scale, cache)
    o_r, h_r = oracle(args, scale, h[:3])
    assert rel(o, o_r) < 1e-5
    check_state(gdn2_state_read(cache)[:3], h_r)
    assert torch.equal(gdn2_state_read(cache)[3], h[3])


def test_shared_prefix_padding_and_dropped_states():
    """Rows that start from one slot, from the zero state, and one that keeps
    nothing, beside each other."""
    args, scale = tokens(5, 3, 2, 128, seed=53)
    cache = Gdn2StateCache(6, 2, 128)
    gdn2_state_write(cache, states(6, 2, 128, seed=9))
    src = torch.tensor([1, 1, -1, 0, -1], device="cuda", dtype=torch.int32)
    dst = torch.tensor([2, 3, 4, -1, -1], device="cuda", dtype=torch.int32)
    h0 = gdn2_state_read(cache, src)
    before = gdn2_state_read(cache)
    o = gdn2_decode_cached(*args, scale, cache, src, dst)
    o_r, h_r = oracle(args, scale, h0)
    assert rel(o, o_r) < 1e-5
    check_state(gdn2_state_read(cache, dst[:3]), h_r[:3])
    assert torch.equal(gdn2_state_read(cache)[[0, 1, 5]], before[[0, 1, 5]])
    # the same through lists, which the host checks
    o2 = gdn2_decode_cached(*args, scale, cache, src.tolist(), dst.tolist())
    assert torch.equal(o, o2)


def test_rows_the_kernel_refuses():
    """A destination that another row reads or writes, or a slot outside the
    cache: NaN for that row, its state untouched, the others right."""
    args, scale = tokens(7, 2, 1, 64, seed=54)
    cache = Gdn2StateCache(8, 1, 64)
    gdn2_state_write(cache, states(8, 1, 64, seed=10))
    before = gdn2_state_read(cache)
    src = torch.tensor([0, 1, 2, 3, 8, -2, 4], device="cuda", dtype=torch.int32)
    dst = torch.tensor([5, 6, 6, 4, 7, 7, 8], device="cuda", dtype=torch.int32)
    # row 0 is fine; 1 and 2 share a destination; 3 writes what 6 reads; the rest lie outside
    h0 = gdn2_state_read(cache, src.clamp(0, 7))
    o = gdn2_decode_cached(*args, scale, cache, src, dst)
    assert torch.isnan(o[1:]).all()
    o_r, h_r = oracle([t[:1] for t in args], scale, h0[:1])
    assert rel(o[:1], o_r) < 1e-5
    now = gdn2_state_read(cache)
    check_state(now[5:6], h_r)
    rest = [0, 1, 2, 3, 4, 6, 7]
    assert torch.equal(now[rest], before[rest])
    # one slot twice in place
    twice = torch.tensor([1, 1], device="cuda", dtype=torch.int32)
    two = [t[:2] for t in args]
    assert torch.isnan(gdn2_decode_cached(*two, scale, cache, twice)).all()
    assert torch.equal(gdn2_state_read(cache), now)


def test_slots_the_host_refuses():
    args, scale = tokens(2, 1, 1, 64, seed=55)
    cache = Gdn2StateCache(4, 1, 64)
    h = states(2, 1, 64)
    bad = gdn2_fwd.Gdn2ShapeError
    for slots in ([0, 0], [0, 4], [-2, 1], [0], [0.5, 1.0], torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(bad):
            gdn2_decode_cached(*args, scale, cache, slots)
        with pytest.raises(bad):
            gdn2_state_write(cache, h, slots)
    for src, dst in (([0, 1], [1, 2]), ([0, 1], [2, 2]), (None, [0, 1]), ([0, 1], [2])):
        with pytest.raises(bad):
            gdn2_decode_cached(*args, scale, cache, src, dst)
    for t in ([x[:, :, :, :32] for x in args], [x.repeat(1, 1, 2, 1) for x in args],
              [x[:0] for x in args], [x.long() for x in args]):
        with pytest.raises(bad):
            gdn2_decode_cached(*t, scale, cache, [0, 1])
    with pytest.raises(bad):
        gdn2_state_write(cache, h[:, :, :32], [0, 1])
    with pytest.raises(bad):
        gdn2_state_write(cache, states(5, 1, 64))
    with pytest.raises(bad):
        gdn2_state_read(cache, [0], dtype=torch.float16)
    with pytest.raises(bad):
        gdn2_state_read(cache, [])


@pytest.mark.parametrize("clip,gscale", [(0.3, 1.0), (1e4, 30.0)])
def test_decode_with_clip_and_fast_gates(clip, gscale):
    gdn2_fwd.CLIP = clip
    args, scale = tokens(2, 12, 2, 128, seed=56)
    args[5] = args[5] * gscale
    cache = Gdn2StateCache(4, 2, 128)
    gdn2_state_write(cache, states(2, 2, 128, seed=11))
    h0 = gdn2_state_read(cache, [0, 1])
    o = gdn2_decode_cached(*args, scale, cache, [0, 1], [2, 3])
    o_r, h_r = oracle(args, scale, h0, clip)
    assert rel(o, o_r) < 1e-5
    check_state(gdn2_state_read(cache, [2, 3]), h_r)


def test_decode_with_raw_gates_and_host_tokens():
    args, scale = tokens(2, 3, 2, 64, seed=57)
    raw = [torch.randn(args[0].shape, generator=torch.Generator().manual_seed(i)).cuda()
           for i in range(3)]
    act = [torch.sigmoid(raw[0]), torch.sigmoid(raw[1]), -torch.nn.functional.softplus(raw[2])]
    cache = Gdn2StateCache(4, 2, 64)
    gdn2_state_write(cache, states(2, 2, 64, seed=12))
    a = gdn2_decode_cached(*args[:3], *act, scale, cache, [0, 1], [2, 3])
    gdn2_fwd.GATES = "raw"
    b = gdn2_decode_cached(*args[:3], *raw, scale, cache, [0, 1], [2, 3])
    assert rel(a, b) < 1e-5
    c = gdn2_decode_cached(*[t.cpu() for t in (*args[:3], *raw)], scale, cache, [0, 1], [2, 3])
    assert c.device.type == "cpu" and torch.equal(c, b.cpu())


def test_captured_decode_follows_its_slots():
    """A captured step reads its slots when it is replayed."""
    args, scale = tokens(2, 1, 3, 128, seed=58)
    cache = Gdn2StateCache(6, 3, 128)
    gdn2_state_write(cache, states(6, 3, 128, seed=13))
    slots = torch.tensor([0, 1], device="cuda", dtype=torch.int32)
    start = cache.codes.clone(), cache.scales.clone()
    gdn2_decode_cached(*args, scale, cache, slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = gdn2_decode_cached(*args, scale, cache, slots)
    for at in ([4, 2], [5, -1]):
        cache.codes.copy_(start[0])
        cache.scales.copy_(start[1])
        slots.copy_(torch.tensor(at))
        g.replay()
        got, state = o.clone(), gdn2_state_read(cache)
        cache.codes.copy_(start[0])
        cache.scales.copy_(start[1])
        assert torch.equal(got, gdn2_decode_cached(*args, scale, cache, at))
        assert torch.equal(state, gdn2_state_read(cache))


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 values: the last slot."""
    H, D = 8, 128
    S = 2 ** 31 // (H * D * D) + 3
    cache = Gdn2StateCache(S, H, D)
    h = states(1, H, D, seed=14)
    gdn2_state_write(cache, h, [S - 1])
    assert torch.equal(gdn2_state_read(cache, [S - 1]), values64(h))
    args, scale = tokens(1, 1, H, D, seed=59)
    o = gdn2_decode_cached(*args, scale, cache, [S - 1], [S - 2])
    o_r, h_r = oracle(args, scale, values64(h))
    assert rel(o, o_r) < 1e-5
    check_state(gdn2_state_read(cache, [S - 2]), h_r)
    assert torch.equal(gdn2_state_read(cache, [S - 1]), values64(h))


def test_prompt_cache_and_generation_together():
    """A prompt through the chunked forward, its state parked, two branches
    decoded from it, and each continued by the chunked forward: against the same
    run in float32.  Each of the two stores rounds a state value by 1/254 of its
    group's largest at most, 0.6% of the state's size on normal values."""
    gdn2_fwd.BT, gdn2_fwd.BC = 64, 16
    args, scale = tokens(1, 128, 2, 128, seed=60)
    _, h = gdn2_pallas_forward(*args, scale)
    cache = Gdn2StateCache(3, 2, 128)
    gdn2_state_write(cache, h, [0])
    more, _ = tokens(2, 4, 2, 128, seed=61)
    o = gdn2_decode_cached(*more, scale, cache, [0, 0], [1, 2])
    o_f, h_f = gdn2_decode(*more, scale, h.expand(2, -1, -1, -1).contiguous())
    assert rel(o, o_f) < 0.02 and rel(gdn2_state_read(cache, [1, 2]), h_f) < 0.02
    tail, _ = tokens(2, 64, 2, 128, seed=62)
    o8, h8 = gdn2_pallas_forward(*tail, scale, gdn2_state_read(cache, [1, 2]))
    o32, h32 = gdn2_pallas_forward(*tail, scale, h_f)
    assert rel(o8, o32) < 0.02 and rel(h8, h32) < 0.02


@pytest.mark.parametrize("T,H,D,dtype", [(3, 4, 128, torch.bfloat16), (4, 8, 128, torch.float32),
                                         (5, 5, 64, torch.float32), (17, 2, 64, torch.bfloat16),
                                         (64, 2, 128, torch.float32)])
def test_several_tokens_of_a_full_batch(T, H, D, dtype):
    """More CTAs than the GPU holds and many tokens a call, so that the warps of a
    CTA drift apart: every run gives the same bits, those of the float64 tokens."""
    B = 512
    args, scale = tokens(B, T, H, D, dtype, seed=63 + T)
    cache = Gdn2StateCache(2 * B, H, D)
    gdn2_state_write(cache, states(B, H, D, seed=15), list(range(B)))
    src = torch.arange(B, device="cuda", dtype=torch.int32)
    dst = src + B
    o = gdn2_decode_cached(*args, scale, cache, src, dst)
    h = gdn2_state_read(cache, dst)
    for _ in range(10):
        cache.codes[B:].zero_()
        assert torch.equal(o, gdn2_decode_cached(*args, scale, cache, src, dst))
        assert torch.equal(h, gdn2_state_read(cache, dst))
    rows = [0, 1, 200, 293, 511]
    o_r, h_r = oracle([t[rows] for t in args], scale, gdn2_state_read(cache, rows))
    assert rel(o[rows], o_r) < 1e-5
    check_state(h[rows], h_r)


def hold():
    """Keeps the current stream busy for some milliseconds, so that what a call
    leaves to it has not run when the call returns."""
    torch.cuda._sleep(20_000_000)


def test_pinned_host_buffers_may_be_refilled_after_a_call():
    """A call that returns nothing to the host has read its host arguments when it
    returns, whatever its stream still has to do."""
    h, x = states(2, 2, 64, seed=16).cpu().pin_memory(), torch.randn(3, 128).pin_memory()
    want_h, want_x = values64(h).cuda(), values64(x)
    cache = Gdn2StateCache(4, 2, 64)
    args, scale = tokens(2, 1, 2, 64, seed=64)
    want_o = gdn2_decode_cached(*args, scale, cache, [0, 1], [2, 3])
    pinned = [t.cpu().pin_memory() for t in args[1:]]
    at, to = (torch.tensor(t, device="cuda", dtype=torch.int32) for t in ([0, 1], [2, 3]))
    hold()
    gdn2_state_write(cache, h, at)   # (slots on the host would be waited for)
    h.fill_(7.0)
    hold()
    kept = gdn2_checkpoint_pack(x)
    x.fill_(7.0)
    assert torch.equal(gdn2_state_read(cache, at), want_h)
    assert torch.equal(gdn2_checkpoint_unpack(kept)[0], want_x)
    cache.codes.zero_()
    hold()
    o = gdn2_decode_cached(args[0], *pinned, scale, cache, at, to)
    for t in pinned:
        t.fill_(7.0)
    assert torch.equal(o, want_o)


def test_captured_write_reads_its_pinned_states_when_it_is_replayed():
    h = states(1, 2, 64, seed=17).cpu().pin_memory()
    cache, at = Gdn2StateCache(2, 2, 64), torch.tensor([1], device="cuda", dtype=torch.int32)
    gdn2_state_write(cache, h, at)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gdn2_state_write(cache, h, at)
    h.mul_(-3.0)
    g.replay()
    assert torch.equal(gdn2_state_read(cache, at), values64(h).cuda())


def test_ties_and_their_neighbours_at_the_top_of_the_range():
    """Groups whose largest value is next to float32's largest, where its
    reciprocal is below the normal range: values on every half step and one
    float32 step to either side of it, and one pair that such a reciprocal puts
    on the wrong side (126.4999944 steps)."""
    gen = torch.Generator().manual_seed(65)
    tops = 2.0 ** (126 + 2 * torch.rand(2000, generator=gen, dtype=torch.float64))
    tops = torch.cat([tops.float(), torch.tensor([2.0 ** 126, 2.0 ** 127, 2e38, 3e38,
                                                  torch.finfo(torch.float32).max])])
    half = (torch.arange(-127, 127) + 0.5)[1:-1].double() * tops.double().view(-1, 1) / 127.0
    half = half.float()
    far = torch.full_like(half, float("inf"))
    x = torch.stack([half, torch.nextafter(half, far), torch.nextafter(half, -far)], 1)
    x = x.view(len(tops), -1, 63)
    x = torch.cat([x, tops.view(-1, 1, 1).expand(-1, x.shape[1], 1)], 2)
    pair = torch.zeros(1, x.shape[1], 64)
    pair[..., 0], pair[..., 1] = 3.3592143e38, 3.372492e38
    x = torch.cat([x, pair]).cuda()
    assert torch.isfinite(x).all()
    kept = gdn2_checkpoint_pack(x)
    codes, scales = pack64(x)
    assert torch.equal(kept.codes[0].long(), codes) and torch.equal(kept.scales[0], scales)


@pytest.mark.parametrize("D,bt,bc", [(64, 64, 16), (64, 256, 128), (256, 256, 128)])
def test_gdn2_int8_backward_runs_under_the_settings_of_its_forward(D, bt, bc):
    """Settings that change between the passes change nothing of the gradients, and
    stay as they were changed."""
    raw = D == 64   # a head dim of 256 takes activated gates alone
    gdn2_fwd.BT, gdn2_fwd.BC, gdn2_fwd.CLIP = 64, 16, 0.5
    gdn2_fwd.GATES = "raw" if raw else "activated"
    inp = make_inputs(1, 128, 2, D, seed=66, h0_std=0.1)
    args = [torch.as_tensor(inp[n]).cuda() for n in NAMES]
    gen = torch.Generator().manual_seed(67)
    if raw:
        args[3:] = [torch.randn(1, 128, 2, D, generator=gen).cuda() for _ in range(3)]
    do, dh = (torch.as_tensor(inp[n]).cuda() for n in ("dout", "dh_final"))
    leaves = [t.clone().requires_grad_(True) for t in args]

    def run():
        return gdn2_pallas_forward_trainable(*leaves, inp["scale"], checkpoint="int8")

    want = torch.autograd.grad(run(), leaves, (do, dh))
    out = run()
    gdn2_fwd.BT, gdn2_fwd.BC, gdn2_fwd.CLIP = bt, bc, 1e4
    gdn2_fwd.GATES = "activated" if raw else "raw"
    got = torch.autograd.grad(out, leaves, (do, dh))
    for n, a, b in zip(NAMES, got, want):
        assert torch.equal(a, b), n
    assert (gdn2_fwd.BT, gdn2_fwd.BC, gdn2_fwd.CLIP) == (bt, bc, 1e4)
    assert gdn2_fwd.GATES == ("activated" if raw else "raw")


@pytest.mark.parametrize("T", [1, 2])
def test_a_state_that_overflows_without_a_clip_reads_back_as_nan(T):
    """CLIP of infinity: a group that holds an infinity is NaN throughout, as in a
    pack or a write, and reads as 0 in the next decode; its neighbours are right."""
    gdn2_fwd.CLIP = float("inf")
    args, scale = tokens(1, T, 1, 128, seed=68)
    for t in args:
        t[:, :-1] = 0   # tokens before the last leave the zero state
    q, k, v, w, b, g = args
    k[0, -1, 0, 3], v[0, -1, 0, 5], w[0, -1, 0, 5] = 4.0, 3e38, 1.0
    cache = Gdn2StateCache(2, 1, 128)
    gdn2_decode_cached(*args, scale, cache, [0], [1])
    h = gdn2_state_read(cache, [1])[0, 0]
    assert torch.isnan(h[3, :64]).all()
    h[3, :64] = 0
    want = (k[0, -1, 0].double().unsqueeze(1) * (w * v)[0, -1, 0].double())
    want[3, :64] = 0
    check_state(h.view(1, 1, 128, 128), want.view(1, 1, 128, 128).cpu())
    # the group counts as 0 from now on; in the other rows column 5 has rounded its
    # neighbours away
    more, _ = tokens(1, 1, 1, 128, seed=69)
    o = gdn2_decode_cached(*more, scale, cache, [1], [-1])
    h0 = gdn2_state_read(cache, [1])
    h0[..., :64] = 0
    o_r, _ = oracle(more, scale, h0, float("inf"))
    assert rel(o[..., 6:], o_r[..., 6:]) < 1e-5
