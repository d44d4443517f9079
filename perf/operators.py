"""The operators beside the GDN-2 chunk kernels, as cases that can be timed and checked.

Four operators, each in its plain form (elementary torch operations) and as the
calls a user makes of the package:

  recurrence   h_t = e^{g_t} h_{t-1} + w_t v_t per channel (gdn2_linear_recurrence,
               gdn2_linear_recurrence_trainable and its int8-checkpointed backward)
  checkpoint   tensors packed to int8 with a float32 scale per 64 values and
               restored (gdn2_checkpoint_pack / gdn2_checkpoint_unpack)
  state        recurrent states written to and read from an int8 cache by slot
               (gdn2_state_write / gdn2_state_read)
  decode       GDN-2 tokens run from and back into that cache (gdn2_decode_cached)

int8 form of a group of 64 values x: code = rint(127 x / max|x|) with ties to
even, decided exactly; scale = max|x| / 127 in float32; value = code * scale.
"""
import math
import os
import sys

import torch

own = False

GROUP = 64      # values that share a scale
INTERVAL = 64   # tokens between the states that the recurrence's backward restarts from
CLIP = 1e4      # the package's default sanitiser bound
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    path = os.path.join(_ROOT, "gdn2-jax-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gdn2_package
    return gdn2_package


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one generated token for each of a serving batch
        dict(name="recurrence token", op="recurrence", B=64, T=1, H=6, D=128, dtype="float32", train=False, int8=False),
        # a prompt of odd length through a small layer
        dict(name="recurrence prompt bf16", op="recurrence", B=3, T=1021, H=5, D=64, dtype="bfloat16", train=False, int8=False),
        # a training step at the benchmark's main shape
        dict(name="recurrence train", op="recurrence", B=8, T=8192, H=6, D=128, dtype="float32", train=True, int8=False),
        # a training step on one long sequence, the benchmark's long-context shape
        dict(name="recurrence train long bf16", op="recurrence", B=1, T=131072, H=8, D=128, dtype="bfloat16", train=True, int8=False),
        # the main shape with the activations kept in 8 bits
        dict(name="recurrence train int8", op="recurrence", B=8, T=8192, H=6, D=128, dtype="float32", train=True, int8=True),
        # the same on a ragged bf16 batch
        dict(name="recurrence train int8 ragged", op="recurrence", B=2, T=4099, H=3, D=64, dtype="bfloat16", train=True, int8=True),
        # what a GDN-2 training step keeps for its backward, at the main shape
        dict(name="checkpoint", op="checkpoint", B=8, T=8192, H=6, D=128, dtype="float32"),
        # the same of a short ragged bf16 step
        dict(name="checkpoint small bf16", op="checkpoint", B=2, T=131, H=3, D=64, dtype="bfloat16"),
        # the states of a full serving batch parked and fetched again
        dict(name="state cache", op="state", B=256, S=600, H=6, D=128),
        # one sequence's states parked and fetched again
        dict(name="state cache one row", op="state", B=1, S=5, H=4, D=64),
        # one token for a full serving batch
        dict(name="decode batch", op="decode", B=256, T=1, H=8, D=128, dtype="bfloat16"),
        # a few tokens at once (a drafted run) for a small batch
        dict(name="decode few tokens", op="decode", B=3, T=5, H=6, D=64, dtype="float32"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "checkpoint", "state", "decode"])
    D = rng.choice([64, 128])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "state":
        B = _log(rng, 1, 256)
        return dict(op=op, B=B, S=B + _log(rng, 1, 350), H=_log(rng, 1, 6), D=D)
    if op == "decode":
        return dict(op=op, B=_log(rng, 1, 256), T=_log(rng, 1, 5), H=_log(rng, 1, 8), D=D, dtype=dtype)
    H = _log(rng, 1, 8)
    # a case holds at most the values of the main training shape
    most = 8 * 8192 * 6 * 128 // (H * D)
    T = _log(rng, 1, min(most, 131072) if op == "recurrence" else 8192)
    B = _log(rng, 1, max(1, min(64, most // T)))
    if op == "checkpoint":
        return dict(op=op, B=B, T=T, H=H, D=D, dtype=dtype)
    train = rng.random() < 0.7
    return dict(op=op, B=B, T=T, H=H, D=D, dtype=dtype, train=train, int8=train and rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = torch.float32 if case["op"] == "state" else getattr(torch, case["dtype"])

    def nrm(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    B, H, D, op = case["B"], case["H"], case["D"], case["op"]
    s = dict(case=dict(case))
    if op == "state":
        s["h"] = _state(nrm, B, H, D)
        s["slots"] = torch.randperm(case["S"], generator=gen, device="cuda")[:B].to(torch.int32)
        if own:
            s["cache"] = _package().Gdn2StateCache(case["S"], H, D, device="cuda")
        return s
    T = case["T"]
    shape = (B, T, H, D)
    if op == "recurrence":
        # slow and fast channels: e^g from about 0.5 to 0.9995
        s["v"] = nrm(*shape).to(dt)
        s["w"] = torch.sigmoid(nrm(*shape)).to(dt)
        s["g"] = (-torch.nn.functional.softplus(1.5 * nrm(*shape) - 3.0)).to(dt)
        s["h0"] = nrm(B, H, D)
        if case["train"]:
            s["do"] = nrm(*shape)
            s["dh"] = nrm(B, H, D)
            for n in ("v", "w", "g", "h0"):
                s[n].requires_grad_(True)
        return s
    unit = torch.nn.functional.normalize
    s["q"] = unit(nrm(*shape), dim=-1).to(dt)
    s["k"] = unit(nrm(*shape), dim=-1).to(dt)
    s["v"] = nrm(*shape).to(dt)
    s["w"] = torch.sigmoid(nrm(*shape)).to(dt)
    s["b"] = torch.sigmoid(nrm(*shape)).to(dt)
    if op == "checkpoint":
        return s
    s["g"] = (-torch.nn.functional.softplus(1.5 * nrm(*shape) - 3.0)).to(dt)
    # the batch's states in slots of their own, and as many free slots for the states after the tokens
    order = torch.randperm(2 * B, generator=gen, device="cuda").to(torch.int32)
    s["src"], s["dst"] = order[:B].contiguous(), order[B:].contiguous()
    s["codes"] = torch.zeros((2 * B, H, D, D), dtype=torch.int8, device="cuda")
    s["scales"] = torch.zeros((2 * B, H, D, D // GROUP), dtype=torch.float32, device="cuda")
    codes, scales = _pack(_state(nrm, B, H, D))
    s["codes"][s["src"].long()] = codes.to(torch.int8).view(B, H, D, D)
    s["scales"][s["src"].long()] = scales.view(B, H, D, D // GROUP)
    if own:
        s["cache"] = _package().Gdn2StateCache.from_tensors(s["codes"], s["scales"])
    return s


def _state(nrm, B, H, D):
    """Recurrent states, whose key rows differ in size."""
    return 0.1 * nrm(B, H, D, D) * torch.exp(0.5 * nrm(B, H, D, 1))


# ---------------------------------------------------------------- plain forms

def _pack(x):
    """Codes (whole numbers in float64) and scales of x in groups of 64 along its last axis."""
    x = x.detach().float().unflatten(-1, (-1, GROUP))
    top = x.abs().amax(-1, keepdim=True)
    fits = torch.isfinite(top)
    small = top < 2.0 ** -100
    # in 64 bits: a quotient next to a half has to fall on its right side
    codes = torch.round(x.double() * 127.0 / top.double())
    codes = torch.where(fits & ~small, codes, torch.zeros_like(codes))
    scales = (top.double() / 127.0).float()
    scales = torch.where(small, torch.zeros_like(scales), scales)
    scales = torch.where(fits, scales, torch.full_like(scales, float("nan")))
    return codes.flatten(-2), scales.squeeze(-1)


def _unpack(codes, scales):
    return (codes.float().unflatten(-1, (-1, GROUP)) * scales.unsqueeze(-1)).flatten(-2)


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along axis 1 from zero, by doubling."""
    step, n = 1, a.shape[1]
    while step < n:
        x = torch.cat([x[:, :step], x[:, step:] + a[:, step:] * x[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return x


def _from(a, x, h0):
    x = x.clone()
    x[:, 0] += a[:, 0] * h0
    return _scan(a, x)


def _plain_recurrence(s):
    case = s["case"]
    v, w, g = (s[n].detach().float() for n in ("v", "w", "g"))
    h0 = s["h0"].detach()
    a = torch.exp(g)
    h = _from(a, w * v, h0)
    out = dict(o=h, h=h[:, -1])
    if not case["train"]:
        return out
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    if case["int8"]:
        # the backward's states restart from the kept ones every INTERVAL tokens and run on the 8-bit values
        v, w = _unpack(*_pack(s["v"])), _unpack(*_pack(s["w"]))
        B, T, H, D = v.shape
        n = -(-T // INTERVAL)
        pad = (0, 0, 0, 0, 0, n * INTERVAL - T)
        cut = lambda t: torch.nn.functional.pad(t, pad).reshape(B * n, INTERVAL, H, D)  # noqa: E731
        kept = before[:, ::INTERVAL].reshape(B * n, H, D)
        again = _from(cut(a), cut(w * v), kept)
        before = torch.cat([kept.unsqueeze(1), again[:, :-1]], 1).reshape(B, n * INTERVAL, H, D)[:, :T]
    x = s["do"].clone()
    x[:, -1] += s["dh"]
    back = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _scan(back.flip(1), x.flip(1)).flip(1)
    dt = s["v"].dtype
    out.update(dv=(w * dh).to(dt), dw=(v * dh).to(dt), dg=(a * before * dh).to(dt), dh0=a[:, 0] * dh[:, 0])
    return out


def _san(x):
    return torch.nan_to_num(x, nan=0.0, posinf=CLIP, neginf=-CLIP).clamp(-CLIP, CLIP)


def _plain_decode(s):
    q, k, v, w, b, g = (s[n].float() for n in ("q", "k", "v", "w", "b", "g"))
    scale = q.shape[-1] ** -0.5
    src = s["src"].long()
    h = _unpack(s["codes"][src], s["scales"][src])
    outs = []
    for t in range(q.shape[1]):
        e = torch.exp(g[:, t])
        W, qg, kg = _san(b[:, t] * k[:, t] * e), _san(q[:, t] * e), _san(k[:, t])
        u = _san(w[:, t] * v[:, t])
        new = u - (W.unsqueeze(-1) * h).sum(-2)
        qk = _san(scale * (q[:, t] * k[:, t]).sum(-1, keepdim=True))
        outs.append(_san(scale * (qg.unsqueeze(-1) * h).sum(-2) + qk * new))
        h = _san(e.unsqueeze(-1) * h + kg.unsqueeze(-1) * new.unsqueeze(-2))
    return dict(o=torch.stack(outs, 1), state=_unpack(*_pack(h)).to(torch.bfloat16))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    op = s["case"]["op"]
    with torch.no_grad():
        if op == "recurrence":
            return _plain_recurrence(s)
        if op == "decode":
            return _plain_decode(s)
        if op == "state":
            return dict(state=_unpack(*_pack(s["h"])))
        return {n: _unpack(*_pack(s[n])).to(s[n].dtype) for n in ("q", "k", "v", "w", "b")}


# ---------------------------------------------------------------- the package's calls

def _run_own(s):
    p = _package()
    case = s["case"]
    if case["op"] == "recurrence":
        if not case["train"]:
            o, h = p.gdn2_linear_recurrence(s["v"], s["w"], s["g"], s["h0"])
            return dict(o=o, h=h)
        leaves = (s["v"], s["w"], s["g"], s["h0"])
        o, h = p.gdn2_linear_recurrence_trainable(*leaves, checkpoint="int8" if case["int8"] else None)
        dv, dw, dg, dh0 = torch.autograd.grad((o, h), leaves, (s["do"], s["dh"]))
        return dict(o=o, h=h, dv=dv, dw=dw, dg=dg, dh0=dh0)
    if case["op"] == "decode":
        o = p.gdn2_decode_cached(s["q"], s["k"], s["v"], s["w"], s["b"], s["g"], case["D"] ** -0.5,
                                 s["cache"], s["src"], s["dst"])
        return dict(o=o, state=p.gdn2_state_read(s["cache"], s["dst"], dtype=torch.bfloat16))
    if case["op"] == "state":
        p.gdn2_state_write(s["cache"], s["h"], s["slots"])
        return dict(state=p.gdn2_state_read(s["cache"], s["slots"]))
    names = ("q", "k", "v", "w", "b")
    kept = p.gdn2_checkpoint_pack(*(s[n] for n in names))
    return dict(zip(names, p.gdn2_checkpoint_unpack(kept)))


# ---------------------------------------------------------------- bytes and operations

def work(case):
    B, H, D, op = case["B"], case["H"], case["D"], case["op"]
    if op == "state":
        n = B * H * D * D
        form = 1 + 4 / GROUP
        return dict(bytes=n * (4 + form + form + 4), flops=4 * n)
    n = B * case["T"] * H * D
    e = 4 if case["dtype"] == "float32" else 2
    form = 1 + 4 / GROUP
    if op == "checkpoint":
        return dict(bytes=5 * n * (e + form + form + e), flops=20 * n)
    if op == "decode":
        # the states read and written in 8 bits, and the bf16 copy that is returned
        m = B * H * D * D
        return dict(bytes=m * (form + form + 2) + n * (6 * e + 4), flops=8 * m * case["T"])
    ends = 4 * B * H * D
    if not case["train"]:
        return dict(bytes=n * (3 * e + 4) + 2 * ends, flops=3 * n)
    kept = (2 * form if case["int8"] else 0) + 4 / INTERVAL
    again = (e + 2 * form if case["int8"] else 3 * e) + 4 / INTERVAL
    return dict(bytes=n * (3 * e + 4 + kept + again + 4 + 3 * e) + 4 * ends, flops=16 * n)


# ---------------------------------------------------------------- in 64 bits

def _values64(x):
    """What the 8-bit form of x stands for, from its definition."""
    parts = x.detach().double().reshape(-1, GROUP)
    top = parts.abs().max(dim=1, keepdim=True).values
    step = top / 127.0
    nearest = torch.floor(parts * 127.0 / top + 0.5)
    # floor(y + 1/2) is the upper neighbour of a tie: take the even one
    tie = (parts * 254.0 == (2.0 * nearest - 1.0) * top) & (torch.remainder(nearest, 2.0) != 0)
    nearest = torch.where(tie, nearest - 1.0, nearest)
    return torch.where(top > 0, nearest * step, torch.zeros_like(parts)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "state":
            return dict(state=_values64(s["h"]))
        if op == "checkpoint":
            return {n: _values64(s[n]) for n in ("q", "k", "v", "w", "b")}
        if op == "decode":
            return _exact_decode(s)
        return _exact_recurrence(s)


def _exact_decode(s):
    q, k, v, w, b, g = (s[n].double() for n in ("q", "k", "v", "w", "b", "g"))
    scale = q.shape[-1] ** -0.5
    src = s["src"].long()
    steps = s["scales"][src].double().repeat_interleave(GROUP, dim=-1)
    h = s["codes"][src].double() * steps
    o = torch.empty_like(v)
    for t in range(q.shape[1]):
        # decay the state, take the erase direction's content out, put the new value in, read with q
        decayed = torch.exp(g[:, t])[..., None] * h
        new = w[:, t] * v[:, t] - torch.einsum("bhk,bhkv->bhv", b[:, t] * k[:, t], decayed)
        h = decayed + torch.einsum("bhk,bhv->bhkv", k[:, t], new)
        o[:, t] = scale * torch.einsum("bhk,bhkv->bhv", q[:, t], h)
    return dict(o=o, state=_values64(h))


def _exact_recurrence(s):
    case = s["case"]
    v, w, g = (s[n].detach().double() for n in ("v", "w", "g"))
    h0 = s["h0"].detach().double()
    T = v.shape[1]
    decay, put = torch.exp(g), w * v
    h, o = h0, torch.empty_like(v)
    for t in range(T):
        h = torch.addcmul(put[:, t], decay[:, t], h, out=o[:, t])
    out = dict(o=o, h=o[:, -1])
    if not case["train"]:
        return out
    if case["int8"]:
        v, w = _values64(s["v"]), _values64(s["w"])
        put = w * v
    dv, dw, dg = torch.empty_like(v), torch.empty_like(v), torch.empty_like(v)
    # dg first as the state before each token, then as its gradient
    for t in range(T):
        if t == 0:
            dg[:, 0] = h0
        elif not case["int8"] or t % INTERVAL == 0:
            dg[:, t] = o[:, t - 1]
        else:
            torch.addcmul(put[:, t - 1], decay[:, t - 1], dg[:, t - 1], out=dg[:, t])
    carry = s["dh"].double()
    total = dv
    for t in range(T - 1, -1, -1):
        torch.add(s["do"][:, t].double(), carry, out=total[:, t])
        carry = decay[:, t] * total[:, t]
    dg.mul_(decay).mul_(total)
    torch.mul(v, total, out=dw)
    dv.mul_(w)
    out.update(dv=dv, dw=dw, dg=dg, dh0=carry)
    return out
