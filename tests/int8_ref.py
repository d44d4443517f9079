"""float64 restatements of the int8 form and of the linear recurrence, for the
tests (test infrastructure only)."""
import torch

U = 2.0 ** -24   # half a step of float32


def pack64(x):
    """(codes, scales) of x in groups of 64 along the last axis, by the
    definition; codes int64, scales float32."""
    g = x.double().unflatten(-1, (-1, 64))
    top = g.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top) & (top >= 2.0 ** -100)
    y = g * 127.0 / torch.where(ok, top, torch.ones_like(top))
    codes = torch.where(ok, torch.round(y), torch.zeros_like(y))
    # the definition in whole numbers: 254 x against (2 code +- 1) max
    tie = (g * 254.0).abs() == (2.0 * codes.abs() + 1.0) * top
    assert not bool((tie & ok & (codes.abs() % 2 == 1)).any())
    t32 = top.float()
    scales = torch.where(ok, t32 / torch.full_like(t32, 127.0), torch.zeros_like(t32))
    scales = torch.where(torch.isfinite(top), scales, torch.full_like(scales, float("nan")))
    return codes.flatten(-2).long(), scales.squeeze(-1)


def values64(x):
    codes, scales = pack64(x)
    return (codes.float().unflatten(-1, (-1, 64)) * scales.unsqueeze(-1)).flatten(-2)


def linrec64(v, w, g, h0, dout=None, dh=None, v8=None, w8=None, raw=False):
    """The recurrence in float64, token by token: o, h and, with dout, the four
    gradients.  Beside each output the size its float32 error is counted in.

    An output is a sum over k of |x_{t-k}| times k decays.  Every decay carries
    2^-22 = 4 U of its exponential and 1 U of a product, every join of two maps
    2 U; there are k / 8 + 26 joins on the way at most, none for k = 0.  So the
    term is off by (5 k + k / 4 + 52 + 4) U <= 32 (k + 1) U of its size (k = 1:
    61 of 64; k = 0: 4 of 32), and N_t = a N_{t-1} + M_t, M_t = a M_{t-1} + |x_t|
    sums (k + 1) times the terms.  An exponential is off by 2 |g| U more: what
    is left of 32 (k + 1) covers that for g above -13 from k = 2 on, and a term
    one token back of such a g weighs under e^-1.5 of its 2 |g| U."""
    v, w, g = v.double(), w.double(), g.double()
    B, T, H, D = v.shape
    h0 = torch.zeros((B, H, D), dtype=torch.float64, device=v.device) if h0 is None else h0.double()
    a = torch.sigmoid(-g) if raw else torch.exp(g)
    act = torch.sigmoid if raw else (lambda z: z)

    def states(v, w, restart):
        h, M, N, before, nb = h0, h0.abs(), h0.abs(), [], []
        for t in range(T):
            if restart is not None and t % 64 == 0:
                h = restart[t]
            before.append(h)
            nb.append(N)
            x = act(w[:, t]) * v[:, t]
            h = a[:, t] * h + x
            M = a[:, t] * M + x.abs()
            N = a[:, t] * N + M
        return h, N, before, nb

    h, N, before, nb = states(v, w, None)
    out = {"o": (torch.stack(before[1:] + [h], 1), torch.stack(nb[1:] + [N], 1)), "h": (h, N)}
    if dout is None:
        return out
    if v8 is not None:
        v, w = v8.double(), w8.double()
        # the restart states are float32 and carry the error counted in nb, so nb stays an upper bound
        _, _, before, nb8 = states(v, w, before)
        nb = [torch.maximum(x, y) for x, y in zip(nb, nb8)]
    wa = act(w)
    c = torch.zeros_like(h0) if dh is None else dh.double()
    M, N = c.abs(), c.abs()
    keys = ("dv", "dw", "dg")
    got = {k: [None] * T for k in keys}
    size = {k: [None] * T for k in keys}
    for t in range(T - 1, -1, -1):
        d = dout[:, t].double() + c
        M = M + dout[:, t].double().abs()
        N = N + M
        c = a[:, t] * d
        got["dv"][t], size["dv"][t] = wa[:, t] * d, wa[:, t].abs() * (N + d.abs())
        dw, sw = v[:, t] * d, v[:, t].abs() * (N + d.abs())
        dg, sg = before[t] * c, a[:, t] * (before[t].abs() * N + nb[t] * d.abs() + nb[t] * 32 * U * N)
        if raw:
            s = wa[:, t]
            # 1 - w is off by 4 U however small it is
            dw, sw = dw * s * (1 - s), sw * s * (1 - s) + (v[:, t] * d * s).abs()
            dg, sg = -dg * torch.sigmoid(g[:, t]), sg * torch.sigmoid(g[:, t])
        got["dw"][t], size["dw"][t] = dw, sw
        got["dg"][t], size["dg"][t] = dg, sg
        M, N = a[:, t] * M, a[:, t] * N
    for k in keys:
        out[k] = (torch.stack(got[k], 1), torch.stack(size[k], 1))
    out["dh0"] = (c, N)
    return out


def assert_close(got, want, size, name):
    """|got - want| <= 32 U size, and the rounding to got's own type.  Below the
    normal range an operation is off by up to 2^-149 whatever its size; at most
    2^4 of them, multiplied by factors below 2^5, meet in a value."""
    err = (got.double() - want).abs()
    allow = 32 * U * size + 2.0 ** -140
    if got.dtype == torch.bfloat16:
        allow = allow + 2.0 ** -8 * (want.abs() + allow)
    bad = ~(err <= allow)
    assert not bool(bad.any()), (name, int(bad.sum()), float((err - allow).max()),
                                 bad.nonzero()[:3].tolist())
