"""The gated linear recurrence: both directions against a float64 token loop,
the int8 checkpoints, autograd, differences, CUDA graphs and streams."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

from int8_ref import assert_close, linrec64, values64  # noqa: E402
from gdn2_package import (_lib, gdn2_fwd, gdn2_linear_recurrence,  # noqa: E402
                          gdn2_linear_recurrence_backward, gdn2_linear_recurrence_trainable,
                          gdn2_linear_recurrence_with_residuals)

GRADS = ("dv", "dw", "dg", "dh0")


@pytest.fixture(autouse=True)
def _gates():
    saved = gdn2_fwd.GATES
    yield
    gdn2_fwd.GATES = saved


def make(B, T, H, D, dtype=torch.float32, seed=0, raw=False, h0=True, g_shift=-3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nrm = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x = dict(v=nrm(B, T, H, D), w=nrm(B, T, H, D), g=1.5 * nrm(B, T, H, D) + g_shift)
    if not raw:
        x["w"] = torch.sigmoid(x["w"])
        x["g"] = -torch.nn.functional.softplus(x["g"])
    x = {n: t.to(dtype) for n, t in x.items()}
    x["h0"] = nrm(B, H, D) if h0 else None
    return x, nrm(B, T, H, D), nrm(B, H, D)


def check(x, do, dh, int8=False, raw=False):
    o, h, res = gdn2_linear_recurrence_with_residuals(**x, checkpoint="int8" if int8 else None)
    grads = gdn2_linear_recurrence_backward(res, do, dh)
    v8, w8 = (values64(x["v"]), values64(x["w"])) if int8 else (None, None)
    want = linrec64(x["v"], x["w"], x["g"], x["h0"], do, dh, v8, w8, raw)
    assert o.dtype == h.dtype == grads[3].dtype == torch.float32
    assert_close(o, *want["o"], "o")
    assert_close(h, *want["h"], "h")
    assert torch.equal(h, o[:, -1])
    for name, got in zip(GRADS, grads):
        assert_close(got, *want[name], name)
        assert name == "dh0" or got.dtype == x["v"].dtype


@pytest.mark.parametrize("B,T,H,D", [(1, 1, 1, 64), (3, 1, 5, 128), (2, 7, 3, 64), (1, 63, 1, 256),
                                     (2, 64, 3, 128), (1, 65, 1, 64), (5, 200, 3, 64),
                                     (1, 513, 3, 128), (2, 1029, 1, 64), (1, 4099, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("int8", [False, True])
def test_both_directions(B, T, H, D, dtype, int8):
    x, do, dh = make(B, T, H, D, dtype, seed=T + H)
    check(x, do, dh, int8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("int8", [False, True])
def test_raw_gates(dtype, int8):
    gdn2_fwd.GATES = "raw"
    x, do, dh = make(2, 150, 3, 64, dtype, seed=5, raw=True)
    check(x, do, dh, int8, raw=True)


def test_raw_gates_at_their_ends():
    """Pre-activations far out on both sides: e^g of 1 and of 0, w of 0 and 1."""
    gdn2_fwd.GATES = "raw"
    x, do, dh = make(1, 96, 1, 64, seed=6, raw=True)
    far = torch.tensor([-float("inf"), -200.0, -30.0, 30.0, 90.0, 200.0], device="cuda")
    x["g"].view(-1)[:6 * 64] = far.repeat_interleave(64)
    x["w"].view(-1)[64 * 6:64 * 12] = far.clamp(-80, 80).repeat_interleave(64)
    check(x, do, dh, raw=True)


@pytest.mark.parametrize("T", [40, 64, 300])
def test_restarts_and_fast_and_slow_decay(T):
    """g of -inf restarts the state; g of 0 keeps it; g of -1e4 is a restart too."""
    x, do, dh = make(2, T, 2, 64, seed=7)
    x["g"][:, T // 3] = -float("inf")
    x["g"][:, T // 2, 0] = -1e4
    x["g"][0, :, 1] = 0.0
    check(x, do, dh)
    o, _ = gdn2_linear_recurrence(**x)
    fresh = torch.isinf(x["g"])
    assert fresh.any() and torch.equal(o[fresh], (x["w"] * x["v"])[fresh])


def test_padded_tokens_leave_the_state():
    """Zero tokens (v = w = g = 0) behind a sequence change nothing before them
    and keep the state.  Its bits may differ: on the way through the padded
    tiles it is formed from joined maps, whose 2 roundings a join the bound of
    linrec64 counts."""
    x, do, dh = make(2, 130, 2, 128, seed=8)
    for n in ("v", "w", "g"):
        x[n][1, 77:] = 0
    o, h = gdn2_linear_recurrence(**x)
    short = {n: t[1:, :77] if n != "h0" else t[1:] for n, t in x.items()}
    o1, h1 = gdn2_linear_recurrence(**short)
    assert torch.equal(o[1:, :77], o1)
    want = linrec64(short["v"], short["w"], short["g"], short["h0"])
    assert_close(h1, *want["h"], "h")
    assert_close(h[1:], *want["h"], "h of the padded row")


def test_no_state_no_final_gradient_and_segments():
    """h0 and dh_final may be missing; a sequence in two calls is the sequence."""
    x, do, _ = make(2, 200, 3, 64, seed=9, h0=False)
    check(x, do, None)
    o, h = gdn2_linear_recurrence(**x)
    a = {n: t[:, :90] for n, t in x.items() if n != "h0"}
    b = {n: t[:, 90:] for n, t in x.items() if n != "h0"}
    oa, ha = gdn2_linear_recurrence(**a)
    ob, hb = gdn2_linear_recurrence(**b, h0=ha)
    want = linrec64(x["v"], x["w"], x["g"], None)
    assert_close(torch.cat([oa, ob], 1), *want["o"], "o")
    assert_close(hb, *want["h"], "h")


@pytest.mark.parametrize("int8", [None, "int8"])
def test_autograd_is_the_backward(int8):
    x, do, dh = make(2, 150, 2, 64, seed=10)
    o, h, res = gdn2_linear_recurrence_with_residuals(**x, checkpoint=int8)
    want = gdn2_linear_recurrence_backward(res, do, dh)
    leaves = [t.clone().requires_grad_(True) for t in x.values()]
    o2, h2 = gdn2_linear_recurrence_trainable(*leaves, checkpoint=int8)
    got = torch.autograd.grad((o2, h2), leaves, (do, dh))
    assert torch.equal(o, o2) and torch.equal(h, h2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # one output used, one leaf wanted, no h0
    o3, _ = gdn2_linear_recurrence_trainable(leaves[0], x["w"], x["g"], checkpoint=int8)
    (dv,) = torch.autograd.grad(o3, leaves[0], do)
    _, _, res = gdn2_linear_recurrence_with_residuals(x["v"], x["w"], x["g"], checkpoint=int8)
    assert torch.equal(dv, gdn2_linear_recurrence_backward(res, do)[0])
    _, h4 = gdn2_linear_recurrence_trainable(*leaves, checkpoint=int8)
    (dh0,) = torch.autograd.grad(h4, leaves[3], dh)
    assert torch.isfinite(dh0).all()


def test_a_changed_input_is_noticed():
    x, do, dh = make(1, 70, 1, 64, seed=11)
    leaves = [t.clone().requires_grad_(True) for t in x.values()]
    o, h = gdn2_linear_recurrence_trainable(*leaves)
    with torch.no_grad():
        leaves[2].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(o, leaves[0], do)


def test_gradients_against_differences():
    """Central differences of sum(o do) + sum(h dh) in float64 on the values the
    kernel saw, with the truncation error of step e bounded by e^2 times the
    third derivative (v, w, h0 enter linearly; g through exponentials below 1)."""
    x, do, dh = make(1, 70, 1, 64, seed=12)
    _, _, res = gdn2_linear_recurrence_with_residuals(**x)
    grads = gdn2_linear_recurrence_backward(res, do, dh)

    def loss(x):
        r = linrec64(x["v"], x["w"], x["g"], x["h0"])
        return (r["o"][0] * do.double()).sum((0, 1, 2)) + (r["h"][0] * dh.double()).sum((0, 1))

    e = 1e-4
    for name, got in zip(("v", "w", "g", "h0"), grads):
        for t in (0, 5, 63, 64, 69):
            up, dn = ({n: a.double().clone() for n, a in x.items()} for _ in range(2))
            at = (0, 0) if name == "h0" else (0, t, 0)
            up[name][at] += e
            dn[name][at] -= e
            want = (loss(up) - loss(dn)) / (2 * e)   # per channel: channels do not mix
            assert torch.allclose(got[at].double(), want, rtol=1e-4, atol=1e-4), (name, t)
            if name == "h0":
                break


@pytest.mark.parametrize("int8", [None, "int8"])
def test_broadcast_leaves(int8):
    """A gate shared by rows and tokens gets the sum of their gradients."""
    x, do, dh = make(3, 70, 2, 64, seed=18)
    w = x["w"][:1, :1].clone().requires_grad_(True)
    g = x["g"][:1].clone().requires_grad_(True)
    o, h = gdn2_linear_recurrence_trainable(x["v"], w.expand(3, 70, 2, 64), g.expand(3, 70, 2, 64),
                                            x["h0"], checkpoint=int8)
    dw, dg = torch.autograd.grad((o, h), (w, g), (do, dh))
    _, _, res = gdn2_linear_recurrence_with_residuals(
        x["v"], w.detach().expand(3, 70, 2, 64), g.detach().expand(3, 70, 2, 64), x["h0"],
        checkpoint=int8)
    full = gdn2_linear_recurrence_backward(res, do, dh)
    assert torch.equal(dw, full[1].sum((0, 1), keepdim=True))
    assert torch.equal(dg, full[2].sum(0, keepdim=True))


@pytest.mark.parametrize("seed", range(12))
def test_shapes_over_the_range(seed):
    """Sizes drawn over their logarithms, every type, gate form and checkpoint."""
    import random
    rng = random.Random(seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    B, T, H, D = log(1, 40), log(1, 1500), log(1, 9), rng.choice([64, 128, 256])
    raw = rng.random() < 0.3
    gdn2_fwd.GATES = "raw" if raw else "activated"
    x, do, dh = make(B, T, H, D, rng.choice([torch.float32, torch.bfloat16]), seed=seed, raw=raw,
                     h0=rng.random() < 0.7)
    check(x, do, dh, rng.random() < 0.5, raw)


def test_one_tile_for_more_chains_than_the_gpu_holds():
    """600 x 3 groups of one tile: every CTA takes several, dealt out by index."""
    x, do, dh = make(600, 40, 3, 64, seed=19)
    check(x, do, dh)
    check(x, do, dh, int8=True)


def test_more_values_than_31_bits():
    """2^31 values and some: the end of the last row, against the same tokens run
    alone from the state before them."""
    T, H, D = 2 ** 20 + 70, 32, 64
    gen = torch.Generator(device="cuda").manual_seed(20)
    v, w, g = (torch.empty((1, T, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(3))
    for t, lo, hi in ((v, -2, 2), (w, 0, 1), (g, -2, 0)):
        t.uniform_(lo, hi, generator=gen)
    o, h, res = gdn2_linear_recurrence_with_residuals(v, w, g, checkpoint="int8")
    cut = T - 200
    tail = [t[:, cut:].contiguous() for t in (v, w, g)]
    before = o[:, cut - 1].contiguous()
    want = linrec64(*tail, before)
    assert_close(o[:, cut:], *want["o"], "o")
    assert torch.equal(h, o[:, -1])
    do = torch.zeros_like(o)
    do[:, -200:].uniform_(-1, 1, generator=gen)
    dv, dw, dg, _ = gdn2_linear_recurrence_backward(res, do)
    # 200 is no multiple of 64: the tail's states restart elsewhere, so dv alone
    v8, w8 = values64(tail[0]), values64(tail[1])
    want = linrec64(*tail, before, do[:, cut:].contiguous(), None, v8, w8)
    assert_close(dv[:, cut:], *want["dv"], "dv")
    assert_close(dw[:, cut:], *want["dw"], "dw")
    assert bool((dv[:, :cut - 400] == 0).all())   # e^-g sums beyond float32's smallest


def test_strided_mixed_and_host_inputs():
    x, do, dh = make(2, 90, 2, 64, seed=13)
    o, h = gdn2_linear_recurrence(**x)
    wide = torch.randn(2, 90, 2, 3 * 64, device="cuda")
    wide[..., 64:128] = x["v"]
    o2, _ = gdn2_linear_recurrence(wide[..., 64:128], x["w"].transpose(1, 2).contiguous().transpose(1, 2),
                                   x["g"], x["h0"])
    assert torch.equal(o, o2)
    flat = torch.empty(x["v"].numel() + 1, device="cuda")
    odd = flat[1:].view(x["v"].shape).copy_(x["v"])   # 4 bytes off a 16-byte boundary
    assert torch.equal(o, gdn2_linear_recurrence(odd, x["w"], x["g"], x["h0"])[0])
    oc, hc = gdn2_linear_recurrence(*[t.cpu() for t in x.values()])
    assert oc.device.type == "cpu" and torch.equal(oc, o.cpu()) and torch.equal(hc, h.cpu())
    # one float32 input makes the call float32; each gradient has its input's type
    vb = x["v"].to(torch.bfloat16)
    om, _, res = gdn2_linear_recurrence_with_residuals(vb, x["w"], x["g"], x["h0"])
    assert torch.equal(om, gdn2_linear_recurrence(vb.float(), x["w"], x["g"], x["h0"])[0])
    gm = gdn2_linear_recurrence_backward(res, do, dh)
    assert gm[0].dtype == torch.bfloat16 and gm[1].dtype == torch.float32


def test_same_answer_every_time_and_on_another_stream():
    x, do, dh = make(4, 3000, 3, 128, seed=14)

    def step():
        o, h, res = gdn2_linear_recurrence_with_residuals(**x, checkpoint="int8")
        return (o, h, *gdn2_linear_recurrence_backward(res, do, dh))

    first = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):   # two calls at once
        got = step()
    with torch.cuda.stream(other):
        more = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, got, more))


@pytest.mark.parametrize("T", [1, 60, 700])
def test_captured_and_replayed(T):
    x, do, dh = make(2, T, 2, 64, seed=15)

    def step():
        o, h, res = gdn2_linear_recurrence_with_residuals(**x)
        return (o, h, *gdn2_linear_recurrence_backward(res, do, dh))

    step()
    torch.cuda.synchronize()
    graphs = []
    pool = torch.cuda.graph_pool_handle()
    for _ in range(2):   # two graphs on one pool: the second reuses the first's scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = step()
        graphs.append((g, out))
    y, _, _ = make(2, T, 2, 64, seed=16)
    for n in x:
        x[n].copy_(y[n])
    want = step()
    for g, out in graphs * 2:
        for o in out:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_a_wait_that_runs_out_is_reported(monkeypatch):
    """A bounded wait for a word that nothing publishes gives up, is in the
    status, and the same scratch and context serve the next call."""
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    ws = torch.empty(lib.gdn2_recur_workspace_bytes(1, 200, 1, 64), dtype=torch.uint8, device="cuda")
    assert lib.gdn2_selftest_recur_timeout(ws.data_ptr(), ws.numel(), 64, stream) == _lib.OK
    assert _lib.workspace_status(ws, stream) == _lib.STATUS_WAIT_TIMEOUT
    with pytest.raises(_lib.Gdn2Error, match="timed out"):
        _lib.check_status(ws, stream, "recurrence", synced=True)
    monkeypatch.setattr(_lib, "CHECK_STATUS", "always")
    x, do, dh = make(1, 200, 1, 64, seed=21)
    check(x, do, dh)
    assert _lib.LAST_STATUS == 0


def test_long_sequence_of_slow_decay():
    """131072 tokens of one head, decays near 1: the joins over 2048 tiles."""
    x, do, dh = make(1, 131072, 1, 64, seed=17, g_shift=-7.0)
    o, h, res = gdn2_linear_recurrence_with_residuals(**x)
    dv, _, _, dh0 = gdn2_linear_recurrence_backward(res, do, dh)
    a, put = torch.exp(x["g"].double()), (x["w"].double() * x["v"].double())
    want = torch.empty_like(put)
    s = x["h0"].double()
    for t in range(131072):
        s = torch.addcmul(put[:, t], a[:, t], s, out=want[:, t])
    # terms k tokens back are off by 32 (k + 1) U and weigh a^k: about 32 U / (1 - a) of the sum
    rel = float((o.double() - want).norm() / want.norm())
    assert rel < 1e-5, rel
    c = dh.double()
    for t in range(131071, -1, -1):
        d = do[:, t].double() + c
        put[:, t] = x["w"][:, t].double() * d
        c = a[:, t] * d
    rel = float((dv.double() - put).norm() / put.norm())
    assert rel < 1e-5, rel
    assert torch.allclose(dh0.double(), c, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("T", [1, 15, 16, 17, 32, 33])
def test_few_tokens(T):
    """The serial walk of short calls, with and without kept states, beside the
    tiles (int8 always takes them)."""
    x, do, dh = make(5, T, 3, 64, seed=30 + T)
    o, h = gdn2_linear_recurrence(**x)
    o1, h1, _ = gdn2_linear_recurrence_with_residuals(**x)
    assert torch.equal(o, o1) and torch.equal(h, h1)
    check(x, do, dh)
    check(x, do, dh, int8=True)


def test_pinned_host_buffers_may_be_refilled_after_a_call():
    """Host arguments beside tensors on the GPU have been read when the call returns."""
    x, do, dh = make(2, 70, 2, 64, seed=22)
    o, h, res = gdn2_linear_recurrence_with_residuals(**x)
    want = gdn2_linear_recurrence_backward(res, do, dh)
    w, h0, d = (t.cpu().pin_memory() for t in (x["w"], x["h0"], do))
    torch.cuda._sleep(20_000_000)   # some milliseconds, in which no copy starts
    got = gdn2_linear_recurrence(x["v"], w, x["g"], h0)
    w.fill_(7.0)
    h0.fill_(7.0)
    assert torch.equal(o, got[0]) and torch.equal(h, got[1])
    torch.cuda._sleep(20_000_000)
    got = gdn2_linear_recurrence_backward(res, d, dh)
    d.fill_(7.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("int8", [None, "int8"])
@pytest.mark.parametrize("T", [40, 64, 150])
def test_raw_gates_that_are_open_or_shut_have_their_slope(T, int8):
    """dw = v dh sigmoid(x) sigmoid(-x) to float32's relative precision at both ends,
    where sigmoid(x) itself is 1 to float32's precision from x = 17 on."""
    gdn2_fwd.GATES = "raw"
    x, do, dh = make(2, T, 2, 64, seed=23, raw=True)
    at = torch.linspace(-80, 80, 64, device="cuda")   # a channel each
    x["w"] = at.expand(2, T, 2, 64).contiguous()
    x["g"].fill_(float("inf"))   # e^g of 0: dh is dout (and dh_final at the end)
    _, _, res = gdn2_linear_recurrence_with_residuals(**x, checkpoint=int8)
    _, dw, _, _ = gdn2_linear_recurrence_backward(res, do, dh)
    v, w = (values64(x["v"]), values64(x["w"])) if int8 else (x["v"], x["w"])
    d = do.clone()
    d[:, -1] += dh   # one rounding, as in the kernel
    w = w.double()
    want = v.double() * d.double() * torch.sigmoid(w) * torch.sigmoid(-w)
    # e^{-|x|} is off by 2^-22 and the rounding of its exponent, |x| 2^-23 at most with
    # that of log2 e; 1 / (1 + e^{-|x|}) by 2^-22, twice; products by 2^-24, four of them
    size = want.abs() * ((2 * w.abs() + 4 + 8 + 4) * 2.0 ** -24)
    err = (dw.double() - want).abs()
    assert bool((err <= size + 2.0 ** -140).all()), float((err / want.abs()).max())


def test_a_wait_that_ran_out_ends_the_others():
    """A wait of the full limit (about two seconds) ends within some thousand polls
    of another's that ran out."""
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    ws = torch.empty(1024, dtype=torch.uint8, device="cuda")
    for polls in (1, 64, 5000):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        assert lib.gdn2_selftest_recur_timeout(ws.data_ptr(), ws.numel(), polls, stream) == _lib.OK
        end.record()
        assert _lib.workspace_status(ws, stream) == _lib.STATUS_WAIT_TIMEOUT
        assert start.elapsed_time(end) < 300
