"""Faults that the sequence operators and the readout once had, each by the smallest call that shows it, against the
definitions in 64 bits."""
import math

import pytest
import torch

from tests.seq_ref import UNIT, f64, near

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rnd(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(DEV)


def slope(p, act):
    """act'(p), also where exp(-p) passes 64 bits."""
    if act == "gelu":
        return 0.5 * torch.erfc(-p / math.sqrt(2.0)) + p * torch.exp(-0.5 * p * p) / math.sqrt(2.0 * math.pi)
    q = torch.sigmoid(p)
    return q * (1.0 + p * (1.0 - q))


def litter(*sizes):
    """Leaves NaN in the memory that torch hands out next for these sizes (bytes)."""
    bad = [torch.full((n // 4,), float("nan"), device=DEV) for n in sizes for _ in range(4)]
    del bad


# ------------------------------------------------------------------------ layer norm ----
@pytest.mark.parametrize("D,dtype", [(64, F32), (8193, BF16), (66_000, BF16), (5000, F32), (66_000, F32)])
def test_layer_norm_of_no_rows(D, dtype):
    """The parameters' gradients are sums of nothing, at every width."""
    from v1_glif_model_amd import sequence as seq
    x = torch.empty(0, D, dtype=dtype, device=DEV, requires_grad=True)
    w, b = (torch.ones(D, device=DEV, requires_grad=True) for _ in range(2))
    y = seq.layer_norm(x, w, b)
    litter(4 * D, 8 * D, 8 * D + 256)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, D) and not dw.any() and not db.any()


@pytest.mark.parametrize("D", [40_000, 66_001])
@pytest.mark.parametrize("value", [0.1, 0.7, 1.2345, -3.3])
def test_layer_norm_of_one_active_neuron(D, value):
    """Wide float32 rows of zeros with one value, first among a thread's own or not: the spread is all that value's."""
    from v1_glif_model_amd import sequence as seq
    x, dy, w = torch.zeros(4, D, device=DEV), rnd(10, 4, D), rnd(11, D, shift=1.0, scale=0.3)
    for r, c in enumerate((0, 4, 1777, D - 1)):
        x[r, c] = value
    xs = x.requires_grad_(True)
    y = seq.layer_norm(xs, w)
    (dx,) = torch.autograd.grad(y, xs, dy)
    x6, g6, w6 = (f64(t, False) for t in (x, dy, w))
    mean = x6.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x6 - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    xh, far = (x6 - mean) * rstd, (x6.abs() + x6.abs().mean(-1, keepdim=True)) * rstd
    near(y, xh * w6, far * w6.abs(), "y")
    gw, ga = g6 * w6, g6.abs() * w6.abs()
    near(dx, rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True)),
         rstd * (ga + ga.mean(-1, keepdim=True) * (1 + far) + far * (ga * far).mean(-1, keepdim=True)), "dx")


@pytest.mark.parametrize("D", [2 ** 30, 2 ** 31 - 1])
def test_layer_norm_of_the_longest_rows(D):
    """Millions of terms a thread, as exact as a hundred; and 2^31 - 1 columns, whose last piece ends where 31 bits do."""
    from v1_glif_model_amd import sequence as seq
    step = 2 ** 28
    x, dy = torch.empty(1, D, dtype=F16, device=DEV), torch.empty(1, D, dtype=F16, device=DEV)
    g = torch.Generator(DEV).manual_seed(12)
    for at in range(0, D, step):
        n = min(step, D - at)
        x[0, at:at + n].copy_(torch.randn(n, generator=g, device=DEV))
        dy[0, at:at + n].copy_(torch.rand(n, generator=g, device=DEV) + x[0, at:at + n])
    xs = x.requires_grad_(True)
    y = seq.layer_norm(xs)
    (dx,) = torch.autograd.grad(y, xs, dy)
    cut = [slice(at, min(at + step, D)) for at in range(0, D, step)]
    with torch.no_grad():
        mean = sum(x[0, c].double().sum() for c in cut) / D
        rstd = 1.0 / torch.sqrt(sum(((x[0, c].double() - mean) ** 2).sum() for c in cut) / D + 1e-5)
        size = sum(x[0, c].double().abs().sum() for c in cut) / D
        sums = [0.0] * 4
        for c in cut:
            xh, far, gw = (x[0, c].double() - mean) * rstd, (x[0, c].double().abs() + size) * rstd, dy[0, c].double()
            sums = [a + float(b) / D for a, b in zip(sums, (gw.sum(), (gw * xh).sum(), gw.abs().sum(), (gw.abs() * far).sum()))]
        for c in (slice(0, 70), slice(D // 2, D // 2 + 70), slice(D - 70, D)):
            x6, gw = x[0, c].double().cpu(), dy[0, c].double().cpu()
            m, r = mean.cpu(), rstd.cpu()
            xh, far = (x6 - m) * r, (x6.abs() + size.cpu()) * r
            near(y[0, c], xh, far, "y")
            near(dx[0, c], r * (gw - sums[0] - xh * sums[1]), r * (gw.abs() + sums[2] * (1 + far) + far * sums[3]), "dx")


def test_layer_norm_of_more_rows_than_a_launch_holds():
    """2^29 rows of two: their threads pass 32 bits.  The last rows are those of a small call."""
    from v1_glif_model_amd import sequence as seq
    x = torch.empty(2 ** 29 + 3, 2, dtype=F16, device=DEV)
    for part in x.split(2 ** 26):
        part.normal_(generator=torch.Generator(DEV).manual_seed(14))
    xs = x.requires_grad_(True)
    y = seq.layer_norm(xs)
    (dx,) = torch.autograd.grad(y, xs, x.detach())
    for part in (slice(0, 100), slice(2 ** 28 - 50, 2 ** 28 + 50), slice(-100, None)):
        own = x.detach()[part].clone().requires_grad_(True)
        few = seq.layer_norm(own)
        assert torch.equal(y[part], few) and torch.equal(dx[part], torch.autograd.grad(few, own, own.detach())[0])


def test_parameters_of_more_channels_than_a_launch_joins():
    """The joins of the parameters' sums, 8 threads a sum: one row's and one tick's gradients are products."""
    from v1_glif_model_amd import sequence as seq
    D = 2 ** 29 + 77
    x = torch.empty(1, D, dtype=F16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(15))
    b = torch.zeros(D, dtype=F16, device=DEV, requires_grad=True)
    (db,) = torch.autograd.grad(seq.layer_norm(x, None, b), b, x)
    assert torch.equal(db, x[0])
    del b, db
    D = 2 ** 26 + 77
    x = x[0, :D].reshape(1, 1, D)
    w = torch.ones(D, 8, dtype=F16, device=DEV, requires_grad=True)
    y, _ = seq.short_conv(x, w)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(y, x) and torch.equal(dw[:, 7], x[0, 0]) and not dw[:, :7].any()


# ---------------------------------------------------------------------------- linear ----
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_keeps_the_activations_argument_in_full(dtype, act):
    """The bias's gradient of a few rows, whose terms are products of dy and the slope alone: off by the float32 sums'
    rounding (1e-5 of dp's terms, of which the slope turns by at most 0.8 per unit), with nothing for an argument in 16 bits
    (which would be 2^-9 and 2^-12 of up to 0.35 dy)."""
    from v1_glif_model_amd import sequence as seq
    M, N, K = 3, 200, 4
    x, w = rnd(1, M, K, dtype=dtype), rnd(2, N, K, dtype=dtype, scale=0.7)
    b, dy = rnd(3, N).requires_grad_(True), rnd(4, M, N, dtype=dtype)
    (db,) = torch.autograd.grad(seq.linear(x, w, b, activation=act), b, dy)
    x6, w6, b6, g6 = (f64(t, False) for t in (x, w, b, dy))
    pre = x6 @ w6.t() + b6
    dp = g6 * slope(pre, act)
    terms = dp.abs() + 0.8 * g6.abs() * (x6.abs() @ w6.abs().t() + b6.abs())
    near(db, dp.sum(0), terms.sum(0), "db")


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_float16_arguments_beyond_float16(act):
    """An argument of -7e4, whose activation is 0 and whose slope is 0, and one of 7e4, whose slope is 1, among ordinary ones."""
    from v1_glif_model_amd import sequence as seq
    M, N, K = 40, 24, 16
    x, w = rnd(5, M, K, dtype=F16), rnd(6, N, K, dtype=F16, scale=0.25)
    x[7], w[5], x[20] = 0.0, 0.0, 0.0
    x[7, 3], w[5, 3], x[20, 3] = -256.0, 274.0, 256.0
    b, dy = rnd(7, N), rnd(8, M, N, dtype=F16)
    xs, ws, bs = (t.requires_grad_(True) for t in (x, w, b))
    y = seq.linear(xs, ws, bs, activation=act)
    assert float(y.detach()[7, 5]) == 0.0
    got = torch.autograd.grad(y, (xs, ws, bs), dy)
    x6, w6, b6, g6 = (f64(t, False) for t in (x, w, b, dy))
    pre = x6 @ w6.t() + b6
    assert float(pre[7, 5]) < -65520 and float(pre[20, 5]) > 65520
    dp = g6 * slope(pre, act)
    # float32 sums; |slope'| <= 0.8 and 0 far out, where the terms are large; dp is rounded once for the products
    turn = torch.where(pre.abs() > 1e4, 0.0, 0.8)
    terms = dp.abs() + turn * g6.abs() * (x6.abs() @ w6.abs().t() + b6.abs())
    one = UNIT[F16] * dp.abs()
    near(got[0], dp @ w6, terms @ w6.abs(), "dx", more=one @ w6.abs())
    near(got[1], dp.t() @ x6, terms.t() @ x6.abs(), "dw", more=one.t() @ x6.abs())
    near(got[2], dp.sum(0), terms.sum(0), "db")


# ----------------------------------------------------------------------- state space ----
def scan_leaves(seed, T, B, D, G, N):
    k = iter(range(seed, seed + 9))
    t = [rnd(next(k), T, B, D), rnd(next(k), T, B, D), -torch.exp(rnd(next(k), D, N)), rnd(next(k), T, B, G, N), rnd(next(k), T, B, G, N),
         rnd(next(k), D), rnd(next(k), T, B, D), rnd(next(k), D), rnd(next(k), B, D, N)]
    return [v.requires_grad_(True) for v in t]


@pytest.mark.parametrize("T", [0, 4, 200])
def test_scan_of_an_empty_batch(T):
    """The shared parameters' gradients are sums of nothing; the others are empty, as they are."""
    from v1_glif_model_amd import sequence as seq
    leaf = scan_leaves(20, T, 0, 6, 2, 16)
    u, delta, A, B, C, D, z, bias, state = leaf
    y, last = seq.state_space_scan(u, delta, A, B, C, D, z, bias, initial_state=state)
    assert y.shape == (T, 0, 6) and last.shape == (0, 6, 16)
    litter(6 * 16 * 4, 6 * 4)
    got = torch.autograd.grad((y, last), leaf, (torch.empty_like(y), torch.empty_like(last)))
    for g, v in zip(got, leaf):
        assert g.shape == v.shape and not g.any()


@pytest.mark.parametrize("D,N", [(70, 16), (3, 4), (5, 64)])
def test_scan_steps_that_the_bias_makes(D, N):
    """Plain steps of 0.25, as delta 20.25 less a bias of 20: with a delta of 0, as where a block has no more channels, the
    decays would be infinite.  B's and C's gradients are sums over the channels that there are."""
    from tests import seq_ref as ref
    from v1_glif_model_amd import sequence as seq
    T, B = 19, 2
    u, dy = rnd(50, T, B, D), rnd(51, T, B, D)
    A, Bm, Cm = -torch.linspace(1.0, 8.0, D * N, device=DEV).view(D, N), rnd(52, T, B, 1, N), rnd(53, T, B, 1, N)
    delta, bias = torch.full((T, B, D), 20.25, device=DEV), torch.full((D,), -20.0, device=DEV)
    leaf = [t.requires_grad_(True) for t in (u, delta, A, Bm, Cm, bias)]
    y, _ = seq.state_space_scan(*leaf[:5], delta_bias=bias, delta_softplus=False)
    got = torch.autograd.grad(y, leaf, dy)
    own = [f64(t) for t in leaf]
    y6, _ = ref.scan(*own[:5], bias=own[5], softplus=False)
    want = torch.autograd.grad(y6, own, f64(dy, False))
    ab = [(t if i in (1, 2, 5) else t.abs()).detach().requires_grad_(True) for i, t in enumerate(own)]
    ya, _ = ref.scan(*ab[:5], bias=ab[5], softplus=False, sums=True)
    near(y, y6, ya.detach(), "y")
    for g, e, s, name in zip(got, want, torch.autograd.grad(ya, ab, f64(dy, False).abs()), ("u", "delta", "A", "B", "C", "bias")):
        near(g, e, s.abs(), "d" + name)


def test_scan_of_growing_states_that_are_zero():
    """Rates above 0, steps of 2, inputs in the last ticks and dy in the first: states and adjoints are 0 over most of 600
    ticks, over which they would grow by e^1200, and finite.  Time is cut into segments here."""
    from tests import seq_ref as ref
    from v1_glif_model_amd import sequence as seq
    T, B, D, N = 600, 1, 3, 16
    u, dy = rnd(60, T, B, D), rnd(61, T, B, D)
    u[:-5], dy[5:] = 0.0, 0.0
    A, Bm, Cm = torch.ones(D, N, device=DEV), rnd(62, T, B, 1, N), rnd(63, T, B, 1, N)
    leaf = [t.requires_grad_(True) for t in (u, torch.full((T, B, D), 2.0, device=DEV), A, Bm, Cm)]
    y, last = seq.state_space_scan(*leaf, delta_softplus=False)
    got = torch.autograd.grad(y, leaf, dy)
    own = [f64(t) for t in leaf]
    y6, last6 = ref.scan(*own, softplus=False)
    want = torch.autograd.grad(y6, own, f64(dy, False))
    ab = [t.detach().abs().requires_grad_(True) for t in own]
    ya, la = ref.scan(*ab, softplus=False, sums=True)
    near(y, y6, ya.detach(), "y")
    near(last, last6, la.detach(), "last")
    assert bool(last.isfinite().all()) and float(last.detach().abs().max()) > 1
    for g, e, s, name in zip(got, want, torch.autograd.grad(ya, ab, f64(dy, False).abs()), ("u", "delta", "A", "B", "C")):
        assert bool(e.isfinite().all())
        near(g, e, s.abs(), "d" + name)


def test_scan_of_growth_past_float32_over_a_segment():
    """A state of 1e-30 that grows by e^96 over the first of two segments of time and by e^6 over the second, and adjoints of
    1e-30 the other way: everything stays within float32, the growth does not."""
    from tests import seq_ref as ref
    from v1_glif_model_amd import sequence as seq
    T, B, D, N = 128, 1, 5, 4
    delta = torch.full((T, B, D), 1.5, device=DEV)
    delta[64:] = 0.1
    t = [rnd(70, T, B, D, scale=1e-30), delta, torch.ones(D, N, device=DEV), rnd(71, T, B, 1, N), rnd(72, T, B, 1, N)]
    state, dy = rnd(73, B, D, N, scale=1e-30), rnd(74, T, B, D, scale=1e-30)
    leaf = [v.requires_grad_(True) for v in (*t, state)]
    y, last = seq.state_space_scan(*leaf[:5], delta_softplus=False, initial_state=state)
    got = torch.autograd.grad(y, leaf, dy)
    own = [f64(v) for v in leaf]
    y6, last6 = ref.scan(*own[:5], softplus=False, state=own[5])
    want = torch.autograd.grad(y6, own, f64(dy, False))
    ab = [v.detach().abs().requires_grad_(True) for v in own]
    ya, la = ref.scan(*ab[:5], softplus=False, state=ab[5], sums=True)
    # a growth of e^96 carries the float32 rounding of its exponent, 2^-24 of 96 a step of the sum: 64 x 96 x 2^-24 = 4e-4
    near(y, y6, 40 * ya.detach(), "y")
    near(last, last6, 40 * la.detach(), "last")
    for g, e, s, name in zip(got, want, torch.autograd.grad(ya, ab, f64(dy, False).abs()), ("u", "delta", "A", "B", "C", "state")):
        near(g, e, 40 * s.abs(), "d" + name)


@pytest.mark.parametrize("T", [16, 21, 700])
def test_scan_of_rates_of_minus_infinity(T):
    """States that keep nothing (exp(log_rate) past float32) hold the last live tick's input, at every length: the ticks behind
    one, and those that fill a chunk of ticks up, leave the state alone."""
    from v1_glif_model_amd import sequence as seq
    B, D, N = 4, 6, 5
    lens = torch.tensor([T, 1, T // 2, T - 1], dtype=torch.int32, device=DEV)
    u, delta, Bm, Cm = rnd(80, T, B, D), rnd(81, T, B, D), rnd(82, T, B, 1, N), rnd(83, T, B, 1, N)
    A = -torch.exp(rnd(84, D, N))
    A[:, 1], A[2] = -math.inf, -math.inf
    for ln in (None, lens):
        end = (ln if ln is not None else torch.full((B,), T, device=DEV)).long() - 1
        y, last = seq.state_space_scan(u, delta, A, Bm, Cm, lengths=ln)
        i = torch.arange(B, device=DEV)
        want = (torch.nn.functional.softplus(delta.double()) * u.double())[end, i][..., None] * Bm.double()[end, i]
        dead = A == -math.inf
        assert bool(y.isfinite().all()) and bool(last.isfinite().all())
        near(last[:, dead], want[:, dead].cpu(), want[:, dead].abs().cpu(), "last")


def test_scan_of_as_many_groups_as_a_launch_holds():
    """2^23 groups of two channels are right to the last; 2^24 of one, whose threads pass 32 bits, are refused."""
    from v1_glif_model_amd import sequence as seq
    G = 2 ** 23
    u, delta = rnd(90, 1, 1, 2).repeat(1, 1, G), rnd(91, 1, 1, 2).repeat(1, 1, G)
    A, maps = -torch.ones(2 * G, 1, device=DEV), torch.ones(1, 1, G, 1, device=DEV)
    maps[..., -1, :] = 3.0
    y, last = seq.state_space_scan(u, delta, A, maps, maps)
    one, end = seq.state_space_scan(u[..., :2].contiguous(), delta[..., :2].contiguous(), A[:2], maps[:, :, :1], maps[:, :, :1])
    assert torch.equal(y[..., :-2].unflatten(-1, (-1, 2)), one.unsqueeze(-2).expand(1, 1, G - 1, 2))
    assert torch.equal(y[..., -2:], 3 * (3 * end.view(1, 1, 2))) and torch.equal(last[:, -2:], 3 * end)
    maps = torch.ones(1, 1, 2 * G, 1, device=DEV)
    with pytest.raises(ValueError, match="groups"):
        seq.state_space_scan(u, delta, A, maps, maps)
    with pytest.raises(ValueError, match="groups"):
        seq.state_space_step(u[0], torch.zeros(1, 2 * G, 1, device=DEV), delta[0], A, maps[0], maps[0])


def test_other_operators_of_an_empty_batch():
    from v1_glif_model_amd import sequence as seq
    x, w, b = (rnd(30, *s).requires_grad_(True) for s in ((7, 0, 12), (12, 4), (12,)))
    st = torch.empty(0, 3, 12, device=DEV, requires_grad=True)
    litter(12 * 4 * 4, 12 * 4)
    y, last = seq.short_conv(x, w, b, "silu", st)
    got = torch.autograd.grad((y, last), (x, w, b, st), (torch.empty_like(y), torch.empty_like(last)))
    assert all(g.shape == v.shape and not g.any() for g, v in zip(got, (x, w, b, st)))
    lw, lb = rnd(31, 5, 12).requires_grad_(True), rnd(32, 5).requires_grad_(True)
    y = seq.linear(x, lw, lb, activation="gelu")
    got = torch.autograd.grad(y, (x, lw, lb), torch.empty_like(y))
    assert y.shape == (7, 0, 5) and all(g.shape == v.shape and not g.any() for g, v in zip(got, (x, lw, lb)))


# ------------------------------------------------------------- forward-mode derivatives ----
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """Every operator on an input with a tangent, and the readout: none may answer as if it had none."""
    from torch.autograd import forward_ad

    from v1_glif_model_amd import sequence as seq
    from v1_glif_model_amd.readout import SequenceReadout
    x, w, cw = rnd(40, 6, 2, 8), rnd(41, 5, 8), rnd(42, 8, 4)
    A, maps = -torch.exp(rnd(43, 8, 4)), rnd(44, 6, 2, 1, 4)
    mem, h = rnd(45, 2, 3, 8), rnd(46, 2, 8, 4)
    mem0, h0 = mem.clone(), h.clone()
    m = SequenceReadout(8, 3, width=16, channels=8, states=4, rank=2, dtype=F32).eval()
    calls = [lambda v: seq.layer_norm(v), lambda v: seq.dropout(v, 0.5, 1), lambda v: seq.dropout(x, 0.5, 1, residual=v),
             lambda v: seq.linear(v, w), lambda v: seq.linear(x, v[0, 0, :, None].expand(8, 8).contiguous()),
             lambda v: seq.short_conv(v, cw), lambda v: seq.short_conv(x, cw, initial_state=v[:2, :, :3].reshape(2, 3, 8)),
             lambda v: seq.state_space_scan(v, x, A, maps, maps), lambda v: seq.state_space_scan(x, x, A, maps, maps, z=v),
             lambda v: seq.short_conv_step(v[0], mem, cw), lambda v: seq.state_space_step(x[0], h, v[0], A, maps[0], maps[0]),
             lambda v: m(v)]
    for k, call in enumerate(calls):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            with pytest.raises((NotImplementedError, RuntimeError)):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
                print("not refused:", k)
    assert torch.equal(mem, mem0) and torch.equal(h, h0)
    with torch.no_grad(), forward_ad.dual_level():      # a level alone changes nothing
        assert torch.equal(seq.layer_norm(x), seq.layer_norm(x.clone().requires_grad_(True)).detach())


# --------------------------------------------------------------------------- the readout ----
def small_readout(dtype, **kw):
    from v1_glif_model_amd.readout import SequenceReadout
    return SequenceReadout(20, 5, width=16, channels=24, states=4, groups=2, taps=3, rank=3, dtype=dtype, seed=4, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("how", ["step", "load"])
def test_ticks_go_on_with_the_readout_their_state_was_made_for(dtype, how):
    """Parameters that change in place between two ticks change nothing for a state that is under way, and all for a new one."""
    import copy
    m = small_readout(dtype).eval()
    old, other = copy.deepcopy(m), small_readout(dtype).eval()
    with torch.no_grad():
        for k, p in other.named_parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=torch.Generator().manual_seed(5)).to(DEV))
    x = rnd(95, 4, 3, 20)
    state, want = m.zero_state(3), old.zero_state(3)
    assert not {t.data_ptr() for t in state.weights.values()} & {p.data_ptr() for p in m.parameters()}
    assert torch.equal(m.tick(x[0], state), old.tick(x[0], want))
    if how == "load":
        m.load_state_dict(other.state_dict())
    else:
        with torch.no_grad():
            for p, q in zip(m.parameters(), other.parameters()):
                p.copy_(q)
    for t in range(1, 4):
        assert torch.equal(m.tick(x[t], state), old.tick(x[t], want)), t
    new, want = m.zero_state(3), other.zero_state(3)
    for t in range(4):
        assert torch.equal(m.tick(x[t], new), other.tick(x[t], want)), t


def test_training_that_is_resumed_goes_on_with_the_masks(tmp_path):
    """A readout saved between two steps and loaded again draws the masks that the saved one would have drawn next."""
    x = rnd(96, 6, 2, 20)
    m = small_readout(F32, dropout=0.5).train()
    m(x)
    torch.save(m.state_dict(), tmp_path / "m.pt")
    new = small_readout(F32, dropout=0.5).train()
    new.load_state_dict(torch.load(tmp_path / "m.pt", weights_only=True))
    assert new.drawn == m.drawn == 6 * 2 * 16
    assert torch.equal(new(x).detach(), m(x).detach())
    assert not torch.equal(new(x).detach(), small_readout(F32, dropout=0.5).train()(x).detach())
    whole = torch.nn.ModuleList([small_readout(F32, dropout=0.5)])
    whole.load_state_dict({"0." + k: v for k, v in m.state_dict().items()})
    assert whole[0].drawn == m.drawn
    named = dict(m.named_parameters())                      # as it was saved before the masks' place was in it
    new.load_state_dict({k: v.detach() for k, v in named.items()})
    assert new.drawn == 3 * 6 * 2 * 16
    with pytest.raises(RuntimeError, match="head_bias"):
        new.load_state_dict({k: v.detach() for k, v in named.items() if k != "head_bias"})


@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing_draws_one_mask(reentrant):
    """A forward that is run again in the backward pass: with its place in the stream the gradients are those of one run, bit
    by bit, whatever ran in between; without it, it is refused."""
    from torch.utils.checkpoint import checkpoint
    m, plain = (small_readout(F32, dropout=0.5).train() for _ in range(2))
    x, y = rnd(97, 6, 2, 20).requires_grad_(True), rnd(98, 7, 2, 20).requires_grad_(True)
    a = checkpoint(m, x, None, m.draw(6, 2), use_reentrant=reentrant)
    b = checkpoint(m, y, None, m.draw(7, 2), use_reentrant=reentrant)
    (a.square().sum() + b.square().sum()).backward()
    got = [x.grad, y.grad, *(p.grad for p in m.parameters())]
    x.grad = y.grad = None
    pa, pb = plain(x), plain(y)
    assert torch.equal(a, pa) and torch.equal(b, pb) and m.drawn == plain.drawn == 13 * 2 * 16
    (pa.square().sum() + pb.square().sum()).backward()
    for g, w in zip(got, [x.grad, y.grad, *(p.grad for p in plain.parameters())]):
        # a parameter's two gradients are added in either order, and are the same
        assert torch.equal(g, w)
    out = checkpoint(m, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="draw"):
        out.sum().backward()
    m.eval()
    checkpoint(m, x, use_reentrant=reentrant).sum().backward()     # no masks, no place
