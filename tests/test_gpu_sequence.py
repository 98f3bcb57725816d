"""GPU parity of the sequence operators (layer norm, dropout, linear, short convolution, state space) with their
definitions in 64 bits (tests/seq_ref.py), at the sizes, strides, lengths and masked places where they can go wrong; their
gradients against the formulas' and against differences; their refusals."""
import math

import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import UNIT, f64, near

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
F32 = torch.float32


def rnd(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(DEV)


def grads(out, dout, *wrt):
    return torch.autograd.grad(out, [t for t in wrt if t is not None], dout, allow_unused=True)


# ------------------------------------------------------------------------ layer norm ----
def norm_case(x, w, b, dy, eps=1e-5):
    from v1_glif_model_amd import sequence as seq
    xs, ws, bs = (None if t is None else t.detach().requires_grad_(True) for t in (x, w, b))
    y = seq.layer_norm(xs, ws, bs, eps)
    assert torch.equal(y.detach(), seq.layer_norm(x, w, b, eps))
    got = list(grads(y, dy, xs, ws, bs))
    x6, w6, b6 = f64(x), f64(w), f64(b)
    y6 = ref.layer_norm(x6, w6, b6, eps)
    want = list(grads(y6, f64(dy, False), x6, w6, b6))
    with torch.no_grad():
        one = torch.ones((), dtype=ref.F64)
        wa = one if w is None else w6.abs()
        mean = x6.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt(((x6 - mean) ** 2).mean(-1, keepdim=True) + eps)
        far = (x6.abs() + x6.abs().mean(-1, keepdim=True)) * rstd      # what the mean's rounding weighs against
        ga = f64(dy, False).abs() * wa
        near(y, y6, far * wa + (0.0 if b is None else b6.abs()), "y")
        near(got.pop(0), want.pop(0), rstd * (ga + ga.mean(-1, keepdim=True) * (1 + far) + far * (ga * far).mean(-1, keepdim=True)), "dx")
        lead = tuple(range(x.dim() - 1))
        if w is not None:
            near(got.pop(0), want.pop(0), (f64(dy, False).abs() * far).sum(lead), "dw")
        if b is not None:
            near(got.pop(0), want.pop(0), f64(dy, False).abs().sum(lead), "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (5, 512), (3, 7), (17, 64), (33, 1000), (9, 1025), (6, 4097), (3, 8192), (4, 12007),
                                   (2, 66000), (1, 131075), (700, 130), (4, 5, 96)])
def test_layer_norm(shape, dtype):
    x, dy = rnd(1, *shape, dtype=dtype), rnd(2, *shape, dtype=dtype)
    norm_case(x, rnd(3, shape[-1], shift=1.0, scale=0.3), rnd(4, shape[-1]), dy)


@pytest.mark.parametrize("rows,D,dtype", [(1200, 66001, torch.bfloat16), (1200, 30001, torch.float32), (1100, 50000, torch.float16),
                                          (700, 80000, torch.bfloat16)])
def test_layer_norm_over_more_than_the_caches_hold(rows, D, dtype):
    """Long rows and results larger than the caches, in several rounds of the backward: every row's ends and middle, and all
    columns' sums, against 64 bits taken on the device."""
    from v1_glif_model_amd import sequence as seq
    x, dy = (torch.randn(rows, D, generator=torch.Generator(DEV).manual_seed(k), device=DEV).to(dtype) for k in (1, 2))
    w, b = rnd(3, D, shift=1.0, scale=0.3).requires_grad_(True), rnd(4, D).requires_grad_(True)
    xs = x.requires_grad_(True)
    y = seq.layer_norm(xs, w, b)
    dx, dw, db = grads(y, dy, xs, w, b)
    with torch.no_grad():
        x6, g6, w6 = x.double(), dy.double(), w.double()
        mean = x6.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt(((x6 - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
        xh = (x6 - mean) * rstd
        far = (x6.abs() + x6.abs().mean(-1, keepdim=True)) * rstd
        gw, ga = g6 * w6, g6.abs() * w6.abs()
        dx6 = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
        terms = rstd * (ga + ga.mean(-1, keepdim=True) * (1 + far) + far * (ga * far).mean(-1, keepdim=True))
        for part in (slice(0, 70), slice(D // 2, D // 2 + 70), slice(D - 70, D)):
            near(y[:, part], (xh * w6 + b.double())[:, part].cpu(), (far * w6.abs() + b.abs())[:, part].cpu(), "y")
            near(dx[:, part], dx6[:, part].cpu(), terms[:, part].cpu(), "dx")
        near(dw, (g6 * xh).sum(0).cpu(), (g6.abs() * far).sum(0).cpu(), "dw")
        near(db, g6.sum(0).cpu(), g6.abs().sum(0).cpu(), "db")


@pytest.mark.parametrize("given", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(given):
    for dtype, shape in ((torch.bfloat16, (37, 300)), (F32, (21, 66001))):
        w, b = (rnd(5, shape[-1], dtype=dtype) if on else None for on in given)
        norm_case(rnd(6, *shape, dtype=dtype), w, b, rnd(7, *shape, dtype=dtype))


def test_layer_norm_strides():
    """Rows apart, rows that start anywhere, a transposed view, a broadcast gradient."""
    x = rnd(8, 40, 333, dtype=torch.bfloat16)
    w, b = rnd(9, 200), rnd(10, 200)
    norm_case(x[::2, 5:205], w, b, rnd(11, 20, 200, dtype=torch.bfloat16))
    norm_case(x[3:23, 1:201], w, b, x[1:21, 2:202])
    norm_case(rnd(12, 200, 40).t(), w, b, rnd(13, 1, 200).expand(40, 200))
    norm_case(rnd(14, 6, 5, 400)[:, 1:4, 100:300], w, b, rnd(15, 6, 3, 200))


def test_layer_norm_far_from_zero():
    """The variance is of differences from the mean: a mean of 1000 deviations costs no more than its rounding."""
    norm_case(rnd(16, 11, 3000, shift=1000.0), rnd(17, 3000), rnd(18, 3000), rnd(19, 11, 3000))
    from v1_glif_model_amd import sequence as seq
    y = seq.layer_norm(torch.full((3, 70), 5.0, device=DEV), None, rnd(20, 70))
    assert torch.equal(y, rnd(20, 70).expand(3, 70))


def test_layer_norm_not_finite_and_empty():
    from v1_glif_model_amd import sequence as seq
    x = rnd(21, 9, 260)
    clean = seq.layer_norm(x)
    x[2, 3], x[5, 0] = float("nan"), float("inf")
    y = seq.layer_norm(x)
    other = [r for r in range(9) if r not in (2, 5)]
    assert torch.equal(y[other], clean[other]) and bool(y[2].isnan().all()) and bool(y[5].isnan().all())
    x0 = torch.empty(0, 64, device=DEV, requires_grad=True)
    w0, b0 = (torch.ones(64, device=DEV, requires_grad=True) for _ in range(2))
    y0 = seq.layer_norm(x0, w0, b0)
    dx, dw, db = grads(y0, torch.empty(0, 64, device=DEV), x0, w0, b0)
    assert y0.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


# --------------------------------------------------------------------------- dropout ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,offset", [(1, 0), (3, 1), (64, 3), (1023, 2), (100_003, 5), (7, 2 ** 34 + 1), (4096, 2 ** 62 + 3)])
def test_dropout(n, offset, dtype):
    """The kept elements are those that inputs.bernoulli leaves 0 at p on the same words."""
    from v1_glif_model_amd import sequence as seq
    from v1_glif_model_amd.inputs import bernoulli
    x, res, dy = (rnd(30 + k, n, dtype=dtype) for k in range(3))
    p, seed = 0.3, 2 ** 63 + 12345
    drop = bernoulli(torch.full((n,), p, device=DEV), seed, offset).bool().cpu()
    xs, rs = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    y = seq.dropout(xs, p, seed, offset, residual=rs)
    want = torch.where(drop, torch.zeros((), dtype=ref.F64), f64(x, False) / (1.0 - p))
    near(y, want + f64(res, False), want.abs() + f64(res, False).abs(), "y")
    dx, dres = grads(y, dy, xs, rs)
    near(dx, torch.where(drop, torch.zeros((), dtype=ref.F64), f64(dy, False) / (1.0 - p)), 0.0, "dx",
         more=2.0 ** -22 * f64(dy, False).abs())
    assert torch.equal(dres, dy)
    assert not dx.cpu()[drop].any()


def test_dropout_edges():
    from v1_glif_model_amd import sequence as seq
    x = rnd(35, 3, 50, 41)
    assert torch.equal(seq.dropout(x, 0.0, 7), x)
    assert not seq.dropout(x, 1.0, 7).any() and torch.equal(seq.dropout(x, 1.0, 7, residual=x), x)
    # a stream in pieces, views that start anywhere, other layouts: elements count in row-major order
    whole = seq.dropout(x, 0.5, 9, 4)
    flat = x.reshape(-1)
    parts = [seq.dropout(flat[a:b], 0.5, 9, 4 + a) for a, b in ((0, 1), (1, 1000), (1000, 1003), (1003, flat.numel()))]
    assert torch.equal(torch.cat(parts), whole.reshape(-1))
    t = x.transpose(0, 2)
    assert torch.equal(seq.dropout(t, 0.5, 9), seq.dropout(t.contiguous(), 0.5, 9))
    # what is dropped is 0 whatever it was
    bad = torch.full((5000,), float("nan"), device=DEV)
    kept = seq.dropout(torch.ones(5000, device=DEV), 0.5, 11) != 0
    y = seq.dropout(bad, 0.5, 11)
    assert torch.equal(y.isnan(), kept) and not y[~kept].any()
    share = float((seq.dropout(torch.ones(1_000_000, device=DEV), 0.1, 13) == 0).float().mean())
    assert abs(share - 0.1) < 5 * math.sqrt(0.1 * 0.9 / 1e6)
    assert seq.dropout(torch.empty(0, 4, device=DEV), 0.1, 1).shape == (0, 4)


# ---------------------------------------------------------------------------- linear ----
def linear_case(x, w, b, act, res, dy):
    from v1_glif_model_amd import sequence as seq
    xs, ws, bs, rs = (None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, res))
    y = seq.linear(xs, ws, bs, activation=act, residual=rs)
    assert torch.equal(y.detach(), seq.linear(x, w, b, activation=act, residual=res))
    got = list(grads(y, dy, xs, ws, bs, rs))
    x6, w6, b6, r6 = (f64(t) for t in (x, w, b, res))
    dy6 = f64(dy, False)
    y6 = ref.linear(x6, w6, b6, act, r6)
    want = list(grads(y6, dy6, x6, w6, b6, r6))
    with torch.no_grad():
        pre = ref.linear(x6, w6, b6, None, None)
        terms = x6.abs() @ w6.abs().t() + (0.0 if b is None else b6.abs())
        near(y, y6, 1.2 * terms + (0.0 if res is None else r6.abs()), "y")
        # the slope is at most 1.13 and turns by at most 0.8 per unit of pre; 16-bit types keep pre and dp rounded, and
        # |slope'(pre) pre| <= 0.35
        dp = (dy6 * ref.slope(pre, act)).abs()
        dps, half = dp + 0.8 * dy6.abs() * terms * (act is not None), dp + 0.35 * dy6.abs()
        unit = ref.UNIT[x.dtype] if act else 0.0
        if act == "relu":   # the kink: where pre is within its error of 0 the slope may be either
            near_kink = (pre.abs() <= 1e-5 * terms).double() * dy6.abs()
            half = half + near_kink / max(unit, 1e-30)
        flat = lambda t: t.reshape(-1, t.shape[-1])   # noqa: E731
        near(got.pop(0), want.pop(0), dps @ w6.abs(), "dx", more=unit * (half @ w6.abs()))
        near(got.pop(0), want.pop(0), flat(dps).t() @ flat(x6).abs(), "dw", more=unit * (flat(half).t() @ flat(x6).abs()))
        if b is not None:
            near(got.pop(0), want.pop(0), flat(dps).sum(0), "db", more=unit * flat(half).sum(0))
        if res is not None:
            assert torch.equal(got.pop(0), dy)


LINEAR = [(1, 1, 1), (5, 3, 1), (1, 10, 64), (2, 17, 300), (5, 512, 1000), (16, 16, 32), (17, 64, 33), (33, 129, 257),
          (64, 64, 64), (65, 200, 96), (128, 256, 512), (200, 130, 1001), (257, 255, 128), (360, 257, 203), (300, 520, 2056),
          (7, 40, 12007), (1000, 20, 31), (3, 2000, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear(M, N, K, dtype):
    act = [None, "relu", "gelu", "silu"][(M + N + K) % 4]
    res = rnd(44, M, N, dtype=dtype) if (M + K) % 2 else None
    linear_case(rnd(40, M, K, dtype=dtype), rnd(41, N, K, dtype=dtype, scale=K ** -0.5), rnd(42, N, dtype=dtype), act, res,
                rnd(43, M, N, dtype=dtype))


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_linear_activations(act):
    for dtype, bias in ((F32, F32), (torch.bfloat16, F32), (torch.bfloat16, torch.bfloat16), (torch.float16, None)):
        linear_case(rnd(45, 150, 72, dtype=dtype, scale=3.0), rnd(46, 96, 72, dtype=dtype, scale=0.3),
                    rnd(47, 96, dtype=bias) if bias else None, act, rnd(48, 150, 96, dtype=dtype), rnd(49, 150, 96, dtype=dtype))


def test_linear_strides():
    bf = torch.bfloat16
    x = rnd(50, 90, 401, dtype=bf)
    w = rnd(51, 70, 401, dtype=bf, scale=0.1)
    b = rnd(52, 70, dtype=bf)
    linear_case(x[:, 1:334], w[:, 3:336], b, "gelu", x[:, 300:370], rnd(53, 90, 70, dtype=bf))
    linear_case(x[::3, 8:392], w[:, :384], b, None, None, rnd(54, 1, 70, dtype=bf).expand(30, 70))
    linear_case(rnd(55, 64, 40, dtype=bf).t(), rnd(56, 64, 70, dtype=bf).t(), b, "silu", None, rnd(57, 70, 40, dtype=bf).t())
    linear_case(rnd(58, 4, 5, 6, 50), rnd(59, 9, 50), rnd(60, 9), "relu", rnd(61, 4, 5, 6, 9), rnd(62, 4, 5, 6, 9))


def test_linear_empty_and_not_finite():
    from v1_glif_model_amd import sequence as seq
    w, b = rnd(63, 12, 40), rnd(64, 12)
    for shape, wt in (((0, 40), w), ((3, 0), w[:, :0]), ((3, 40), w[:0])):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        wt = wt.detach().clone().requires_grad_(True)
        bt = b[:wt.shape[0]].clone().requires_grad_(True)
        y = seq.linear(x, wt, bt, activation="silu")
        assert y.shape == (shape[0], wt.shape[0])
        dx, dw, db = grads(y, torch.ones_like(y), x, wt, bt)
        assert dx.shape == x.shape and dw.shape == wt.shape and not dx.isnan().any()
        if shape[0] == 0:
            assert not dw.any() and not db.any()
        if shape[1] == 0:
            near(y, ref.act(f64(b, False), "silu").expand(3, 12), 1.2 * f64(b, False).abs(), "K = 0")
        if wt.shape[0] == 0:
            assert not dx.any()
    x = rnd(65, 70, 40)
    clean = seq.linear(x, w, b)
    x[7, 39], x[60, 0] = float("inf"), float("nan")
    y = seq.linear(x, w, b)
    other = [r for r in range(70) if r not in (7, 60)]
    assert torch.equal(y[other], clean[other]) and not y[7].isfinite().any() and bool(y[60].isnan().all())


@pytest.mark.parametrize("M,N,K,dtype", [(512, 66_000, 640, torch.bfloat16), (66_001, 250, 640, torch.float16), (300, 50_007, 520, F32),
                                         (33_003, 500, 641, torch.bfloat16)])
def test_linear_of_a_few_tiles_more_than_whole_rounds(M, N, K, dtype):
    """Products of whole rounds of tiles and a rest: every row's and column's ends and middle, with all of the epilogue."""
    from v1_glif_model_amd import sequence as seq
    x, w = rnd(67, M, K, dtype=dtype).requires_grad_(True), rnd(68, N, K, dtype=dtype, scale=K ** -0.5).requires_grad_(True)
    b, res, dy = rnd(69, N).requires_grad_(True), rnd(70, M, N, dtype=dtype), rnd(71, M, N, dtype=dtype)
    y = seq.linear(x, w, b, activation="silu", residual=res)
    dx, dw, db = grads(y, dy, x, w, b)
    with torch.no_grad():
        x6, w6, b6, g6, r6 = (t.double() for t in (x, w, b, dy, res))
        pre = x6 @ w6.t() + b6
        q = torch.sigmoid(pre)
        mass = x6.abs() @ w6.abs().t() + b6.abs()
        kept = UNIT[dtype] * pre.abs() if dtype is not F32 else 0.0       # the kept argument's rounding
        dp, ga = g6 * q * (1 + pre * (1 - q)), g6.abs() * (q * (1 + pre.abs() * (1 - q)))
        ga_more = g6.abs() * (0.5 * kept + 2e-5 * mass) + UNIT[dtype] * dp.abs()   # |silu''| <= 1/2; dp is rounded for the products
        spots = lambda n: torch.cat([torch.arange(0, 40), torch.arange(n // 2, n // 2 + 40), torch.arange(n - 700, n)] if n > 800
                                    else [torch.arange(n)]).to(DEV)
        i, j, k = spots(M)[:, None], spots(N)[None], spots(K)
        near(y.detach()[i, j], (pre * q + r6)[i, j].cpu(), (1.1 * mass + r6.abs())[i, j].cpu(), "y")
        i = i[:, 0]
        near(dx[i], (dp[i] @ w6).cpu(), (ga[i] @ w6.abs()).cpu(), "dx", (ga_more[i] @ w6.abs()).cpu())
        j = j[0]
        near(dw[j], (dp[:, j].t() @ x6).cpu(), (ga[:, j].t() @ x6.abs()).cpu(), "dw", (ga_more[:, j].t() @ x6.abs()).cpu())
        near(db, dp.sum(0).cpu(), ga.sum(0).cpu(), "db", (g6.abs() * (0.5 * kept + 2e-5 * mass)).sum(0).cpu())


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("rows", [3, 70])
def test_linear_nan_stays(rows, act):
    """A row that holds NaN answers NaN through every activation, and its gradients are NaN; the other rows' are not."""
    from v1_glif_model_amd import sequence as seq
    x, w, b = rnd(66, rows, 40), rnd(63, 12, 40), rnd(64, 12)
    x[1, 7] = float("nan")
    xs = x.requires_grad_(True)
    y = seq.linear(xs, w, b, activation=act)
    other = [r for r in range(rows) if r != 1]
    assert bool(y[1].isnan().all()) and not y[other].isnan().any()
    (dx,) = grads(y, torch.ones_like(y), xs)
    assert not dx[other].isnan().any()
    if act in ("gelu", "silu"):
        assert bool(dx[1].isnan().all())


# ----------------------------------------------------------------- short convolution ----
def conv_case(x, w, b, act, state, lengths, dy, dlast, poison=False):
    """poison: what the op must not look at is NaN in its inputs, 0 in the reference's."""
    from v1_glif_model_amd import sequence as seq
    T, B, D = x.shape
    W = w.shape[1]
    live = torch.ones(T, B, 1, dtype=torch.bool, device=DEV)
    if lengths is not None:
        live = (torch.arange(T, device=DEV)[:, None] < lengths)[..., None]
    xp, dyp = (torch.where(live, t, torch.full_like(t, float("nan"))) if poison else t for t in (x, dy))
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (xp, w, b, state)]
    y, last = seq.short_conv(leaves[0], leaves[1], leaves[2], activation=act, initial_state=leaves[3], lengths=lengths)
    y0, last0 = seq.short_conv(xp, w, b, activation=act, initial_state=state, lengths=lengths)
    assert torch.equal(y, y0) and torch.equal(last, last0)
    got = list(grads((y, last), (dyp, dlast), *leaves))
    x6, w6, b6, s6 = f64(torch.where(live, x, torch.zeros_like(x))), f64(w), f64(b), f64(state)
    l6, dy6, dl6 = (f64(t, False) for t in (lengths, torch.where(live, dy, torch.zeros_like(dy)), dlast))
    y6, last6 = ref.short_conv(x6, w6, b6, act, s6, l6)
    want = list(grads((y6, last6), (dy6, dl6), *[t for t in (x6, w6, b6, s6)]))
    want = [torch.zeros_like(t) if g is None else g for g, t in zip(want, [t for t in (x6, w6, b6, s6) if t is not None])]
    ab = [None if t is None else t.detach().abs().requires_grad_(True) for t in (x6, w6, b6, s6)]
    ya, la = ref.short_conv(ab[0], ab[1], ab[2], None, ab[3], l6)
    near(y, y6, y6.detach().abs() + 1.2 * ya.detach(), "y")
    assert torch.equal(last.cpu().double(), last6.detach())
    pre = ref.short_conv(x6, w6, b6, None, s6, l6)[0].detach()
    dps = dy6.abs() * (ref.slope(pre, act).abs() + (0.5 * ya.detach() if act else 0.0))
    sums = grads((ya, la), (dps, dl6.abs()), *ab)
    for g, e, s, what in zip(got, want, sums, [n for n, t in zip(("dx", "dw", "db", "dstate"), ab) if t is not None]):
        near(g, e, torch.zeros_like(e) if s is None else s, what)
    if lengths is not None:
        assert not got[0][~live.expand_as(x)].any() and not y.detach()[~live.expand_as(x)].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8])
def test_short_conv(W, dtype):
    for T, B, D in ((1, 1, 1), (2, 3, 5), (W, 2, 64), (33, 2, 70), (70, 3, 257)):
        act = "silu" if (T + W) % 2 else None
        state = rnd(70, B, W - 1, D, dtype=dtype) if T != 33 else None
        conv_case(rnd(71, T, B, D, dtype=dtype), rnd(72, D, W, scale=W ** -0.5), rnd(73, D) if T != 2 else None, act, state,
                  None, rnd(74, T, B, D, dtype=dtype), rnd(75, B, W - 1, D, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_short_conv_lengths(dtype):
    """Trials of their own lengths, 0 and more than T among them, with NaN behind them."""
    for T, W, D in ((40, 4, 48), (67, 3, 9), (5, 6, 130)):
        lens = torch.tensor([0, 1, 2, T // 2, T - 1, T, T + 9, -3], dtype=torch.int32, device=DEV)
        B = lens.numel()
        conv_case(rnd(76, T, B, D, dtype=dtype), rnd(77, D, W, dtype=dtype), rnd(78, D, dtype=dtype), "silu",
                  rnd(79, B, W - 1, D, dtype=dtype), lens, rnd(80, T, B, D, dtype=dtype), rnd(81, B, W - 1, D, dtype=dtype),
                  poison=True)


def test_short_conv_strides_and_no_ticks():
    from v1_glif_model_amd import sequence as seq
    x = rnd(82, 3, 50, 90, dtype=torch.bfloat16)
    w, b = rnd(83, 60, 4), rnd(84, 60)
    dl = rnd(85, 3, 3, 60, dtype=torch.bfloat16)
    conv_case(x.transpose(0, 1)[:, :, 1:61], w, b, "silu", None, None, x.transpose(0, 1)[:, :, 7:67], dl)
    conv_case(x.transpose(0, 1)[::2, :, :60], w, b, None, dl, None, rnd(86, 1, 1, 60, dtype=torch.bfloat16).expand(25, 3, 60), dl)
    st = rnd(87, 2, 3, 60, dtype=torch.bfloat16)
    y, last = seq.short_conv(torch.empty(0, 2, 60, device=DEV, dtype=torch.bfloat16), w, b, initial_state=st)
    assert y.shape == (0, 2, 60) and torch.equal(last, st)
    y, last = seq.short_conv(torch.empty(7, 0, 60, device=DEV, dtype=torch.bfloat16), w, b)
    assert y.shape == (7, 0, 60) and last.shape == (0, 3, 60)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [1, 2, 4, 7])
def test_short_conv_ticks_equal_the_sequence(W, dtype):
    from v1_glif_model_amd import sequence as seq
    for D in (5, 264):
        x, w, b, st = rnd(88, 20, 3, D, dtype=dtype), rnd(89, D, W), rnd(90, D), rnd(91, 3, W - 1, D, dtype=dtype)
        y, last = seq.short_conv(x, w, b, activation="silu", initial_state=st)
        mem, v0 = st.clone(), None
        for t in range(20):
            v0 = mem._version
            yt = seq.short_conv_step(x[t], mem, w, b, activation="silu")
            assert torch.equal(yt, y[t]), t
        assert torch.equal(mem, last) and mem._version > v0
        a, mid = seq.short_conv(x[:9], w, b, activation="silu", initial_state=st)
        c, end = seq.short_conv(x[9:], w, b, activation="silu", initial_state=mid)
        assert torch.equal(torch.cat([a, c]), y) and torch.equal(end, last)


# ------------------------------------------------------------------------ state space ----
def scan_inputs(seed, T, B, D, G, N, dtype):
    k = iter(range(seed, seed + 20))
    A = -torch.exp(rnd(next(k), D, N))
    return dict(u=rnd(next(k), T, B, D, dtype=dtype), delta=rnd(next(k), T, B, D, dtype=dtype, scale=0.5), A=A,
                B=rnd(next(k), T, B, G, N, dtype=dtype), C=rnd(next(k), T, B, G, N, dtype=dtype), D=rnd(next(k), D),
                z=rnd(next(k), T, B, D, dtype=dtype), bias=rnd(next(k), D, shift=-1.5), state=rnd(next(k), B, D, N),
                dy=rnd(next(k), T, B, D, dtype=dtype), dlast=rnd(next(k), B, D, N))


NAMES = ("u", "delta", "A", "B", "C", "D", "z", "bias", "state")


def scan_call(t, softplus, lengths):
    from v1_glif_model_amd import sequence as seq
    return seq.state_space_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], softplus, t["state"], lengths)


def scan_case(t, softplus=True, lengths=None, poison=False):
    T, B, _ = t["u"].shape
    live = torch.ones(T, B, 1, dtype=torch.bool, device=DEV)
    if lengths is not None:
        live = (torch.arange(T, device=DEV)[:, None] < lengths)[..., None]
    masked = ("u", "delta", "z", "dy", "B", "C")

    def fill(name, value):
        v = t[name]
        if v is None or name not in masked or lengths is None:
            return v
        on = live if v.dim() == 3 else live[..., None]
        return torch.where(on, v, torch.full_like(v, value))
    own = {n: fill(n, float("nan") if poison else 0.0) for n in t}
    leaf = {n: None if own[n] is None else own[n].detach().requires_grad_(True) for n in NAMES}
    y, last = scan_call(leaf, softplus, lengths)
    y0, last0 = scan_call({**own}, softplus, lengths)
    near(y0, f64(y, False), f64(y, False).abs(), "with and without gradient")
    near(last0, f64(last, False), f64(last, False).abs(), "with and without gradient")
    got = grads((y, last), (own["dy"], own["dlast"]), *leaf.values())
    r = {n: f64(fill(n, 0.0)) for n in t}
    l6 = f64(lengths, False)
    call = lambda v, sums: ref.scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], softplus,     # noqa: E731
                                    v["state"], l6, sums)
    y6, last6 = call(r, False)
    dy6, dl6 = r["dy"].detach(), r["dlast"].detach()
    want = grads((y6, last6), (dy6, dl6), *[r[n] for n in NAMES])
    ab = {n: None if r[n] is None else (r[n] if n in ("A", "delta", "z", "bias") else r[n].abs()).detach().requires_grad_(True) for n in NAMES}
    ya, la = call(ab, True)
    near(y, y6, ya.detach(), "y")
    near(last, last6, la.detach(), "last")
    sums = grads((ya, la), (dy6.abs(), dl6.abs()), *[ab[n] for n in NAMES])
    given = [n for n in NAMES if t[n] is not None]
    assert len(got) == len(want) == len(sums) == len(given)
    for n, g, e, s in zip(given, got, want, sums):
        zero = torch.zeros_like(ab[n])
        near(g, zero if e is None else e, zero if s is None else s.abs(), "d" + n)
    if lengths is not None:
        assert not y.detach()[~live.expand_as(y)].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 3, 4, 5, 8, 16, 17, 33, 64])
def test_scan(N, dtype):
    for T, B, D, G in ((1, 1, 1, 1), (2, 2, 6, 2), (16, 1, 17, 1), (37, 2, 30, 3)):
        scan_case(scan_inputs(100 + N, T, B, D, G, N, dtype))


@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("T,B,D,G,N", [(15, 1, 70, 1, 16), (17, 3, 65, 1, 16), (130, 1, 8, 4, 16), (300, 2, 5, 1, 11), (65, 1, 260, 2, 4),
                                       (600, 1, 3, 1, 16)])
def test_scan_sizes(T, B, D, G, N, dtype):
    scan_case(scan_inputs(130, T, B, D, G, N, dtype))


@pytest.mark.parametrize("without", [("D",), ("z",), ("bias",), ("state",), ("D", "z", "bias", "state")])
def test_scan_optional_arguments(without):
    t = scan_inputs(140, 21, 2, 10, 1, 16, F32)
    t.update({n: None for n in without})
    scan_case(t)
    scan_case(t, softplus=True, lengths=torch.tensor([21, 4], dtype=torch.int32, device=DEV))


def test_scan_plain_steps():
    t = scan_inputs(150, 40, 2, 9, 3, 16, F32)
    t["delta"], t["bias"] = t["delta"].abs() * 0.3, None
    scan_case(t, softplus=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_lengths(dtype):
    """Trials of their own lengths, 0 and more than T among them, with NaN behind them."""
    for T, D, G, N in ((40, 20, 2, 16), (130, 3, 1, 5)):
        lens = torch.tensor([0, 1, 16, T // 2, T - 1, T, T + 5, -1], dtype=torch.int32, device=DEV)
        scan_case(scan_inputs(160, T, lens.numel(), D, G, N, dtype), lengths=lens, poison=True)


def test_scan_strides():
    T, B, D, N = 30, 3, 24, 16
    t = scan_inputs(170, T, B, D, 2, N, torch.bfloat16)
    wide = rnd(171, B, T, 4 * D + 4 * N, dtype=torch.bfloat16).transpose(0, 1)    # one projection's output, cut up
    t["u"], t["delta"], t["z"] = wide[..., :D], wide[..., D:2 * D], wide[..., 2 * D:3 * D]
    t["B"], t["C"] = (wide[..., at:at + 2 * N].unflatten(-1, (2, N)) for at in (3 * D, 3 * D + 2 * N))
    t["dy"] = rnd(172, T, 1, D, dtype=torch.bfloat16).expand(T, B, D)
    scan_case(t)
    t["A"], t["state"] = t["A"].t().contiguous().t(), t["state"].transpose(0, 1).contiguous().transpose(0, 1)
    t["u"] = t["u"].transpose(0, 2).contiguous().transpose(0, 2)
    t["B"] = t["B"].transpose(2, 3).contiguous().transpose(2, 3)
    scan_case(t)


def test_scan_extreme_steps():
    """Steps from 0 to where every decay is 0, and softplus far out on both sides."""
    t = scan_inputs(180, 25, 1, 12, 1, 16, F32)
    t["delta"] = torch.linspace(-100.0, 60.0, 25 * 12, device=DEV).view(25, 1, 12)
    scan_case(t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_ticks_follow_the_sequence(dtype):
    from v1_glif_model_amd import sequence as seq
    for D, G, N in ((7, 1, 16), (260, 2, 5), (64, 1, 64)):
        t = scan_inputs(190, 12, 3, D, G, N, dtype)
        args = lambda k: (t["delta"][k], t["A"], t["B"][k], t["C"][k], t["D"], t["z"][k], t["bias"])      # noqa: E731
        y, last = scan_call(t, True, None)
        h = t["state"].clone()
        for k in range(12):
            v = h._version
            yk = seq.state_space_step(t["u"][k], h, *args(k))
            assert h._version > v
            r = {n: f64(t[n], False) for n in NAMES}
            near(yk, f64(y[k], False), 4.0 * ref.UNIT[dtype] * 1e5 * f64(y[k], False).abs() + 1.0, "tick")
        near(h, f64(last, False), f64(last, False).abs() + 1.0, "state")
        a, mid = scan_call({n: (v[:5] if n in ("u", "delta", "z", "B", "C") else v) for n, v in t.items()}, True, None)
        b, end = scan_call({**{n: (v[5:] if n in ("u", "delta", "z", "B", "C") else v) for n, v in t.items()}, "state": mid}, True, None)
        near(torch.cat([a, b]), f64(y, False), 4.0 * ref.UNIT[dtype] * 1e5 * f64(y, False).abs() + 1.0, "pieces")
        near(end, f64(last, False), f64(last, False).abs() + 1.0, "pieces' state")
        # the step against the definition
        h1 = t["state"].clone()
        y1 = seq.state_space_step(t["u"][0], h1, *args(0))
        one = {n: (v[:1] if n in ("u", "delta", "z", "B", "C") else v) for n, v in r.items()}
        y6, h6 = ref.scan(one["u"], one["delta"], one["A"], one["B"], one["C"], one["D"], one["z"], one["bias"], True, one["state"])
        ab = {n: v if n in ("A", "delta", "z", "bias") else v.abs() for n, v in one.items()}
        ya, ha = ref.scan(ab["u"], ab["delta"], ab["A"], ab["B"], ab["C"], ab["D"], ab["z"], ab["bias"], True, ab["state"], None, True)
        near(y1, y6[0], ya[0], "y of a tick")
        near(h1, h6, ha, "state of a tick")


def test_scan_no_ticks():
    from v1_glif_model_amd import sequence as seq
    t = scan_inputs(200, 0, 2, 6, 1, 16, F32)
    leaf = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    y, last = scan_call(leaf, True, None)
    assert y.shape == (0, 2, 6) and torch.equal(last, t["state"])
    g = grads((y, last), (t["dy"], t["dlast"]), *[leaf[n] for n in NAMES])
    assert torch.equal(g[NAMES.index("state")], t["dlast"]) and not g[NAMES.index("A")].any()
    y, last = seq.state_space_scan(*(torch.empty(4, 0, 6, device=DEV) for _ in range(2)), t["A"],
                                   *(torch.empty(4, 0, 1, 16, device=DEV) for _ in range(2)))
    assert y.shape == (4, 0, 6) and last.shape == (0, 6, 16)


# ------------------------------------------------------------- differences, repetition ----
def test_gradients_against_differences():
    """<gradient, direction> against the definition's central difference along it, in 64 bits (step 1e-4: the difference's
    own error is 1e-8 of the third derivative); the gradient's elements carry 1e-5 of their terms, the sum over a
    random direction no more than 1e-4 of the sum of |gradient x direction|."""
    from v1_glif_model_amd import sequence as seq
    x, w, b = rnd(210, 6, 20), rnd(211, 20), rnd(212, 20)
    lw, lb = rnd(213, 9, 20, scale=0.3), rnd(214, 9)
    cw, cb, x3 = rnd(215, 20, 4, scale=0.5), rnd(216, 20), rnd(217, 15, 2, 20)
    t = scan_inputs(218, 18, 2, 6, 2, 5, F32)
    cases = [
        (lambda x, w, b: seq.layer_norm(x, w, b), lambda x, w, b: ref.layer_norm(x, w, b, 1e-5), (x, w, b)),
        (lambda x, w, b: seq.linear(x, w, b, activation="gelu"), lambda x, w, b: ref.linear(x, w, b, "gelu", None), (x, lw, lb)),
        (lambda x, w, b: seq.linear(x, w, b, activation="silu"), lambda x, w, b: ref.linear(x, w, b, "silu", None), (x, lw, lb)),
        (lambda x, w, b: seq.short_conv(x, w, b, activation="silu")[0], lambda x, w, b: ref.short_conv(x, w, b, "silu", None, None)[0],
         (x3, cw, cb)),
        (lambda *v: scan_call(dict(zip(NAMES, v)), True, None)[0],
         lambda *v: ref.scan(*v[:8], True, v[8])[0], tuple(t[n] for n in NAMES)),
    ]
    for k, (own, plain, args) in enumerate(cases):
        leaf = [a.clone().requires_grad_(True) for a in args]
        y = own(*leaf)
        dy = rnd(230 + k, *y.shape)
        got = grads(y, dy, *leaf)
        for i, a in enumerate(args):
            v = f64(rnd(240 + i, *a.shape), False)
            base = [f64(q, False) for q in args]
            up, down = (plain(*[q + s * v if j == i else q for j, q in enumerate(base)]) for s in (1e-4, -1e-4))
            diff = float(((up - down) * f64(dy, False)).sum() / 2e-4)
            g = f64(got[i], False)
            assert abs(diff - float((g * v).sum())) <= 1e-4 * float((g * v).abs().sum()) + 1e-6, (k, i)


def test_same_bits_every_time():
    """Every call's sums run in a fixed order."""
    from v1_glif_model_amd import sequence as seq
    bf = torch.bfloat16
    t = scan_inputs(250, 150, 3, 100, 1, 16, bf)
    x, w, b = rnd(251, 700, 1000, dtype=bf), rnd(252, 130, 1000, dtype=bf, scale=0.03), rnd(253, 130, dtype=bf)
    nw, nb = rnd(254, 1000), rnd(255, 1000)
    cw, cb = rnd(256, 100, 4), rnd(257, 100)

    def once():
        out = []
        for f, args in ((lambda *a: seq.layer_norm(*a), (x, nw, nb)),
                        (lambda *a: seq.linear(*a, activation="gelu"), (x, w, b)),
                        (lambda *a: seq.short_conv(*a, activation="silu")[0], (t["u"], cw, cb)),
                        (lambda *a: scan_call(dict(zip(NAMES, a)), True, None)[0], tuple(t[n] for n in NAMES))):
            leaf = [a.clone().requires_grad_(True) for a in args]
            y = f(*leaf)
            out += [y.detach(), *grads(y, torch.ones_like(y), *leaf)]
        return out
    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


# ------------------------------------------------------------ more than 2^31 elements ----
def big(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV, dtype=torch.bfloat16)


def test_layer_norm_and_dropout_past_32_bits():
    from v1_glif_model_amd import sequence as seq
    x = big(1, 33_000, 66_000)
    n = 70 * 66_000
    end = x[-70:].clone()
    y = seq.dropout(x, 0.3, 5, 7)
    assert torch.equal(y[-70:], seq.dropout(end, 0.3, 5, 7 + x.numel() - n)) and torch.equal(y[:1], seq.dropout(x[:1], 0.3, 5, 7))
    xs, dy = x.requires_grad_(True), y
    w = torch.ones(66_000, device=DEV, requires_grad=True)
    out = seq.layer_norm(xs, w)
    dx, dw = grads(out, dy, xs, w)
    x6, g6 = f64(end, False), f64(dy[-70:], False)
    mean = x6.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x6 - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    xh = (x6 - mean) * rstd
    far = (x6.abs() + x6.abs().mean(-1, keepdim=True)) * rstd
    near(out[-70:], xh, far, "y")
    near(dx[-70:], rstd * (g6 - g6.mean(-1, keepdim=True) - xh * (g6 * xh).mean(-1, keepdim=True)),
         rstd * (g6.abs() + g6.abs().mean(-1, keepdim=True) * (1 + far) + far * (g6.abs() * far).mean(-1, keepdim=True)), "dx")
    assert bool(dw.isfinite().all())


def test_sequences_past_32_bits():
    """The last channels of the last entry: a channel's convolution is the same arithmetic wherever it lies; its state space
    is cut into segments of time here and not there, by float32 roundings of the carried state (1e-5 of the largest)."""
    from v1_glif_model_amd import sequence as seq
    T, B, D, N = 16_400, 64, 2048, 4
    x = big(2, T, B, D)
    w = rnd(91, D, 4)
    y, last = seq.short_conv(x, w, activation="silu")
    part = x[:, -1:, -64:].contiguous()
    yp, lp = seq.short_conv(part, w[-64:].contiguous(), activation="silu")
    assert torch.equal(y[:, -1:, -64:], yp) and torch.equal(last[-1:, :, -64:], lp)
    del y
    maps, A = big(3, T, B, 1, N), -torch.exp(rnd(92, D, N))
    y, last = seq.state_space_scan(x, x, A, maps, maps)
    yp, lp = seq.state_space_scan(part, part, A[-64:].contiguous(), maps[:, -1:], maps[:, -1:])
    a, b = y[:, -1:, -64:].double(), yp.double()
    assert float(((a - b).abs() - 2.0 ** -7 * b.abs()).max()) <= 1e-5 * float(b.abs().max())
    assert float((last[-1:, -64:] - lp).abs().max()) <= 1e-5 * float(lp.abs().max())


def test_linear_past_32_bits():
    from v1_glif_model_amd import sequence as seq
    x, w = big(4, 33_000, 32).requires_grad_(True), big(5, 66_000, 32)
    y = seq.linear(x, w)
    x6, w6 = f64(x[-70:], False), f64(w, False)
    near(y[-70:], x6 @ w6.t(), x6.abs() @ w6.abs().t(), "y")
    (dx,) = grads(y, y, x)
    g6 = f64(y[-70:], False)
    near(dx[-70:], g6 @ w6, g6.abs() @ w6.abs(), "dx")



def test_streams_and_capture():
    """Work follows the current stream, and a captured graph replays: every replay on new inputs against the eager result."""
    from v1_glif_model_amd import sequence as seq
    bf = torch.bfloat16
    x, w, b = rnd(260, 5, 512, dtype=bf), rnd(261, 96, 512, dtype=bf, scale=0.05), rnd(262, 96, dtype=bf)
    h, A = rnd(263, 5, 96, 16), -torch.exp(rnd(264, 96, 16))
    Bm, Cm = rnd(265, 5, 1, 16, dtype=bf), rnd(266, 5, 1, 16, dtype=bf)
    mem, cw = rnd(267, 5, 3, 96, dtype=bf), rnd(268, 96, 4)

    def tick(x, mem, h):
        q = seq.linear(seq.layer_norm(x), w, b, activation="silu")
        q = seq.short_conv_step(q, mem, cw, activation="silu")
        return seq.dropout(seq.state_space_step(q, h, q, A, Bm, Cm), 0.25, 3, residual=q)
    side = torch.cuda.Stream()
    big = torch.empty(1 << 26, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m1, h1 = mem.clone(), h.clone()
        big.fill_(1.0)                       # the stream is busy when the calls are made
        x1 = x * 2
        got = tick(x1, m1, h1)
    torch.cuda.current_stream().wait_stream(side)
    m2, h2 = mem.clone(), h.clone()
    assert torch.equal(tick(x * 2, m2, h2), got) and torch.equal(m1, m2) and torch.equal(h1, h2)
    xs, ms, hs = x.clone(), mem.clone(), h.clone()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        tick(xs, ms, hs)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = tick(xs, ms, hs)
    torch.cuda.synchronize()
    me, he = mem.clone(), h.clone()
    ms.copy_(mem), hs.copy_(h)
    for k in range(5):
        new = rnd(270 + k, 5, 512, dtype=bf)
        xs.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, tick(new, me, he)), k
        assert torch.equal(ms, me) and torch.equal(hs, he), k
        big.fill_(float(k))


# -------------------------------------------------------------------------- refusals ----
def test_refusals():
    from v1_glif_model_amd import sequence as seq
    x, x3 = rnd(280, 4, 8), rnd(281, 6, 2, 8)
    w, b = rnd(282, 5, 8), rnd(283, 5)
    t = scan_inputs(284, 6, 2, 8, 2, 4, F32)
    st = rnd(285, 2, 3, 8)
    cw = rnd(286, 8, 4)

    def scan(**new):
        v = {**t, **new}
        return seq.state_space_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, v["state"],
                                    v.get("lengths"))
    bad = [
        (lambda: seq.layer_norm(x.cpu()), "GPU"), (lambda: seq.layer_norm(x.double()), "float32, bfloat16 or float16"),
        (lambda: seq.layer_norm(x, rnd(1, 7)), "shape"), (lambda: seq.layer_norm(x, rnd(1, 8, dtype=torch.bfloat16)), "type"),
        (lambda: seq.layer_norm(x.bfloat16(), rnd(1, 8), rnd(1, 8, dtype=torch.bfloat16)), "one type"),
        (lambda: seq.layer_norm(x[:, :0]), "at least one"), (lambda: seq.layer_norm(x, eps=-1.0), "eps"),
        (lambda: seq.layer_norm(x, eps=float("nan")), "eps"),
        (lambda: seq.dropout(x, 1.5, 0), "p must"), (lambda: seq.dropout(x, float("nan"), 0), "p must"),
        (lambda: seq.dropout(x, 0.1, 0, offset=-1), "offset"), (lambda: seq.dropout(x, 0.1, 0, residual=x[:2]), "shape"),
        (lambda: seq.dropout(x, 0.1, 0, residual=x.half()), "type"),
        (lambda: seq.linear(x, rnd(1, 5, 7)), "shape"), (lambda: seq.linear(x, w.half()), "type"),
        (lambda: seq.linear(x, w, b, activation="tanh"), "activation"), (lambda: seq.linear(x, w, b[:3]), "shape"),
        (lambda: seq.linear(x, w, residual=rnd(1, 1, 5)), "shape"), (lambda: seq.linear(x, w.cpu()), "GPU"),
        (lambda: seq.linear(x, None), "GPU"),
        (lambda: seq.short_conv(x, cw), "T, B, D"), (lambda: seq.short_conv(x3, rnd(1, 8, 9)), "taps"),
        (lambda: seq.short_conv(x3, rnd(1, 8, 0)), "taps"), (lambda: seq.short_conv(x3, rnd(1, 7, 4)), "shape"),
        (lambda: seq.short_conv(x3, cw, activation="relu"), "activation"),
        (lambda: seq.short_conv(x3, cw, initial_state=st[:1]), "shape"), (lambda: seq.short_conv(x3, cw, initial_state=st.half()), "type"),
        (lambda: seq.short_conv(x3, cw, lengths=torch.tensor([1, 2], device=DEV)), "type"),
        (lambda: seq.short_conv(x3, cw, lengths=torch.tensor([1, 2], dtype=torch.int32)), "GPU"),
        (lambda: seq.short_conv(x3, cw, lengths=torch.zeros(3, dtype=torch.int32, device=DEV)), "shape"),
        (lambda: seq.short_conv_step(x3, st, cw), "B, D"), (lambda: seq.short_conv_step(x3[0], st[:1], cw), "shape"),
        (lambda: seq.short_conv_step(x3[0], rnd(1, 2, 8, 3).transpose(1, 2), cw), "contiguous"),
        (lambda: seq.short_conv_step(x3[0].clone().requires_grad_(True), st, cw), "no gradient"),
        (lambda: scan(u=t["u"][0]), "T, B, D"), (lambda: scan(delta=t["delta"][:2]), "shape"), (lambda: scan(A=t["A"].half()), "type"),
        (lambda: scan(A=rnd(1, 8, 65)), "64"), (lambda: scan(B=rnd(1, 6, 2, 3, 4)), "divide"), (lambda: scan(C=rnd(1, 6, 2, 1, 4)), "shape"),
        (lambda: scan(C=t["C"].bfloat16()), "type"), (lambda: scan(D=t["D"].double()), "type"), (lambda: scan(z=t["z"].half()), "type"),
        (lambda: scan(state=t["state"][:, :3]), "shape"), (lambda: scan(bias=rnd(1, 9)), "shape"),
        (lambda: scan(lengths=torch.zeros(2, 1, dtype=torch.int32, device=DEV)), "shape"),
        (lambda: seq.state_space_step(t["u"][0], t["state"].transpose(1, 2).contiguous().transpose(1, 2), t["delta"][0], t["A"],
                                      t["B"][0], t["C"][0]), "contiguous"),
        (lambda: seq.state_space_step(t["u"][0], t["state"], t["delta"][0], t["A"], t["B"][0], t["C"][0],
                                      rnd(1, 8).requires_grad_(True)), "no gradient"),
        (lambda: seq.state_space_step(t["u"], t["state"], t["delta"], t["A"], t["B"], t["C"]), "B, D"),
    ]
    for k, (call, words) in enumerate(bad):
        with pytest.raises(ValueError, match=words):
            call()
            print("not refused:", k)


def test_no_second_gradient():
    """The backwards are not recorded: a graph of them is refused."""
    from v1_glif_model_amd import sequence as seq
    x = rnd(295, 4, 8).requires_grad_(True)
    for y in (seq.layer_norm(x), seq.dropout(x, 0.5, 1), seq.linear(x, rnd(296, 3, 8), activation="gelu"),
              seq.short_conv(x[:, None], rnd(297, 8, 2))[0]):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_c_entries_refuse():
    """The C entries check for themselves: status codes and a message, nothing launched."""
    import ctypes as C
    from v1_glif_model_amd import _lib
    L = _lib.lib()
    x = rnd(290, 4, 8)
    p = _lib.ptr(x)
    codes = [
        L.glif_layer_norm_fwd(p, 8, None, None, 7, 0, 4, 8, 1e-5, p, None), L.glif_layer_norm_fwd(p, 8, None, None, 0, 1, 4, 8, 1e-5, p, None),
        L.glif_layer_norm_fwd(p, 8, None, None, 0, 0, 4, 0, 1e-5, p, None), L.glif_layer_norm_fwd(None, 8, None, None, 0, 0, 4, 8, 1e-5, p, None),
        L.glif_dropout(p, None, 0, -1, 0.5, 0, 0, p, None), L.glif_dropout(p, None, 0, 4, 2.0, 0, 0, p, None),
        L.glif_dropout(None, None, 0, 4, 0.5, 0, 0, p, None),
        L.glif_linear_fwd(p, 8, p, 8, None, None, 0, 0, 0, 4, 4, 8, 9, p, None, None, 0, None),
        L.glif_linear_fwd(p, 8, None, 8, None, None, 0, 0, 0, 4, 4, 8, 0, p, None, None, 0, None),
        L.glif_short_conv_fwd(p, 8, 8, p, None, None, None, 0, 0, 1, 1, 8, 9, 0, p, None, None),
        L.glif_short_conv_step(p, 8, None, p, None, 0, 0, 1, 8, 2, 0, p, None),
        L.glif_scan_fwd(None, p, None, None, None, 0, None), L.glif_scan_step(C.byref(_lib.Scan()), p, p, None),
    ]
    assert all(c == _lib.GLIF_EINVAL for c in codes), codes
    assert L.glif_layer_norm_bwd(p, 8, p, 8, None, 0, 0, 4, 8, 1e-5, p, p, p, None, 0, None) == _lib.GLIF_ENOMEM
    assert L.glif_linear_bwd(p, 4, p, p, 8, p, 8, 0, 0, 4, 4, 8, 1, p, p, p, None, 0, None) == _lib.GLIF_ENOMEM
    assert b"workspace" in L.glif_last_error()
