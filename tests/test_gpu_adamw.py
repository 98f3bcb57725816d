"""GPU parity of AdamW with its definition in 64 bits and, of its 8-bit moments, with the same float32 operations in numpy.

Bounds, in units of 2^-24 (a rounding's half step): a moment is two products of constants that are rounded themselves and a sum
(second moments: a square more): 4 of its terms' sum S.  A variable keeps p (1 - lr decay) to 4 of |p|; the update m / (sqrt(v) root
+ eps) times its size takes 4 (m) + 2 (v under the root) + 2 + 2 (the hardware's root and reciprocal, an ulp each) + 10 (constants,
products and sums) of its absolute terms, under 24; then the variable's own rounding."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [(1,), (3, 5), (255,), (256,), (257,), (0,), (40, 103), (4096,), (9001,)]
LR, B1, B2, EPS, DECAY = 3e-3, 0.9, 0.99, 1e-8, 0.02


def rnd(seed, shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def host(t):
    return t.detach().cpu().double().numpy()


def near(got, want, bound, what):
    over = np.abs(host(got) - want) - bound
    assert not (over > 0).any() and not np.isnan(over).any(), (what, over.max())


def check_variable(p, want, before, update, dtype, what):
    bound = UNIT[dtype] * np.abs(want) + U * (4 * np.abs(before) + 24 * update) * (1 + UNIT[dtype])
    near(p, want, bound + (2.0 ** -25 if dtype is torch.float16 else 0.0), what)


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("wide", [False, True])
def test_steps_in_32_bits(dtype, wide):
    """Three steps of tensors of many sizes; gradients of the variables' type and in float32."""
    from v1_glif_model_amd.optim import AdamW
    ps = [rnd(i, s, dtype) for i, s in enumerate(SIZES)]
    opt = AdamW(ps, LR, B1, B2, EPS, DECAY)
    for t in range(1, 4):
        gs = [rnd(100 * t + i, s, torch.float32 if wide else dtype, 10.0 ** (i % 5 - 3)) for i, s in enumerate(SIZES)]
        before, state = [host(p) for p in ps], [[host(x) for x in xs] for xs in opt.moments()]
        opt.apply_gradients(gs)
        m, v = opt.moments()
        for i, s in enumerate(SIZES):
            wp, wm, wv, sm, up = ref.step(before[i], host(gs[i]), state[0][i], state[1][i], t, LR, B1, B2, EPS, DECAY)
            near(m[i], wm, 4 * U * sm, (t, s, "m"))
            near(v[i], wv, 4 * U * wv, (t, s, "v"))
            check_variable(ps[i], wp, before[i], up, dtype, (t, s))
    assert opt.iterations == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_in_8_bits(dtype):
    """The codes, the scales and what the variables make of them, over steps that start from the last one's codes."""
    from v1_glif_model_amd.optim import AdamW
    seed = 2 ** 40 + 77
    ps = [rnd(i, s, dtype) for i, s in enumerate(SIZES)]
    opt = AdamW(ps, LR, B1, B2, EPS, DECAY, state_bits=8, seed=seed)
    homes = np.cumsum([0] + [-(-p.numel() // 256) * 256 for p in ps])
    F = np.float32
    for t in range(1, 5):
        gs = [rnd(100 * t + i, s, dtype) * (rnd(100 * t + 50 + i, s, dtype) * 3).exp() for i, s in enumerate(SIZES)]
        gs[6][:, 50:] = 0     # blocks of zeros among them
        before, old = [host(p) for p in ps], opt.state_dict()
        opt.apply_gradients(gs)
        new = opt.state_dict()
        values = opt.moments()
        for i, s in enumerate(SIZES):
            if not ps[i].numel():
                continue
            code = [[x.cpu().numpy() for x in old[k][i]] for k in ("first", "second")]
            m, v = (ref.decode(c, z, top) for (c, z), top in zip(code, (127, 255)))
            g = gs[i].float().cpu().numpy()
            wp, _, _, sm, up = ref.step(before[i], g, m, v, t, LR, B1, B2, EPS, DECAY)
            check_variable(ps[i], wp, before[i], up, dtype, (t, s))
            m = m * F(B1) + g * F(1 - B1)
            v = v * F(B2) + (g * g) * F(1 - B2)
            word = ref.words(ps[i].numel(), seed, int((t - 1) * homes[-1] + homes[i]))
            for k, x, top, u in (("first", m, 127, word & 0xFFFF), ("second", v, 255, word >> 16)):
                want, most = ref.encode(x, top, u)
                got, scale = (y.cpu().numpy() for y in new[k][i])
                np.testing.assert_array_equal(scale, most)
                np.testing.assert_array_equal(got.reshape(-1), want)
                assert top == 127 or ((got > 0) == (x > 0)).all()
                near(values[top == 255][i], ref.decode(got, scale, top).astype(np.float64), 0.0, (t, s, k))


def test_moments_in_8_bits_keep_their_mean():
    """Second moments far above their gradients' squares shrink as they do in 32 bits, though one step is less than half a code: the
    mean of 65,536 roundings is within six deviations (each within 1.6 % of the value, so that the mean's are below 1e-4)."""
    from v1_glif_model_amd.optim import AdamW
    n = 65536
    p = torch.zeros(n, device=DEV)
    opt = AdamW([p], 0.0, 0.9, 0.999, state_bits=8, seed=5)
    g = torch.full((n,), 1e-3, device=DEV)
    g[::256] = 1.0                       # holds the scale
    want = torch.zeros(n, dtype=torch.float64)
    opt.apply_gradients([g])
    want = 0.001 * host(g) ** 2
    for _ in range(40):
        opt.apply_gradients([g * 30])
        want = 0.999 * want + 0.001 * (30 * host(g)) ** 2
    v = host(opt.moments()[1][0]).reshape(-1, 256)[:, 1:]
    # steps of a code here are under 2 % of the largest's 1/1000: 4 (1/255) (1e-6)^(3/4) of the scale, 41 roundings of them
    step = 4 / 255 * (1e-6) ** 0.75 * want.max()
    assert abs(v.mean() - want.reshape(-1, 256)[:, 1:].mean()) <= 6 * step * np.sqrt(41 / v.size)


def test_more_tensors_than_a_launch_takes_and_absent_gradients():
    """150 variables; some have no gradient, and stay with their moments."""
    from v1_glif_model_amd.optim import AdamW
    ps = [rnd(i, (1 + 37 * i,)) for i in range(150)]
    alone = [p.clone() for p in ps]
    opt = AdamW(ps, LR, weight_decay=DECAY)
    gs = [None if i % 7 == 3 else rnd(200 + i, p.shape) for i, p in enumerate(ps)]
    opt.apply_gradients(gs)
    opt.apply_gradients(gs)
    for i in range(150):
        if gs[i] is None:
            assert torch.equal(ps[i], alone[i]) and not opt.moments()[0][i].any()
        else:
            one = AdamW([alone[i]], LR, weight_decay=DECAY)
            one.apply_gradients([gs[i]])
            one.apply_gradients([gs[i]])
            assert torch.equal(ps[i], alone[i]), i
    assert opt.iterations == 2
    opt.apply_gradients([None] * 150)
    assert opt.iterations == 2


def test_gradients_of_autograd_views_and_strides():
    """The variables' own grad by default; a gradient that is not contiguous; variables that start anywhere in memory."""
    from v1_glif_model_amd.optim import AdamW
    base = rnd(1, (1001,))
    a, b = base[1:301].view(30, 10), base[501:1000]
    c, d = a.clone(), b.clone()
    g = rnd(2, (10, 30))
    one, two = AdamW([a, b], LR), AdamW([c, d], LR)
    version = c._version
    one.apply_gradients([g.t(), g.reshape(-1)[:1].expand(499)])
    two.apply_gradients([g.t().contiguous(), g.reshape(-1)[:1].repeat(499)])
    assert torch.equal(a, c) and torch.equal(b, d) and c._version > version
    w = rnd(3, (20,)).requires_grad_(True)
    x = w.detach().clone()
    (w * w).sum().backward()
    AdamW([w], LR).apply_gradients()
    AdamW([x], LR).apply_gradients([2 * x])
    assert torch.equal(w.detach(), x)


@pytest.mark.parametrize("bits", [8, 32])
def test_repeats_resumes_and_replays(bits):
    """The same bits again, from a state that was saved, and from a captured step that is replayed with eager work between."""
    from v1_glif_model_amd.optim import AdamW
    shapes, steps = [(300, 7), (1,), (5000,)], 6
    grads = [[rnd(10 * t + i, s) for i, s in enumerate(shapes)] for t in range(steps)]

    def make():
        ps = [rnd(i, s) for i, s in enumerate(shapes)]
        return ps, AdamW(ps, LR, state_bits=bits, seed=9)

    ps, opt = make()
    for t in range(steps):
        opt.apply_gradients(grads[t])
        if t == 2:
            saved, values = opt.state_dict(), [p.clone() for p in ps]
    again, other = make()
    for p, v in zip(again, values):
        p.copy_(v)
    other.load_state_dict(saved)
    for t in range(3, steps):
        other.apply_gradients(grads[t])
    assert all(torch.equal(a, b) for a, b in zip(ps, again)) and other.iterations == steps
    caught, third = make()
    held = [g.clone() for g in grads[0]]
    third.apply_gradients(grads[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        third.apply_gradients(held)
    for t in range(1, steps):
        for h, g in zip(held, grads[t]):
            h.copy_(g)
        graph.replay()
        assert third.iterations == t + 1
    assert all(torch.equal(a, b) for a, b in zip(ps, caught))
    assert all(torch.equal(x, y) for xs, ys in zip(opt.moments(), third.moments()) for x, y in zip(xs, ys))


def test_values_that_are_not_finite():
    """NaN and infinities stay where they are in 32 bits, and within their block of 256 in 8."""
    from v1_glif_model_amd.optim import AdamW
    for bad in (float("nan"), float("inf")):
        g = rnd(1, (1000,))
        clean = [rnd(2, (1000,)) for _ in range(2)]
        for bits, touched in ((32, slice(300, 301)), (8, slice(256, 512))):
            p, q = rnd(2, (1000,)), rnd(2, (1000,))
            with_bad, without = AdamW([p], LR, state_bits=bits), AdamW([q], LR, state_bits=bits)
            h = g.clone()
            h[300] = bad
            with_bad.apply_gradients([h])
            without.apply_gradients([g])
            rest = torch.ones(1000, dtype=torch.bool, device=DEV)
            rest[300] = False
            assert not p[300].isfinite() or bad == float("inf")
            assert torch.equal(p[rest], q[rest])
            with_bad.apply_gradients([g])
            without.apply_gradients([g])
            rest[touched] = False
            assert torch.equal(p[rest], q[rest])
            assert not with_bad.moments()[1][0][touched].isfinite().any()
    tiny = torch.full((300,), 1e-30, device=DEV)
    p = torch.ones(300, device=DEV)
    opt = AdamW([p], LR, weight_decay=0.0, state_bits=8)
    opt.apply_gradients([tiny])
    assert p.isfinite().all() and opt.moments()[0][0].isfinite().all()


def test_another_stream():
    from v1_glif_model_amd.optim import AdamW
    p, q, g = rnd(1, (70000,)), rnd(1, (70000,)), rnd(2, (70000,))
    one, two = AdamW([p], LR, state_bits=8), AdamW([q], LR, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one.apply_gradients([g])
        m = one.moments()
    torch.cuda.current_stream().wait_stream(side)
    two.apply_gradients([g])
    assert torch.equal(p, q) and torch.equal(m[0][0], two.moments()[0][0])


def test_refusals():
    from v1_glif_model_amd.optim import AdamW
    p = rnd(1, (8, 4))
    for args, kw in (([], {}), ([[p], ], dict(state_bits=16)), ([[p], ], dict(beta_1=1.0)), ([[p], ], dict(beta_2=-0.1)),
                     ([[p], ], dict(epsilon=-1.0)), ([[p], ], dict(weight_decay=float("nan"))), ([[p, p], ], {}),
                     ([[p, p[2:3]], ], {}), ([[p.t()], ], {}), ([[p.cpu()], ], {}), ([[p.double()], ], {}), ([["p"], ], {})):
        with pytest.raises(ValueError):
            AdamW(*(args or [[]]), **kw)
    opt = AdamW([p, rnd(2, (3,))])
    g = [rnd(3, (8, 4)), rnd(4, (3,))]
    for bad in (g[:1], [g[0], rnd(5, (4,))], [g[0].half(), g[1]], [g[0].cpu(), g[1]], [g[0], 1.0]):
        with pytest.raises(ValueError):
            opt.apply_gradients(bad)
    assert opt.iterations == 0
    state = opt.state_dict()
    for change in (dict(first=state["first"][:1]), dict(iterations=-1), dict(second=state["second"][::-1]),
                   dict(first=AdamW(opt.variables, state_bits=8).state_dict()["first"])):
        with pytest.raises(ValueError):
            opt.load_state_dict({**state, **change})


@pytest.mark.parametrize("eps", [0.0, 1e-30, 9e-13, float("inf"), float("nan")])
def test_refuses_an_epsilon_below_what_squares_leave(eps):
    from v1_glif_model_amd.optim import AdamW
    with pytest.raises(ValueError, match="epsilon"):
        AdamW([rnd(0, (4,))], epsilon=eps)


@pytest.mark.parametrize("bits", [32, 8])
def test_smallest_epsilon_and_gradients_whose_squares_vanish(bits):
    """Gradients of 1e-30 to 1e-18 and 0, of which the update is m size / epsilon to what is left of sqrt(v): the second moment of
    the largest, 1e-36 (1 - b2) = 1e-38, has a root of 1e-19 and, made up for (1 - b2 = 0.01), 1e-18; that is 1e-6 of epsilon."""
    from v1_glif_model_amd.optim import AdamW
    p = torch.zeros(1024, device=DEV)
    g = torch.cat([torch.zeros(256), torch.logspace(-30, -18, 256), torch.full((256,), 1e-20), -torch.logspace(-25, -19, 256)]).to(DEV)
    AdamW([p], LR, B1, B2, 1e-12, 0.0, state_bits=bits).apply_gradients([g])
    assert not p[:256].any()
    # the first step takes its gradient itself for m / (1 - b1), before a moment is ever a code
    near(p, -LR * host(g) / 1e-12, (1e-6 + 24 * U) * LR * np.abs(host(g)) / 1e-12, bits)


def test_refuses_sparse_gradients_and_variables():
    from v1_glif_model_amd.optim import AdamW
    p = rnd(0, (6, 4))
    before, opt = p.clone(), AdamW([p])
    for g in (p.to_sparse(), p.to_sparse_csr()):
        with pytest.raises(ValueError, match="gradient"):
            opt.apply_gradients([g])
        with pytest.raises(ValueError, match="variables"):
            AdamW([g])
    assert torch.equal(p, before) and opt.iterations == 0
