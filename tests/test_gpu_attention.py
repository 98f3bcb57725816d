"""GPU parity of linear attention with its definition in 64 bits, tick by tick (tests/seq_ref.py).

Bounds: a result is its sum in float32, rounded once (near(): the type's unit of the value and 1e-5 of the sum S of the absolute
terms).  Of bfloat16 sequences every term of y and of the gradients of q, k and v has one factor more that is rounded to bfloat16 (a
score or a state): 2^-8 of S more.  States are float32 whatever the sequences are."""
import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import UNIT, f64, near

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def rates(H):
    """From a head that remembers all to one that sees its own tick."""
    r = -torch.exp(torch.linspace(-9.0, 1.0, max(H, 2)))[:H]
    if H > 2:
        r[0], r[-1] = 0.0, float("-inf")
    return r.to(DEV)


def rounded(dtype):
    return 2.0 ** -8 if dtype is BF16 else 0.0


def case(q, k, v, decay, scale=None, state=None, lengths=None, dy=None, dlast=None, more=None):
    """Forward and all gradients against 64 bits."""
    from v1_glif_model_amd import sequence as seq
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, v, state)]
    given = [t for t in leaves if t is not None]
    y, last = seq.linear_attention(*leaves[:3], decay, scale, leaves[3], lengths)
    with torch.no_grad():
        y0, last0 = seq.linear_attention(q, k, v, decay, scale, state, lengths)
    assert torch.equal(y.detach(), y0) and torch.equal(last.detach(), last0) and last.dtype is F32 and y.dtype is q.dtype
    s = q.shape[-1] ** -0.5 if scale is None else scale
    ends = None if lengths is None else lengths.cpu()
    l6 = [f64(t) for t in (q, k, v, state)]
    y6, last6 = ref.linear_attention(*l6[:3], f64(decay, False), s, l6[3], ends)
    ab = [None if t is None else t.detach().abs().requires_grad_(True) for t in l6]
    ya, lasta = ref.linear_attention(*ab[:3], f64(decay, False), abs(s), ab[3], ends)
    more = rounded(q.dtype) if more is None else more
    near(y, y6, ya.detach(), "y", more * ya.detach())
    near(last, last6, lasta.detach(), "last")
    dy = rnd(91, *y.shape, dtype=q.dtype) if dy is None else dy
    dlast = rnd(92, *last.shape) if dlast is None else dlast
    got = torch.autograd.grad((y, last), given, (dy, dlast))
    again = torch.autograd.grad(seq.linear_attention(*leaves[:3], decay, scale, leaves[3], lengths), given, (dy, dlast))
    want = torch.autograd.grad((y6, last6), [t for t in l6 if t is not None], (f64(dy, False), f64(dlast, False)))
    terms = torch.autograd.grad((ya, lasta), [t for t in ab if t is not None], (f64(dy, False).abs(), f64(dlast, False).abs()))
    for name, a, b, w, t in zip(("dq", "dk", "dv", "dstate"), got, again, want, terms):
        assert torch.equal(a, b), name
        near(a, w, t, name, (more if a.dtype is BF16 else 0.0) * t)


def make(T, B, H, G, K, V, dtype, state=True):
    return (rnd(1, T, B, H, K, dtype=dtype), rnd(2, T, B, G, K, dtype=dtype), rnd(3, T, B, G, V, dtype=dtype), rates(H), None,
            rnd(4, B, H, K, V) if state else None)


SHAPES = [(1, 1, 1, 1, 1, 1), (1, 3, 2, 1, 16, 16), (2, 1, 3, 3, 7, 5), (31, 2, 2, 2, 32, 32), (32, 1, 4, 2, 33, 64), (33, 2, 1, 1, 64, 33),
          (63, 1, 2, 2, 64, 64), (64, 1, 3, 1, 24, 40), (65, 2, 3, 3, 128, 16), (100, 1, 2, 1, 65, 100), (130, 2, 2, 2, 128, 128),
          (97, 1, 6, 2, 100, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    case(*make(*shape, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(700, 2, 2, 1, 20, 36), (1030, 1, 3, 3, 64, 70), (1030, 1, 2, 2, 64, 64), (600, 2, 2, 2, 128, 128)])
def test_time_in_segments(shape, dtype):
    """Few heads and many ticks: segments of the time go at once."""
    T, B = shape[:2]
    case(*make(*shape, dtype))
    case(*make(*shape, dtype, state=False), lengths=torch.tensor([T // 3, T - 1][:B], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,K,V", [(1, 20, 24), (3, 64, 64)])
def test_lengths(G, K, V, dtype):
    """Ticks behind a length may hold anything; lengths of nothing and beyond the end."""
    T, B = 70, 6
    q, k, v, decay, scale, state = make(T, B, 3, G, K, V, dtype)
    lengths = torch.tensor([0, 1, 64, 65, 70, 99], dtype=torch.int32, device=DEV)
    dy = rnd(5, T, B, 3, V, dtype=dtype)
    case(q, k, v, decay, 0.3, state, lengths, dy)
    from v1_glif_model_amd import sequence as seq

    def run(q, k, v, dy):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, state)]
        out = seq.linear_attention(*leaves[:3], decay, 0.3, leaves[3], lengths)
        return (*out, *torch.autograd.grad(out, leaves, (dy, rnd(6, *state.shape))))

    clean = run(q, k, v, dy)
    dead = (torch.arange(T, device=DEV)[:, None] >= lengths)[:, :, None, None]
    spoilt = [torch.where(dead, torch.full_like(t, bad), t) for t, bad in zip((q, k, v, dy), (float("nan"), float("inf"), float("nan"), float("-inf")))]
    for a, b in zip(clean, run(*spoilt)):
        assert torch.equal(a, b)
    assert not clean[0].masked_select(dead).any() and not clean[2].masked_select(dead).any()
    assert torch.equal(clean[1][0], state[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("K,V", [(40, 48), (64, 64), (128, 128)])
def test_what_is_not_finite_does_not_go_back_in_time(K, V, where, dtype):
    from v1_glif_model_amd import sequence as seq
    T = 90
    x = dict(zip("qkv", make(T, 1, 2, 2, K, V, dtype)[:3]))
    decay = torch.tensor([-0.1, -1.0], device=DEV)
    clean, last = seq.linear_attention(*x.values(), decay)
    for tick, bad in ((0, float("nan")), (20, float("inf")), (63, float("nan")), (64, float("-inf")), (89, float("nan"))):
        y = {n: t.clone() for n, t in x.items()}
        y[where][tick, 0, 1, 3] = bad
        out, end = seq.linear_attention(*y.values(), decay)
        # the last digits may differ where a chunk goes tick by tick: scores of float32 sums either way
        near(out[:tick, :, 1], f64(clean[:tick, :, 1], False), 0.0, where, (UNIT[dtype] + 2 * rounded(dtype) + 1e-4) * 40.0)
        assert torch.equal(out[:, :, 0], clean[:, :, 0]) and torch.equal(end[:, 0], last[:, 0])
        assert not out[tick, 0, 1].isfinite().all() and (where == "q" or not end[0, 1].isfinite().all())
        if where == "v":     # only its own channel
            rest = [c for c in range(V) if c != 3]
            assert out[:, :, 1][..., rest].isfinite().all() and end[0, 1][:, rest].isfinite().all()
        if where == "k":
            assert end[0, 1][[c for c in range(K) if c != 3]].isfinite().all()
    # two of them in one chunk: what lies between sees only the first
    y = {n: t.clone() for n, t in x.items()}
    y["v"][10, 0, 1, 3], y["k"][30, 0, 1, 5] = float("nan"), float("nan")
    out, _ = seq.linear_attention(*y.values(), decay)
    assert out[:30, 0, 1][:, [c for c in range(V) if c != 3]].isfinite().all() and out[30:, 0, 1].isnan().all()
    assert out[:10].isfinite().all() and out[10:, 0, 1, 3].isnan().all()


@pytest.mark.parametrize("B,K,V", [(2, 40, 48), (1, 64, 64), (600, 64, 64), (1, 128, 128), (300, 128, 128)])
def test_scores_of_bfloat16_keep_16_bits(B, K, V):
    """32 ticks are one chunk, and without a state before it and a gradient of that behind it there are only scores, which are two
    bfloat16 values: what the first leaves is 2^-8 of it, what the second leaves 2^-8 of that."""
    case(*make(32, B, 3, 3, K, V, BF16, state=False), dlast=torch.zeros(B, 3, K, V, device=DEV), more=2.0 ** -16)


@pytest.mark.parametrize("K,V", [(40, 48), (64, 64), (128, 128)])
def test_an_infinite_state_stays_one(K, V):
    """Positive queries and keys: a column of the state that is infinite gives infinite answers, of its sign, in the scores of the
    same chunk as in those of later ones; the others are as they were."""
    from v1_glif_model_amd import sequence as seq
    q, k, v = (rnd(i, 150, 1, 1, d, dtype=BF16).abs() + 0.1 for i, d in ((1, K), (2, K), (3, V)))
    decay, state = torch.tensor([-0.1], device=DEV), rnd(4, 1, 1, K, V)
    clean, _ = seq.linear_attention(q, k, v, decay, None, state)
    spoilt = state.clone()
    spoilt[0, 0, :, 2], spoilt[0, 0, 5, 7] = float("-inf"), float("inf")
    out, end = seq.linear_attention(q, k, v, decay, None, spoilt)
    rest = [c for c in range(V) if c not in (2, 7)]
    assert (out[..., 2] == float("-inf")).all() and (out[..., 7] == float("inf")).all() and (end[0, 0, :, 2] == float("-inf")).all()
    assert torch.equal(out[..., rest], clean[..., rest])
    k[70, 0, 0, 5] = float("inf")     # an infinite key: its row of the state is not finite (infinite or NaN), and nothing before it
    out, end = seq.linear_attention(q, k, v, decay, None, state)
    assert torch.equal(out[:70], clean[:70]) and not out[70:].isfinite().any() and not end[0, 0, 5].isfinite().any()
    assert end[0, 0][[c for c in range(K) if c != 5]].isfinite().all()


def test_large_states_of_float16():
    """Scores and states beyond 65,504 that outputs within it are made of."""
    q, k, v = rnd(1, 40, 1, 1, 16, dtype=F16, scale=1e-3), rnd(2, 40, 1, 1, 16, dtype=F16, scale=300.0), rnd(3, 40, 1, 1, 16, dtype=F16, scale=300.0)
    case(q, k, v, torch.zeros(1, device=DEV), 1.0, dy=rnd(4, 40, 1, 1, 16, dtype=F16, scale=1e-4), dlast=rnd(5, 1, 1, 16, 16, scale=1e-5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Heads split off one projection, rows that start anywhere, broadcast heads, transposed layouts, a broadcast gradient."""
    T, B, H, K, V = 45, 2, 4, 10, 6
    qkv = rnd(1, T, B, H * (2 * K + V) + 3, dtype=dtype)[..., 1:-2]
    q, k, v = (t.unflatten(-1, (H, -1)) for t in qkv.split((H * K, H * K, H * V), -1))
    case(q, k, v, rates(H), None, rnd(2, H, B, K, V).transpose(0, 1), dy=rnd(3, T, 1, 1, V, dtype=dtype).expand(T, B, H, V))
    q, k, v = rnd(4, B, H, K, T, dtype=dtype).permute(3, 0, 1, 2), rnd(5, B, T, 1, K, dtype=dtype).transpose(0, 1), rnd(6, B, T, 1, V, dtype=dtype).transpose(0, 1)
    case(q, k.expand(T, B, H, K), v.expand(T, B, H, V), rates(2 * H)[::2], 2.0)
    case(q, k, v, rates(H), -0.5)


def test_heads_of_64_off_16_bytes():
    """They go by way of registers, the others straight into LDS."""
    T, B, H = 70, 2, 2
    wide = [rnd(i, T, B, H, 65, dtype=BF16) for i in range(3)]
    case(*(t[..., 1:] for t in wide), rates(H))
    flat = [rnd(i, T * B * H * 64 + 1, dtype=BF16) for i in range(3)]
    off = [t[1:].view(T, B, H, 64) for t in flat]
    case(*off, rates(H))
    case(*(t.clone() for t in off), rates(H))   # (in chunks of other lengths: not the same bits)


def test_gradients_against_differences():
    """y and the last state are linear in each input: differences of any size are exact but for the rounding of both sums."""
    from v1_glif_model_amd import sequence as seq
    q, k, v, decay, _, state = make(75, 2, 4, 2, 12, 9, F32)
    dy, dlast = rnd(7, 75, 2, 4, 9), rnd(8, 2, 4, 12, 9)

    def loss(*x):
        y, last = seq.linear_attention(*x[:3], decay, None, x[3])
        return (y.double() * dy).sum() + (last.double() * dlast).sum(), (y.double() * dy).abs().sum() + (last.double() * dlast).abs().sum()

    x = [t.requires_grad_(True) for t in (q, k, v, state)]
    got = torch.autograd.grad(loss(*x)[0], x)
    for i in range(4):
        d = rnd(10 + i, *x[i].shape)
        with torch.no_grad():
            up, size = loss(*x[:i], x[i] + 0.5 * d, *x[i + 1:])
            down, _ = loss(*x[:i], x[i] - 0.5 * d, *x[i + 1:])
            # float32 sums of 75 ticks and 12 channels: each loss's terms to 1e-5 of their sizes
            assert abs(float(up - down - (got[i].double() * d).sum())) <= 4e-5 * float(size), i


def test_partial_gradients():
    """Any one input alone gets the gradient that it gets beside the others."""
    from v1_glif_model_amd import sequence as seq
    for T in (50, 600):
        x = list(make(T, 1, 2, 1, 16, 16, BF16)[:4])
        x.insert(3, rnd(9, 1, 2, 16, 16))
        dy, dlast = rnd(7, T, 1, 2, 16, dtype=BF16), rnd(8, 1, 2, 16, 16)
        leaves = [t.requires_grad_(True) for t in x[:4]]
        out = seq.linear_attention(*leaves[:3], x[4], None, leaves[3])
        whole = torch.autograd.grad(out, leaves, (dy, dlast))
        for i in range(4):
            one = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
            out = seq.linear_attention(*one[:3], x[4], None, one[3])
            assert torch.equal(torch.autograd.grad(out, [one[i]], (dy, dlast))[0], whole[i]), i
        y, last = seq.linear_attention(*leaves[:3], x[4], None, leaves[3])
        only = torch.autograd.grad(last, [leaves[0], leaves[3]], dlast, allow_unused=True)
        assert not only[0].any() and only[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 24, 40), (2, 3, 3, 33, 70), (5, 8, 1, 128, 128), (2, 2, 2, 64, 3)])
def test_ticks_and_prompts_agree(shape, dtype):
    """Ticks one by one from a prompt's state, against 64 bits."""
    from v1_glif_model_amd import sequence as seq
    B, H, G, K, V = shape
    q, k, v, decay, _, state = make(20, B, H, G, K, V, dtype)
    _, st = seq.linear_attention(q[:12], k[:12], v[:12], decay, None, state)
    ys = []
    for t in range(12, 20):
        version = st._version
        ys.append(seq.linear_attention_step(q[t], k[t], v[t], st, decay))
        assert st._version > version
    l6 = [f64(t, False) for t in (q, k, v)]
    y6, last6 = ref.linear_attention(*l6, f64(decay, False), K ** -0.5, f64(state, False))
    ya, la = ref.linear_attention(*(t.abs() for t in l6), f64(decay, False), K ** -0.5, f64(state, False).abs())
    near(torch.stack(ys), y6[12:], ya[12:], "y")
    near(st, last6, la, "state")


def test_empty():
    from v1_glif_model_amd import sequence as seq
    for T, B in ((0, 2), (3, 0)):
        q, k, v = (torch.empty(T, B, 2, 8, dtype=BF16, device=DEV, requires_grad=True) for _ in range(3))
        state = rnd(1, B, 2, 8, 8).requires_grad_(True)
        y, last = seq.linear_attention(q, k, v, rates(2), None, state)
        assert y.shape == (T, B, 2, 8) and torch.equal(last, state)
        g = torch.autograd.grad((y, last), (q, k, v, state), (torch.empty_like(y), torch.ones_like(last)))
        assert g[0].shape == q.shape and torch.equal(g[3], torch.ones_like(state))
        if T == 0:
            assert not seq.linear_attention(q, k, v, rates(2))[1].any()
    assert seq.linear_attention_step(*(torch.empty(0, 2, 8, device=DEV) for _ in range(3)), torch.empty(0, 2, 8, 8, device=DEV), rates(2)).shape == (0, 2, 8)


def test_capture_and_streams():
    """A captured forward and backward, and captured ticks, replayed with eager work between; another stream."""
    from v1_glif_model_amd import sequence as seq
    x = [t.requires_grad_(True) for t in make(600, 1, 2, 1, 16, 16, BF16)[:3]]
    decay, dy, dlast = rates(2), rnd(7, 600, 1, 2, 16, dtype=BF16), rnd(8, 1, 2, 16, 16)

    def run(x):
        out = seq.linear_attention(*x, decay)
        return (*out, *torch.autograd.grad(out, x, (dy, dlast)))

    def ticks(state):
        return [seq.linear_attention_step(x[0][t], x[1][t], x[2][t], state, decay) for t in range(3)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = run(x)
    torch.cuda.current_stream().wait_stream(side)
    del warm
    state, whole, single = torch.zeros(1, 2, 16, 16, device=DEV), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(whole, stream=side):
        held = run(x)
    with torch.no_grad(), torch.cuda.graph(single, stream=side):
        held_ticks = ticks(state)
    beside = torch.zeros_like(state)
    for n in range(4):
        with torch.no_grad():
            for i, t in enumerate(x):
                t.copy_(rnd(20 + 3 * n + i, *t.shape, dtype=BF16))
        whole.replay()
        single.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run([t.detach().requires_grad_(True) for t in x])):
            assert torch.equal(a, b)
        with torch.no_grad():
            for a, b in zip(held_ticks, ticks(beside)):
                assert torch.equal(a, b)
        assert torch.equal(state, beside)


def test_refusals():
    from v1_glif_model_amd import sequence as seq
    good = dict(zip(("q", "k", "v", "log_decay"), make(4, 2, 4, 2, 8, 6, F32)[:4]))
    bad = [dict(q=good["q"].cpu()), dict(q=good["q"][0]), dict(q=good["q"].double()), dict(k=good["k"].half()), dict(k=good["k"][:, :, :1]),
           dict(k=rnd(1, 4, 2, 3, 8), v=rnd(1, 4, 2, 3, 6)), dict(k=good["k"][..., :7]), dict(v=good["v"][:3]),
           dict(q=rnd(1, 4, 2, 4, 129), k=rnd(1, 4, 2, 2, 129)), dict(v=rnd(1, 4, 2, 2, 129)), dict(v=rnd(1, 4, 2, 2, 0)),
           dict(log_decay=good["log_decay"][:3]), dict(log_decay=good["log_decay"].double()), dict(log_decay=None),
           dict(log_decay=good["log_decay"].clone().requires_grad_(True)), dict(initial_state=rnd(1, 2, 4, 8, 7)),
           dict(initial_state=rnd(1, 2, 4, 8, 6, dtype=BF16)), dict(lengths=torch.ones(2, device=DEV)),
           dict(lengths=torch.ones(3, dtype=torch.int32, device=DEV))]
    for change in bad:
        with pytest.raises(ValueError):
            seq.linear_attention(**{**good, **change})
    tick = {n: t[0] if n != "log_decay" else t for n, t in good.items()}
    state = rnd(2, 2, 4, 8, 6)
    for change in (dict(state=state[:1]), dict(state=state.double()), dict(state=rnd(2, 2, 4, 6, 8).transpose(2, 3)), dict(q=good["q"]),
                   dict(q=tick["q"].clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            seq.linear_attention_step(**{**tick, "state": state, **change})
    x = good["q"].clone().requires_grad_(True)
    y, _ = seq.linear_attention(**{**good, "q": x})
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
