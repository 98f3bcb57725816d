"""GPU parity of linear attention on the ways that sizes choose: time in segments, whose states a first launch makes, and the kernel of
many blocks, whose chunks are of 32 ticks.

Sizes follow the rules, not numbers: whether time is in segments shows in the workspace, and blocks are one for each head of an
entry, pass and segment.  Bounds: near()'s, and 2^-16 of the absolute terms' sum for what bfloat16 sequences multiply as two values."""
from ctypes import byref

import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import UNIT, f64, near
from tests.test_gpu_attention import BF16, DEV, DTYPES, F32, case, make, rates, rnd

pytestmark = pytest.mark.gpu


def more(dtype):
    return 2.0 ** -16 if dtype is BF16 else 0.0


def has_segments(T, B, H, G, K, V, dtype):
    """(forward, backward): whether the workspace has states for more than the sums of shared heads' gradients."""
    from v1_glif_model_amd import _lib
    from v1_glif_model_amd.sequence import DTYPES as CODES
    s = _lib.Attention()
    for name in ("q", "k", "v", "log_decay"):
        setattr(s, name, 1 << 20)
    s.dtype, s.n_ticks, s.n_batch, s.n_heads, s.n_groups, s.d_key, s.d_value = CODES[dtype], T, B, H, G, K, V
    L, shared = _lib.lib(), (T * B * H * (K + V) * 4 if G < H else 0)
    return L.glif_attention_fwd_workspace(byref(s)) > 0, L.glif_attention_bwd_workspace(byref(s)) > shared + 4096


def ticks_of_segments(B, H, G, K, V, dtype):
    """The fewest ticks, by chunks of 32, that go in segments both ways, and some more."""
    return next(T for T in range(32, 8192, 32) if all(has_segments(T, B, H, G, K, V, dtype))) + 23


CUT = [(2, 2, 1, 20, 36), (1, 3, 3, 64, 64), (2, 2, 2, 128, 128), (1, 4, 2, 128, 128), (1, 6, 2, 40, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dims", CUT)
def test_segments(dims, dtype):
    T, B = ticks_of_segments(*dims, dtype), dims[0]
    case(*make(T, *dims, dtype), more=more(dtype))
    case(*make(T, *dims, dtype, state=False), lengths=torch.tensor([T // 3, T - 1][:B], dtype=torch.int32, device=DEV), more=more(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dims", [(1, 2, 1, 16, 16), (1, 2, 2, 64, 64), (1, 2, 2, 128, 128)])
def test_partial_gradients_of_segments(dims, dtype):
    """Any one input alone gets the gradient that it gets beside the others, the first state among them."""
    from v1_glif_model_amd import sequence as seq
    T = ticks_of_segments(*dims, dtype)
    q, k, v, decay, _, state = make(T, *dims, dtype)
    x, dy, dlast = (q, k, v, state), rnd(7, T, dims[0], dims[1], dims[4], dtype=dtype), rnd(8, *state.shape)

    def grads(want, of):
        leaves = [t.detach().requires_grad_(j in want) for j, t in enumerate(x)]
        out = seq.linear_attention(*leaves[:3], decay, None, leaves[3])
        pairs = [(o, d) for o, d, on in zip(out, (dy, dlast), of) if on]
        return torch.autograd.grad([o for o, _ in pairs], [leaves[i] for i in want], [d for _, d in pairs], allow_unused=True)

    for of in ((1, 1), (1, 0)):
        whole = grads(range(4), of)
        for i in range(4):
            assert torch.equal(grads([i], of)[0], whole[i]), (of, i)
    only = grads(range(4), (0, 1))
    assert not only[0].any() and only[1].any() and only[2].any() and only[3].any()


@pytest.mark.parametrize("dims", [(1, 2, 1, 16, 16), (1, 2, 2, 128, 128)])
def test_segments_in_a_captured_graph(dims):
    """Replays with eager work between, each against the eager call."""
    from v1_glif_model_amd import sequence as seq
    T, (B, H, G, K, V) = ticks_of_segments(*dims, BF16), dims
    x = [t.requires_grad_(True) for t in make(T, *dims, BF16)[:3]]
    decay, dy, dlast = rates(H), rnd(7, T, B, H, V, dtype=BF16), rnd(8, B, H, K, V)

    def run(x):
        out = seq.linear_attention(*x, decay)
        return (*out, *torch.autograd.grad(out, x, (dy, dlast)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = run(x)
    torch.cuda.current_stream().wait_stream(side)
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = run(x)
    for n in range(4):
        with torch.no_grad():
            for i, t in enumerate(x):
                t.copy_(rnd(20 + 3 * n + i, *t.shape, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run([t.detach().requires_grad_(True) for t in x])):
            assert torch.equal(a, b)


def some_entries(q, k, v, decay, state, lengths, pick, grads=True):
    """Entries do not meet: those of ``pick`` against 64 bits."""
    from v1_glif_model_amd import sequence as seq
    leaves = [t.detach().requires_grad_(grads) for t in (q, k, v, state)]
    out = seq.linear_attention(*leaves[:3], decay, None, leaves[3], lengths)
    dy, dlast = rnd(91, *out[0].shape, dtype=q.dtype), rnd(92, *out[1].shape)
    got = (*out, *torch.autograd.grad(out, leaves, (dy, dlast))) if grads else out

    scale, few = q.shape[-1] ** -0.5, [t.detach()[:, pick] for t in (q, k, v)] + [state[pick]]
    ends = None if lengths is None else lengths[pick].cpu()
    l6 = [f64(t, grads) for t in few]
    ab = [f64(t.abs(), grads) for t in few]
    want = ref.linear_attention(*l6[:3], f64(decay, False), scale, l6[3], ends)
    size = ref.linear_attention(*ab[:3], f64(decay, False), scale, ab[3], ends)
    if grads:
        d6 = [f64(t, False) for t in (dy[:, pick], dlast[pick])]
        want = (*want, *torch.autograd.grad(want, l6, d6))
        size = (*size, *torch.autograd.grad(size, ab, [t.abs() for t in d6]))
    for name, a, w, s in zip(("y", "last", "dq", "dk", "dv", "dstate"), got, want, size):
        a = a.detach()[pick] if name in ("last", "dstate") else a.detach()[:, pick]
        near(a, w.detach(), s.detach(), name, (more(q.dtype) if a.dtype is BF16 else 0.0) * s.detach())


# more than 512 blocks of 64 channels, more than 256 of 128, forwards and back
MANY = [(174, 3, 64, 64), (90, 3, 128, 128)]


@pytest.mark.parametrize("T", [33, 70, 100])
@pytest.mark.parametrize("B,H,K,V", MANY)
def test_chunks_of_32_ticks(B, H, K, V, T):
    """A second chunk of one tick, short ones behind two and three; lengths of nothing, of whole chunks and one more or less."""
    q, k, v, decay, _, state = make(T, B, H, H, K, V, BF16)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    lengths[:8] = torch.tensor([0, 1, 31, 32, 33, 64, 65, T])
    some_entries(q, k, v, decay, state, lengths.to(DEV), [*range(8), B - 1])
    some_entries(q, k, v, decay, state, None, [0, B // 2, B - 1])


def test_many_segments_of_64_channels():
    """A states launch of more than 512 blocks."""
    T, B, H = 832, 64, 4
    assert has_segments(T, B, H, H, 64, 64, BF16)[0]
    q, k, v, decay, _, state = make(T, B, H, H, 64, 64, BF16)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    lengths[:4] = torch.tensor([0, 257, 256, T])
    with torch.no_grad():
        some_entries(q, k, v, decay, state, lengths.to(DEV), [0, 1, 2, 3, B - 1], grads=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("B,H,K,V", MANY)
def test_what_is_not_finite_in_chunks_of_32_ticks(B, H, K, V, bad):
    """A value's channel of its head from its tick on, and a gradient's up to it; all else as it was (the same chunk's other channels
    of a wave by another order of the same sums)."""
    from v1_glif_model_amd import sequence as seq
    T = 100
    q, k, v, decay, _, state = make(T, B, H, H, K, V, BF16)
    decay = torch.full_like(decay, -0.05)

    def run(v, dy):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, state)]
        out = seq.linear_attention(*leaves[:3], decay, None, leaves[3])
        return (*(o.detach() for o in out), *torch.autograd.grad(out, leaves[2:], (dy, torch.zeros_like(state))))

    dy = rnd(5, T, B, H, V, dtype=BF16)
    y, last, dv, dstate = run(v, dy)
    tick, entry, head, c = 40, B - 2, 1, 21
    v1, dy1 = v.clone(), dy.clone()
    v1[tick, entry, head, c], dy1[tick, entry, head, c] = bad, bad
    y1, last1, _, _ = run(v1, dy)
    _, _, dv1, dstate1 = run(v, dy1)
    assert not y1[tick:, entry, head, c].isfinite().any() and not last1[entry, head, :, c].isfinite().any()
    assert not dv1[:tick + 1, entry, head, c].isfinite().any() and not dstate1[entry, head, :, c].isfinite().any()
    wide = [t.float().abs() for t in (q, k, v)]
    size, _ = seq.linear_attention(*(t[:, entry:entry + 1] for t in wide), decay, None, state[entry:entry + 1].abs())
    back = [t[:, entry:entry + 1].contiguous() for t in wide]
    back[2].requires_grad_(True)
    back = torch.autograd.grad(seq.linear_attention(*back, decay)[0], back[2], dy[:, entry:entry + 1].float().abs())[0]
    for a, b, s, dead in ((y1, y, size, slice(tick, None)), (dv1, dv, back, slice(0, tick + 1))):
        a, b = a.clone(), b.clone()
        a[dead, entry, head, c], b[dead, entry, head, c] = 0.0, 0.0
        same = torch.ones(B, dtype=torch.bool, device=DEV)
        same[entry] = False
        assert torch.equal(a[:, same], b[:, same])
        w, s = f64(b[:, entry], False), f64(s[:, 0], False)
        near(a[:, entry], w, s, "the entry's others", UNIT[BF16] * w.abs() + (1e-5 + 2 * more(BF16)) * s)


@pytest.mark.parametrize("K,V", [(128, 128), (120, 128)])
def test_sequences_of_more_than_2_to_the_31_elements(K, V):
    """The last entry of a batch against itself alone, whose sums are by other chunks: each within its bound."""
    from v1_glif_model_amd import sequence as seq
    T, B, H = 9200, 64, 32
    assert T * B * H * min(K, V) > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, dy = (torch.randn(T, B, H, d, generator=g, device=DEV, dtype=BF16) for d in (K, K, V, V))
    decay, lengths = -torch.logspace(-3, 0, H, device=DEV), torch.full((B,), T, dtype=torch.int32, device=DEV)
    lengths[-1] = T - 5

    def run(q, k, v, dy, lengths):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = seq.linear_attention(*leaves, decay, None, None, lengths)
        return (*(o.detach() for o in out), *torch.autograd.grad(out[0], leaves, dy))

    got = run(q, k, v, dy, lengths)
    got = [got[0][:, -1:].clone(), got[1][-1:].clone(), *(t[:, -1:].clone() for t in got[2:])]
    one = [t[:, -1:].contiguous() for t in (q, k, v, dy)]
    del q, k, v, dy
    want, size = run(*one, lengths[-1:]), run(*(t.float().abs() for t in one), lengths[-1:])
    for name, a, w, s in zip(("y", "last", "dq", "dk", "dv"), got, want, size):
        assert not name == "y" or (a[-6].any() and not a[-5:].any())
        w, s = f64(w, False), f64(s, False)
        near(a, w, s, name, UNIT[a.dtype] * w.abs() + (1e-5 + (2 * more(BF16) if a.dtype is BF16 else 0.0)) * s)
    torch.cuda.empty_cache()
