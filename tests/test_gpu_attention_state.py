"""GPU parity of what linear attention makes of its state, for bfloat16 sequences.

A state is multiplied as two bfloat16 values: what the first leaves is 2^-8 of it, what the second leaves 2^-8 of that.  So results
are within 2^-16 of the sum of their absolute terms, and what near() allows for float32 sums and the last rounding."""
import pytest
import torch

from tests.test_gpu_attention import BF16, DEV, DTYPES, F32, SHAPES, case, make, rnd
from tests.seq_ref import UNIT, f64, near

pytestmark = pytest.mark.gpu
TWO_VALUES = 2.0 ** -16


def across(x, left, right):
    """x [..., K, V] without what is along left [..., K] or right [..., V], of which products with either are 0."""
    x, a, b = x.double(), left.double(), right.double()
    a, b = a / a.norm(dim=-1, keepdim=True), b / b.norm(dim=-1, keepdim=True)
    x = x - a[..., None] * (a[..., None, :] @ x)
    return (x - (x @ b[..., None]) * b[..., None, :]).float()


def ticks(t, T):
    return t[None].expand(T, *t.shape).contiguous()


@pytest.mark.parametrize("B,K,V", [(2, 40, 48), (2, 128, 24), (1, 64, 64), (400, 64, 64), (1, 128, 128), (300, 128, 128)])
def test_states_keep_16_bits(B, K, V):
    """Queries across the state before the first tick, and keys and values across the gradient of the last: the products are small
    beside their terms, and there are no others.  Few blocks and many, whole chunks and a short one."""
    from v1_glif_model_amd import sequence as seq
    T, H = 70, 2
    decay, scale = torch.tensor([0.0, -0.02], device=DEV), 0.125
    lam = torch.exp(f64(decay, False))
    n = torch.arange(T, dtype=torch.float64)
    q, dy, k, v = rnd(1, B, H, K, dtype=BF16), rnd(2, B, H, V, dtype=BF16), rnd(3, B, H, K, dtype=BF16), rnd(4, B, H, V, dtype=BF16)
    few = slice(0, 3)

    def bound(left, x, right, times):   # both products of all ticks, and their absolute terms: [T, B, H, ...]
        left, x, right = (f64(t[few], False) for t in (left, x, right))
        a, b = (left[..., None, :] @ x)[..., 0, :], (x @ right[..., None])[..., 0]
        aa, bb = (left.abs()[..., None, :] @ x.abs())[..., 0, :], (x.abs() @ right.abs()[..., None])[..., 0]
        times = times[:, None, :, None]
        return [(times * p, times * s) for p, s in ((a, aa), (b, bb))]

    state = across(rnd(5, B, H, K, V), q, dy)
    zeros = [torch.zeros(T, B, H, d, dtype=BF16, device=DEV) for d in (K, V)]
    leaves = [ticks(q, T).requires_grad_(True), *zeros]
    y, _ = seq.linear_attention(*leaves, decay, scale, state)
    dq, = torch.autograd.grad(y, leaves[0], ticks(dy, T))
    (want, terms), (wantq, termsq) = bound(q, state, dy, scale * lam[None] ** (n[:, None] + 1))
    near(y[:, few], want, terms, "y", TWO_VALUES * terms)
    near(dq[:, few], wantq, termsq, "dq", TWO_VALUES * termsq)

    dlast = across(rnd(6, B, H, K, V), k, v)
    leaves = [zeros[0], ticks(k, T).requires_grad_(True), ticks(v, T).requires_grad_(True)]
    y, last = seq.linear_attention(*leaves, decay, scale)
    dk, dv = torch.autograd.grad((y, last), leaves[1:], (torch.zeros_like(y), dlast))
    (want, terms), (wantk, termsk) = bound(k, dlast, v, lam[None] ** (T - 1 - n[:, None]))
    near(dv[:, few], want, terms, "dv", TWO_VALUES * terms)
    near(dk[:, few], wantk, termsk, "dk", TWO_VALUES * termsk)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] > 32] + [(260, 1, 2, 2, 64, 64), (260, 1, 2, 1, 128, 128), (260, 1, 2, 2, 24, 40)])
def test_shapes_of_several_chunks(shape):
    case(*make(*shape, BF16), more=TWO_VALUES)


@pytest.mark.parametrize("K,V", [(40, 48), (64, 64), (128, 128)])
def test_a_prompt_answers_as_its_ticks_do(K, V):
    """Both are within half a step of the float32 answer: of each other within the steps' sum."""
    from v1_glif_model_amd import sequence as seq
    T, B, H = 140, 2, 3
    q, k, v, decay, _, state = make(T, B, H, H, K, V, BF16)
    y, last = seq.linear_attention(q, k, v, decay, None, state)
    st = state.clone()
    steps = torch.stack([seq.linear_attention_step(q[t], k[t], v[t], st, decay) for t in range(T)])
    terms, size = seq.linear_attention(*(t.abs().to(F32) for t in (q, k, v)), decay, None, state.abs())
    terms, size = f64(terms, False), f64(size, False)
    near(y, f64(steps, False), terms, "y", 2.0 ** -8 * f64(steps, False).abs() + (1e-5 + TWO_VALUES) * terms)
    near(last, f64(st, False), size, "state", 1e-5 * size)


def positive(T, K, V, dtype):
    """Queries and keys above 0: an infinity anywhere makes infinities of its own sign, never their difference."""
    q, k = (rnd(i, T, 1, 2, K, dtype=dtype).abs() + 0.1 for i in (1, 2))
    return q, k, rnd(3, T, 1, 2, V, dtype=dtype), torch.tensor([-0.1, -2.0], device=DEV)


WIDTHS = [(16, 128), (40, 48), (64, 64), (128, 24), (128, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [150, 1100])
@pytest.mark.parametrize("K,V", WIDTHS)
def test_an_infinite_value_makes_its_channel_infinite(K, V, T, dtype):
    """From its tick on, in the state too, however much is forgotten since, whether segments of the time go at once (the 1100 ticks)
    or not; the other channels stay as they were.  Likewise back in time from an infinite gradient of an answer."""
    from v1_glif_model_amd import sequence as seq
    q, k, v, decay = positive(T, K, V, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)] + [torch.zeros(1, 2, K, V, device=DEV, requires_grad=True)]
    dy = rnd(5, T, 1, 2, V, dtype=dtype)
    y, last = seq.linear_attention(*leaves[:3], decay, None, leaves[3])
    dv, dstate = torch.autograd.grad(y, leaves[2:], dy)
    wide = [t.detach().float().abs().requires_grad_(True) for t in leaves]     # the sums of the absolute terms
    sums = seq.linear_attention(*wide[:3], decay, None, wide[3])
    sums += torch.autograd.grad(sums[0], wide[2:], dy.float().abs())
    rest = [c for c in range(V) if c not in (3, 7)]
    for at in (0, 17, 70, 149):
        spoilt, bad = v.clone(), dy.clone()
        spoilt[at, :, :, 3], spoilt[at, :, :, 7] = float("inf"), float("-inf")
        bad[at, :, :, 3], bad[at, :, :, 7] = float("inf"), float("-inf")
        out, end = seq.linear_attention(q, k, spoilt, decay)
        assert (out[at:, ..., 3] == float("inf")).all() and (out[at:, ..., 7] == float("-inf")).all()
        assert (end[..., 3] == float("inf")).all() and (end[..., 7] == float("-inf")).all()
        y1, last1 = seq.linear_attention(*leaves[:3], decay, None, leaves[3])
        gv, gstate = torch.autograd.grad((y1, last1), leaves[2:], (bad, torch.zeros_like(last)))
        assert (gv[:at + 1, ..., 3] == float("inf")).all() and (gv[:at + 1, ..., 7] == float("-inf")).all()
        assert (gstate[..., 3] == float("inf")).all() and (gstate[..., 7] == float("-inf")).all()
        for a, b, size in zip((out, end, gv, gstate), (y, last, dv, dstate), sums):     # each within its bound of the same sums
            b, size = f64(b[..., rest], False), f64(size[..., rest], False)
            near(a[..., rest], b, size, at, UNIT[a.dtype] * b.abs() + (1e-5 + (2 * TWO_VALUES if a.dtype is BF16 else 0.0)) * size)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [150, 1100])
@pytest.mark.parametrize("K,V", WIDTHS)
def test_an_infinite_state_stays_one_however_much_is_forgotten(K, V, T, dtype):
    from v1_glif_model_amd import sequence as seq
    q, k, v, decay = positive(T, K, V, dtype)
    state = rnd(4, 1, 2, K, V)
    y, last = seq.linear_attention(q, k, v, decay, None, state)
    state[..., 2], state[:, :, 5, 7] = float("-inf"), float("inf")
    out, end = seq.linear_attention(q, k, v, decay, None, state)
    assert (out[..., 2] == float("-inf")).all() and (out[..., 7] == float("inf")).all()
    assert (end[..., 2] == float("-inf")).all() and (end[:, :, 5, 7] == float("inf")).all()
    rest = [c for c in range(V) if c not in (2, 7)]
    assert torch.equal(out[..., rest], y[..., rest]) and torch.equal(end[..., rest], last[..., rest])
