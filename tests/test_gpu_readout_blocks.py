"""The readout with linear attention, a gated feed-forward block and AdamW, run together: against its definition in 64 bits, by
ticks against whole sequences, trained, saved and resumed."""
import math

import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import F64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype=torch.float32, **kw):
    from v1_glif_model_amd.readout import SequenceReadout
    args = dict(n_neurons=130, n_outputs=5, width=48, channels=64, states=12, taps=3, dropout=0.25, dtype=dtype, seed=3, mixer="attention",
                heads=4, feed_forward=56)
    args.update(kw)
    return SequenceReadout(**args)


def spikes(T, B, N, seed=1):
    return (torch.rand(T, B, N, generator=torch.Generator().manual_seed(seed)) < 0.1).float().to(DEV)


def plain(m, p, x, lengths=None):
    eps = 1e-5
    h = ref.linear(ref.layer_norm(x, p["norm_in"], p["norm_in_bias"], eps), p["embed"], p["embed_bias"], None, None)
    c = ref.linear(ref.layer_norm(h, p["norm_mix"], p["norm_mix_bias"], eps), p["mix_in"], None, None, None)
    u, _ = ref.short_conv(c, p["conv"], p["conv_bias"], "silu", None, lengths)
    n = m.heads * m.states
    q, k, v = (t.unflatten(-1, (m.heads, -1)) for t in u.split((n, n, m.channels), -1))
    y, _ = ref.linear_attention(q, k, v, m.log_decay.cpu().to(F64), m.states ** -0.5, None, lengths)
    y = ref.layer_norm(y, p["norm_heads"], p["norm_heads_bias"], eps).flatten(-2)
    h = h + ref.linear(y, p["mix_out"], p["mix_out_bias"], None, None)
    if m.feed_forward:
        g, o = ref.linear(ref.layer_norm(h, p["norm_ff"], p["norm_ff_bias"], eps), p["ff_in"], p["ff_in_bias"], None, None).split(m.feed_forward, -1)
        h = h + ref.linear(ref.act(g, "silu") * o, p["ff_out"], p["ff_out_bias"], None, None)
    return ref.linear(ref.layer_norm(h, p["norm_out"], p["norm_out_bias"], eps), p["head"], p["head_bias"], None, None)


# Ten operators in float32, each off by at most 1e-5 of its terms' sum; norms between them divide by the spread of what they
# get.  A head's norm sees answers of its first ticks as small as a tenth of later ones, which it divides by: ten times more
# for what went before it.  4 x (10 + 10) x 1e-5 of the largest value.
CHAIN = 8e-4


@pytest.mark.parametrize("feed_forward", [0, 56])
@pytest.mark.parametrize("lengths", [None, [7, 12, 1]])
def test_forward_and_gradients(lengths, feed_forward):
    m = make(feed_forward=feed_forward).eval()
    T, B = 12, 3
    x = spikes(T, B, 130).requires_grad_(True)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    seen = torch.ones(T, B, 1, device=DEV) if ln is None else (torch.arange(T, device=DEV)[:, None] < ln[None])[..., None].float()
    out = m(x, ln)
    dy = torch.randn(T, B, 5, generator=torch.Generator().manual_seed(2)).to(DEV) * seen
    out.backward(dy)
    p = {k: v.detach().cpu().to(F64).requires_grad_(True) for k, v in m.named_parameters()}
    x6 = x.detach().cpu().to(F64).requires_grad_(True)
    want = plain(m, p, x6, None if ln is None else ln.cpu())
    want.backward(dy.cpu().to(F64))
    got, s6 = out.detach().cpu().to(F64), seen.cpu().to(F64)
    assert float(((got - want.detach()) * s6).abs().max()) <= CHAIN * float(want.detach().abs().max())
    for k, v in [*m.named_parameters(), ("x", x)]:
        a, e = v.grad.cpu().to(F64), (p[k] if k != "x" else x6).grad
        assert float((a - e).abs().max()) <= CHAIN * float(e.abs().max()) + 1e-7, k


def test_ticks_go_the_way_of_the_sequence():
    """In float32, whose operators take sums in another order only: as above, against the largest value."""
    m = make().eval()
    T, B = 90, 4
    x = spikes(T, B, 130)
    with torch.no_grad():
        whole = m(x)
    state = m.zero_state(B)
    ticks = torch.stack([m.tick(x[t], state) for t in range(T)])
    assert float((whole - ticks).abs().max()) <= CHAIN * float(whole.abs().max())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_training_step_is_repeatable_and_resumes(bits):
    """Forward, backward and step in bfloat16: the same bits from the same state, and from one that was saved."""
    from v1_glif_model_amd.optim import AdamW

    def new():
        m = make(torch.bfloat16, channels=256, states=64).train()
        return m, AdamW(m.parameters(), 1e-3, state_bits=bits, seed=7)

    def step(m, opt, n):
        out = m(spikes(40, 3, 130, seed=n)).float()
        torch.nn.functional.cross_entropy(out.flatten(0, 1), torch.arange(120, device=DEV) % 5).backward()
        opt.apply_gradients()
        m.zero_grad(set_to_none=True)

    one, two = new(), new()
    for n in range(4):
        step(*one, n)
    for n in range(2):
        step(*two, n)
    three = new()
    three[0].load_state_dict(two[0].state_dict())
    three[1].load_state_dict(two[1].state_dict())
    for n in range(2, 4):
        step(*three, n)
    first = new()[0].state_dict()
    for k, v in one[0].state_dict().items():
        assert torch.equal(v, three[0].state_dict()[k]), k
    assert all(v.isfinite().all() for v in one[0].state_dict().values())
    assert any(not torch.equal(v, first[k]) for k, v in one[0].state_dict().items())


@pytest.mark.parametrize("kw", [dict(mixer="attention", feed_forward=64), dict(feed_forward=64, state_bits=8)])
def test_the_example_runs(kw):
    from v1_glif_model_amd import readout
    losses, share = readout.example(steps=3, ticks=70, batch=4, say=lambda *a: None, **kw)
    assert len(losses) == 3 and all(math.isfinite(x) for x in losses) and 0.0 <= share <= 1.0


def test_refusals_and_the_default():
    from v1_glif_model_amd.readout import SequenceReadout
    for kw in (dict(mixer="none"), dict(heads=3), dict(heads=0), dict(channels=1024, heads=4), dict(states=129), dict(feed_forward=-1),
               dict(mixer="state_space", states=65)):
        with pytest.raises(ValueError):
            make(**kw)
    m = make()
    with pytest.raises(ValueError):
        m.tick(spikes(1, 3, 130)[0], m.zero_state(2))
    plain_one = SequenceReadout(20, 3, width=16, channels=16, device=DEV)
    assert set(plain_one.state_dict()) == {
        "norm_in", "norm_in_bias", "embed", "embed_bias", "norm_mix", "norm_mix_bias", "mix_in", "conv", "conv_bias", "maps", "step",
        "step_bias", "log_rate", "skip", "mix_out", "mix_out_bias", "norm_out", "norm_out_bias", "head", "head_bias", "_extra_state"}
