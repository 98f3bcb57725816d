"""The sequence readout: its answers and gradients against its definition in 64 bits, ticks against whole sequences, the
masks of its dropout, and training with the column."""
import pytest
import torch

from tests import seq_ref as ref
from tests.seq_ref import F64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype=torch.float32, **kw):
    from v1_glif_model_amd.readout import SequenceReadout
    args = dict(n_neurons=130, n_outputs=5, width=48, channels=64, states=8, groups=2, taps=3, rank=6, dropout=0.25, dtype=dtype,
                seed=3)
    args.update(kw)
    return SequenceReadout(**args)


def spikes(T, B, N, seed=1):
    return (torch.rand(T, B, N, generator=torch.Generator().manual_seed(seed)) < 0.1).float().to(DEV)


def plain(m, p, x, lengths=None, keep=None):
    """The readout's definition; p: its parameters in 64 bits; keep: the dropout's mask over 1 - p."""
    eps = 1e-5
    h = ref.linear(ref.layer_norm(x, p["norm_in"], p["norm_in_bias"], eps), p["embed"], p["embed_bias"], None, None)
    c, gate = ref.linear(ref.layer_norm(h, p["norm_mix"], p["norm_mix_bias"], eps), p["mix_in"], None, None, None).split(m.channels, -1)
    u, _ = ref.short_conv(c, p["conv"], p["conv_bias"], "silu", None, lengths)
    n = m.groups * m.states
    low, B, C = (u @ p["maps"].t()).split((m.rank, n, n), -1)
    y, _ = ref.scan(u, low @ p["step"].t(), -torch.exp(p["log_rate"]), B.unflatten(-1, (m.groups, m.states)),
                    C.unflatten(-1, (m.groups, m.states)), p["skip"], gate, p["step_bias"], lengths=lengths)
    y = ref.linear(y, p["mix_out"], p["mix_out_bias"], None, None)
    h = h + (y if keep is None else y * keep)
    return ref.linear(ref.layer_norm(h, p["norm_out"], p["norm_out_bias"], eps), p["head"], p["head_bias"], None, None)


def params(m):
    return {k: v.detach().cpu().to(F64).requires_grad_(True) for k, v in m.named_parameters()}


# A chain of seven operators in float32, each off by at most 1e-5 of its terms' sum; the norms between them divide by the
# spread of what they get (about 1 here, of values of about 1), so errors add: 7 x 1e-5 against the largest value, and four
# times that where the terms cancel.
CHAIN = 3e-4


@pytest.mark.parametrize("lengths", [None, [7, 0, 12]])
def test_forward_and_gradients(lengths):
    m = make().eval()
    T, B = 12, 3
    x = spikes(T, B, 130).requires_grad_(True)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    seen = torch.ones(T, B, 1, device=DEV) if ln is None else (torch.arange(T, device=DEV)[:, None] < ln[None])[..., None].float()
    out = m(x, ln)
    dy = torch.randn(T, B, 5, generator=torch.Generator().manual_seed(2)).to(DEV) * seen
    out.backward(dy)
    p, x6 = params(m), x.detach().cpu().to(F64).requires_grad_(True)
    want = plain(m, p, x6, None if ln is None else ln.cpu())
    want.backward(dy.cpu().to(F64))
    s6 = seen.cpu().to(F64)
    got = out.detach().cpu().to(F64)
    assert float(((got - want.detach()) * s6).abs().max()) <= CHAIN * float(want.detach().abs().max())
    for k, v in [*m.named_parameters(), ("x", x)]:
        a, e = v.grad.cpu().to(F64), (p[k] if k != "x" else x6).grad
        assert float((a - e).abs().max()) <= CHAIN * float(e.abs().max()) + 1e-7, k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ticks_go_the_way_of_the_sequence(dtype):
    """A tick's operators round where the sequence's do; a sum taken in another order may move a rounding by a unit, at each
    of seven operators, and the state carries them on: seven units of the largest value, four times that for the carry."""
    m = make(dtype).eval()
    T, B = 40, 4
    x = spikes(T, B, 130)
    with torch.no_grad():
        whole = m(x).float()
    state = m.zero_state(B)
    ticks = torch.stack([m.tick(x[t], state) for t in range(T)]).float()
    unit = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert float((whole - ticks).abs().max()) <= 28 * unit * float(whole.abs().max())


def test_dropout_is_the_streams_and_moves_on():
    from v1_glif_model_amd import sequence as seq
    m = make().train()
    T, B = 9, 2
    x = spikes(T, B, 130)
    n = T * B * m.width
    outs = [m(x).detach() for _ in range(2)]
    assert m.drawn == 2 * n
    for k, out in enumerate(outs):
        keep = seq.dropout(torch.ones(T, B, m.width, device=DEV), m.dropout, m.seed, k * n)
        with torch.no_grad():
            want = plain(m, params(m), x.cpu().to(F64), keep=keep.cpu().to(F64))
        assert float((out.cpu().to(F64) - want).abs().max()) <= CHAIN * float(want.abs().max())
    assert not torch.equal(*outs)


def test_trains_with_the_column():
    """The example: the loss falls under what knowing nothing gives (log 4) by half, and the trained pair, read out by ticks,
    is right more often than chance (1/4) by as much again."""
    from v1_glif_model_amd import readout
    losses, share = readout.example(say=lambda *a: None)
    assert losses[0] > 0.9 and sum(losses[-10:]) / 10 < 0.69
    assert share >= 0.5


def test_gradient_reaches_the_synapses():
    """dL/dz of the readout goes through RSNNRollout as it does when it is handed to the cell's backward."""
    from tests.helpers import tiny_config
    from v1_glif_model_amd import synthetic as sy
    from v1_glif_model_amd.models import RSNNRollout, V1Column
    cfg = tiny_config(rs=2.0, ins=3.0)
    cell = V1Column(sy.make_network(cfg, seed=5, dense_basis=True), mode="deterministic", train_input=True,
                    train_recurrent_per_type=False, gauss_std=0.5, dampening_factor=0.5, pseudo_gauss=True)
    lgn, bkg = (torch.tensor(a, device=DEV) for a in sy.make_inputs(cfg, seed=6, seq_len=30, batch=3))
    w = (cell.recurrent_weight_values, cell.input_weight_values, cell.bkg_input_weights)
    m = make(n_neurons=cfg.n_neurons).eval()
    z, _ = RSNNRollout.apply(cell, lgn, bkg, *w)
    assert float(z.detach().sum()) > 0
    (gz,) = torch.autograd.grad(m(z).square().sum(), z, retain_graph=True)
    m(z).square().sum().backward()
    want = cell.backward(gz=gz, rollout=z.grad_fn.rollout)
    for k, t in zip(("rec", "lgn", "bkg"), w):
        if t.requires_grad:
            assert float(want[k].abs().max()) > 0
            # two runs over the same numbers; the cell's sums over synapses may be taken in another order
            assert float((t.grad - want[k]).abs().max()) <= 1e-5 * float(want[k].abs().max()), k


def test_refusals():
    from v1_glif_model_amd.readout import SequenceReadout
    for kw in (dict(channels=63), dict(states=65), dict(taps=9), dict(width=0), dict(dropout=1.5), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            make(**kw)
    m = make()
    with pytest.raises(ValueError):
        m(spikes(4, 2, 131))
    with pytest.raises(ValueError):
        m.tick(spikes(4, 2, 130), m.zero_state(2))
    with pytest.raises(ValueError):
        m.tick(spikes(1, 3, 130)[0], m.zero_state(2))
    assert SequenceReadout.__doc__
