"""A trained readout of the column's activity, over whole rollouts and tick by tick.

The reference reads its rollouts out with a Dense layer or a pool of neurons (models.py:1138-1209, 1213-1392), whose memory
is the column's own.  ``SequenceReadout`` is a selective state space over the spikes, from the operators of ``sequence``:
it is trained over a rollout's ``z`` [T, B, N] (with the column, where ``z`` comes from ``RSNNRollout``: the gradient goes
on into the synaptic weights), and answers one tick at a time beside ``V1Column.call``, at a cost that does not grow with
the ticks behind it.  Its mixing can be linear attention with a decay for each head instead, and a gated feed-forward block can
follow it.

``python -m v1_glif_model_amd.readout`` trains one with a small column to tell which of four groups of LGN units is active,
and reads the trained pair out tick by tick (``--mixer attention``, ``--feed-forward 128``, ``--state-bits 8``).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import nn

from . import _lib
from .sequence import (dropout, gated_linear, layer_norm, linear, linear_attention, linear_attention_step, short_conv,
                       short_conv_step, state_space_scan, state_space_step)

__all__ = ["SequenceReadout", "ReadoutState"]


class ReadoutState(NamedTuple):
    """What tick-by-tick reading carries: the last inputs of the convolution, the state space's or the attention's state, and all
    of the readout's parameters as they were when the state was made (matrices in the activations' type): training goes on beside
    it unseen."""
    conv: torch.Tensor      # [B, taps - 1, channels]; of attention, keys and queries among the channels
    scan: torch.Tensor      # [B, channels, states], float32; of attention [B, heads, states, channels / heads]
    weights: dict


class SequenceReadout(nn.Module):
    """``head(norm(h + dropout(mix(norm(h)))))``, ``h = embed(norm(x))``: x [T, B, n_neurons] to [T, B, n_outputs].

    ``mix`` is a projection to ``channels`` and as many gates, a short convolution of ``taps`` ticks, the state space with
    step, input and output maps projected from the convolved channels (the step through ``rank``), and a projection back.

    ``mixer="attention"``: ``mix`` is a projection to queries, keys (``states`` channels a head) and values (``channels`` in all)
    of ``heads`` heads, the short convolution of all of them, linear attention whose heads remember from 4 ticks to 1000, a norm
    of each head, and the projection back.  ``feed_forward``: where it is not 0, ``h + back(silu(gate(n)) * up(n))``, ``n =
    norm(h)``, of that many channels follows the mixing.

    Parameters are float32; products run in ``dtype`` (float32, bfloat16 or float16).  ``seed`` sets the first weights and
    names the stream of the dropout's masks; ``drawn``, how much of it training has used, is part of the ``state_dict``."""

    def __init__(self, n_neurons: int, n_outputs: int, width: int = 256, channels: int = 512, states: int = 16, groups: int = 1,
                 taps: int = 4, rank: int = 16, dropout: float = 0.1, dtype=torch.bfloat16, seed: int = 0, device="cuda",
                 mixer: str = "state_space", heads: int = 4, feed_forward: int = 0):
        super().__init__()
        _lib.require_gpu()
        for name, v in dict(n_neurons=n_neurons, n_outputs=n_outputs, width=width, channels=channels, states=states,
                            groups=groups, taps=taps, rank=rank, heads=heads).items():
            if int(v) < 1:
                raise ValueError(f"{name} must be >= 1, got {v}")
        if channels % groups:
            raise ValueError(f"groups ({groups}) must divide channels ({channels})")
        if mixer not in ("state_space", "attention"):
            raise ValueError(f"mixer must be 'state_space' or 'attention', got {mixer!r}")
        attends = mixer == "attention"
        if attends and (channels % heads or channels // heads > 128):
            raise ValueError(f"heads ({heads}) must divide channels ({channels}) into at most 128")
        if int(feed_forward) < 0:
            raise ValueError(f"feed_forward must be >= 0, got {feed_forward}")
        if states > (128 if attends else 64) or taps > 8:
            raise ValueError(f"at most 64 states (128 of attention) and 8 taps, got {states} and {taps}")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout must be in [0, 1], got {dropout}")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        self.n_neurons, self.n_outputs, self.width, self.channels = n_neurons, n_outputs, width, channels
        self.states, self.groups, self.taps, self.rank = states, groups, taps, rank
        self.dropout, self.dtype, self.seed = float(dropout), dtype, int(seed)
        self.mixer, self.heads, self.feed_forward = mixer, heads, int(feed_forward)
        self.drawn = 0                               # words of the masks' stream that training has used so far
        g = torch.Generator().manual_seed(self.seed)

        def matrix(n, k):
            return nn.Parameter((torch.randn(n, k, generator=g) / math.sqrt(k)).to(device))

        def filled(v, *shape):
            return nn.Parameter(torch.full(shape, float(v), device=device))

        self.norm_in, self.norm_in_bias = filled(1, n_neurons), filled(0, n_neurons)
        self.embed, self.embed_bias = matrix(width, n_neurons), filled(0, width)
        self.norm_mix, self.norm_mix_bias = filled(1, width), filled(0, width)
        if attends:
            keys = heads * states
            self.mix_in = matrix(2 * keys + channels, width)
            self.conv, self.conv_bias = matrix(2 * keys + channels, taps), filled(0, 2 * keys + channels)
            self.norm_heads, self.norm_heads_bias = filled(1, channels // heads), filled(0, channels // heads)
            ticks = torch.exp(torch.linspace(math.log(4.0), math.log(1000.0), heads))
            self.register_buffer("log_decay", (-1.0 / ticks).to(device))
        else:
            self.mix_in = matrix(2 * channels, width)
            self.conv, self.conv_bias = matrix(channels, taps), filled(0, channels)
            self.maps = matrix(rank + 2 * groups * states, channels)
            self.step = matrix(channels, rank)
            # steps of 1 to 100 ms at a zero argument, and decay rates of 1 to `states`
            step = torch.exp(torch.rand(channels, generator=g) * math.log(100.0) + math.log(0.001))
            self.step_bias = nn.Parameter((step + torch.log(-torch.expm1(-step))).to(device))
            self.log_rate = nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32)).repeat(channels, 1).to(device))
            self.skip = filled(1, channels)
        self.mix_out, self.mix_out_bias = matrix(width, channels), filled(0, width)
        self.norm_out, self.norm_out_bias = filled(1, width), filled(0, width)
        self.head, self.head_bias = matrix(n_outputs, width), filled(0, n_outputs)
        self._matrices = ["embed", "mix_in", "mix_out", "head"] + ([] if attends else ["maps", "step"])
        self._vectors = ["norm_in", "norm_in_bias", "embed_bias", "norm_mix", "norm_mix_bias", "conv", "conv_bias", "mix_out_bias",
                         "norm_out", "norm_out_bias", "head_bias"]
        self._vectors += ["norm_heads", "norm_heads_bias", "log_decay"] if attends else ["step_bias", "skip"]
        if self.feed_forward:
            self.norm_ff, self.norm_ff_bias = filled(1, width), filled(0, width)
            self.ff_in, self.ff_in_bias = matrix(2 * self.feed_forward, width), filled(0, 2 * self.feed_forward)
            self.ff_out, self.ff_out_bias = matrix(width, self.feed_forward), filled(0, width)
            self._matrices += ["ff_in", "ff_out"]
            self._vectors += ["norm_ff", "norm_ff_bias", "ff_in_bias", "ff_out_bias"]

    def get_extra_state(self):
        return torch.tensor(self.drawn, dtype=torch.int64)

    def set_extra_state(self, state):
        self.drawn = int(state)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, *more):
        """A state without the stream's place leaves it where it is."""
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, *more)
        if prefix + "_extra_state" in missing_keys:
            missing_keys.remove(prefix + "_extra_state")

    def _weights(self, own: bool = False):
        """All that the operators read: the matrices in the activations' type, the decay rates, and the rest as it is.  own:
        none of it shares memory with a parameter."""
        w = {k: getattr(self, k).to(self.dtype, copy=own) for k in self._matrices}
        w.update((k, getattr(self, k).clone() if own else getattr(self, k)) for k in self._vectors)
        if self.mixer == "state_space":
            w["A"] = -torch.exp(self.log_rate)
        return w

    def _into(self, x, w):
        """The residual stream h, and the convolution's input and the gates (of attention None)."""
        h = linear(layer_norm(x, w["norm_in"], w["norm_in_bias"]), w["embed"], w["embed_bias"])
        c = linear(layer_norm(h, w["norm_mix"], w["norm_mix_bias"]), w["mix_in"])
        return (h, c, None) if self.mixer == "attention" else (h, *c.split(self.channels, -1))

    def _attended(self, u):
        """The queries, keys and values of convolved channels."""
        keys = self.heads * self.states
        return (t.unflatten(-1, (self.heads, -1)) for t in u.split((keys, keys, self.channels), -1))

    def _of_heads(self, y, w):
        """The attention's answers, each head normed, as channels."""
        return layer_norm(y, w["norm_heads"], w["norm_heads_bias"]).flatten(-2)

    def _maps(self, u, w):
        """The state space's step, input and output maps at every tick of u."""
        n = self.groups * self.states
        low, B, C = linear(u, w["maps"]).split((self.rank, n, n), -1)
        shape = (self.groups, self.states)
        return linear(low, w["step"]), B.unflatten(-1, shape), C.unflatten(-1, shape)

    def _out(self, h, w):
        if self.feed_forward:
            y = gated_linear(layer_norm(h, w["norm_ff"], w["norm_ff_bias"]), w["ff_in"], w["ff_in_bias"])
            h = linear(y, w["ff_out"], w["ff_out_bias"], residual=h)
        return linear(layer_norm(h, w["norm_out"], w["norm_out_bias"]), w["head"], w["head_bias"])

    def _input(self, x, dims):
        if not isinstance(x, torch.Tensor) or x.dim() != dims or x.shape[-1] != self.n_neurons:
            raise ValueError(f"x must be a tensor [{'T, ' * (dims - 2)}B, {self.n_neurons}]")
        return x.to(self.dtype)

    def draw(self, ticks: int, batch_size: int) -> int:
        """Takes the words of one forward off the masks' stream and returns the first: ``drawn`` for a forward that is run
        more than once, as under activation checkpointing (``checkpoint(readout, z, None, readout.draw(T, B))``)."""
        first = self.drawn
        self.drawn += ticks * batch_size * self.width
        return first

    def forward(self, x: torch.Tensor, lengths=None, drawn=None) -> torch.Tensor:
        """x [T, B, n_neurons] (a rollout's spikes or voltages, any floating type) to [T, B, n_outputs] of ``dtype``.
        ``lengths`` (int32 [B] on the device): the ticks of each batch entry; what is behind them is left out of the mixing
        and its outputs mean nothing (x must be finite there, and a loss leaves them out).  ``drawn``: the first word of the
        masks in their stream, from ``draw``; None: the next one, which a forward inside a backward pass (a checkpoint's
        second) cannot know and refuses."""
        x, w = self._input(x, 3), self._weights()
        masks = self.training and self.dropout > 0.0
        if masks and drawn is None:
            if torch._C._current_graph_task_id() != -1:
                raise RuntimeError("a readout that is run again in a backward pass needs the masks of its first run: give it "
                                   "drawn=readout.draw(ticks, batch_size)")
            drawn = self.draw(x.shape[0], x.shape[1])
        h, c, gate = self._into(x, w)
        u, _ = short_conv(c, w["conv"], w["conv_bias"], activation="silu", lengths=lengths)
        if self.mixer == "attention":
            y, _ = linear_attention(*self._attended(u), w["log_decay"], lengths=lengths)
            y = self._of_heads(y, w)
        else:
            delta, B, C = self._maps(u, w)
            y, _ = state_space_scan(u, delta, w["A"], B, C, w["skip"], gate, w["step_bias"], lengths=lengths)
        y = linear(y, w["mix_out"], w["mix_out_bias"])
        if masks:
            h = dropout(y, self.dropout, self.seed, drawn, residual=h)
        else:
            h = h + y
        return self._out(h, w)

    @torch.no_grad()
    def zero_state(self, batch_size: int) -> ReadoutState:
        """The state before the first tick, for ``tick``."""
        dev = self.embed.device
        shape = (self.heads, self.states, self.channels // self.heads) if self.mixer == "attention" else (self.channels, self.states)
        return ReadoutState(torch.zeros(batch_size, self.taps - 1, self.conv.shape[0], dtype=self.dtype, device=dev),
                            torch.zeros(batch_size, *shape, dtype=torch.float32, device=dev), self._weights(own=True))

    @torch.no_grad()
    def tick(self, x: torch.Tensor, state: ReadoutState) -> torch.Tensor:
        """One tick: x [B, n_neurons] to [B, n_outputs], without dropout or gradient; ``state`` is moved on in place."""
        x, w = self._input(x, 2), state.weights
        h, c, gate = self._into(x, w)
        u = short_conv_step(c, state.conv, w["conv"], w["conv_bias"], activation="silu")
        if self.mixer == "attention":
            q, k, v = self._attended(u)
            y = self._of_heads(linear_attention_step(q, k, v, state.scan, w["log_decay"]), w)
        else:
            delta, B, C = self._maps(u, w)
            y = state_space_step(u, state.scan, delta, w["A"], B, C, w["skip"], gate, w["step_bias"])
        return self._out(linear(y, w["mix_out"], w["mix_out_bias"], residual=h), w)


def example(steps: int = 60, ticks: int = 100, batch: int = 16, classes: int = 4, seed: int = 0, say=print,
            mixer: str = "state_space", feed_forward: int = 0, state_bits: int = 32):
    """Trains a small column and its readout together on which group of LGN units fires, then reads the pair out tick by
    tick; ``mixer`` and ``feed_forward`` are the readout's, ``state_bits`` its optimizer's.  Returns (the losses, the share of right answers over the last quarter of new rollouts, read out by ticks)."""
    import dataclasses

    from . import synthetic
    from .inputs import sample_bkg, sample_lgn
    from .models import RSNNRollout, V1Column
    from .optim import AdamW, ExponentiatedAdam

    cfg = dataclasses.replace(synthetic.CONFIGS[0], n_neurons=400, fanin_mean=40, max_delay=3, n_lgn=100, lgn_fanin=10,
                              n_bkg=10, bkg_fanin=3, recurrent_weight_scale=2.0, input_weight_scale=3.0)
    cell = V1Column(synthetic.make_network(cfg, seed=seed, dense_basis=True), train_input=True, train_recurrent_per_type=False,
                    gauss_std=0.5, dampening_factor=0.5, recurrent_dampening_factor=0.5, pseudo_gauss=True)
    weights = (cell.recurrent_weight_values, cell.input_weight_values, cell.bkg_input_weights)
    positive = (cell.recurrent_weight_positive, cell.input_weight_positive, cell.bkg_weight_positive)
    readout = SequenceReadout(cfg.n_neurons, classes, width=64, channels=128, seed=seed, device=cell.device, mixer=mixer,
                              feed_forward=feed_forward)
    of_column, of_readout = ExponentiatedAdam(1e-3), AdamW(readout.parameters(), 3e-3, weight_decay=0.0, state_bits=state_bits)
    rng = torch.Generator().manual_seed(seed)

    def stimuli(n):
        """Labels, and inputs in which the label's group of LGN units fires at 80 Hz and the rest at 10."""
        label = torch.randint(classes, (batch,), generator=rng)
        group = torch.arange(cfg.n_lgn) * classes // cfg.n_lgn
        rate = torch.where(group[None] == label[:, None], 80.0, 10.0).expand(ticks, batch, cfg.n_lgn)
        bkg = sample_bkg(ticks, batch, cfg.n_bkg, seed + 1, offset=n * ticks * batch * cfg.n_bkg, device=cell.device)
        return label.to(cell.device), sample_lgn(rate, seed + 2, offset=n * ticks * batch * cfg.n_lgn), bkg

    losses = []
    for n in range(steps):
        label, lgn, bkg = stimuli(n)
        z, _ = RSNNRollout.apply(cell, lgn, bkg, *weights)
        logits = readout(z)[ticks // 2:].float()
        loss = nn.functional.cross_entropy(logits.flatten(0, 1), label.repeat(logits.shape[0]))
        loss.backward()
        of_column.apply_gradients([(w.grad, w) for w in weights], {id(w): p for w, p in zip(weights, positive)})
        of_readout.apply_gradients()
        for w in weights:
            w.grad = None
        readout.zero_grad(set_to_none=True)
        losses.append(float(loss.detach()))
        if n % 10 == 9:
            say(f"step {n + 1}: loss {sum(losses[-10:]) / 10:.4f}")
    readout.eval()
    label, lgn, bkg = stimuli(steps)
    state, mine, right = cell.zero_state(batch), readout.zero_state(batch), []
    with torch.no_grad():
        for t in range(ticks):
            (z, _), state = cell.call(lgn[t], state, bkg[t])
            answer = readout.tick(z, mine).argmax(-1)
            if t >= ticks - ticks // 4:
                right.append((answer == label).float().mean())
    share = float(torch.stack(right).mean())
    say(f"read out by ticks: {100 * share:.1f} % right")
    return losses, share


if __name__ == "__main__":
    import argparse

    of = argparse.ArgumentParser(description="Trains a small column with its readout, and reads the pair out by ticks.")
    of.add_argument("--mixer", choices=("state_space", "attention"), default="state_space")
    of.add_argument("--feed-forward", type=int, default=0, metavar="CHANNELS")
    of.add_argument("--state-bits", type=int, choices=(8, 32), default=32, help="of the readout's moments")
    example(**vars(of.parse_args()))
