"""ExponentiatedAdam and SignedConstraint on the GPU (v1_model_utils/optimizers.py:154-390,
models.py:419-427), and AdamW for a readout's variables.

Same names and arguments as the reference.  ``apply_gradients`` runs the dense
``update_step`` and then the variable's sign constraint in one libglif kernel
(``glif_exp_adam``) per variable; the moment slots live on the device beside the
weights.  Weight vectors are fp32 device tensors updated in place.

``AdamW`` steps all of its variables in one launch, with moments in 32 bits or in 8.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from ._lib import check, lib, ptr, require_gpu, stream_ptr
from .sequence import DTYPES, _on, _p

__all__ = ["ExponentiatedAdam", "SignedConstraint", "AdamW"]


class SignedConstraint:
    """``w -> where(positive, relu(w), -relu(-w))`` (models.py:419-427).

    ``positive``: bool / uint8 tensor, True where the weight must stay >= 0."""

    def __init__(self, positive):
        self.condition = torch.as_tensor(positive).to(torch.uint8).contiguous()

    def __call__(self, w):
        return torch.where(self.condition.bool().to(w.device), torch.relu(w), -torch.relu(-w))


class ExponentiatedAdam:
    """Adam moments with the exponentiated update ``w <- w * exp(-alpha * m / (sqrt(v) + eps)
    * sign(w))`` (sign(0) = +1), optionally AMSGrad; the dense branch of
    ``ExponentiatedAdam.update_step`` (optimizers.py:268-376, dense branch :354-376)."""

    def __init__(self, learning_rate=0.001, beta_1=0.9, beta_2=0.999, epsilon=1e-7, amsgrad=False,
                 name="ExponentiatedAdam"):
        self.learning_rate = learning_rate
        self.beta_1, self.beta_2, self.epsilon = beta_1, beta_2, epsilon
        self.amsgrad = bool(amsgrad)
        self.name = name
        self.iterations = 0
        self._slots = {}

    def _lr(self):
        lr = self.learning_rate
        return float(lr(self.iterations) if callable(lr) else lr)

    def alpha(self):
        """alpha of the next step in fp32, as update_step forms it (optimizers.py:273-283)."""
        f = np.float32
        t = f(self.iterations + 1)
        b1p = np.power(f(self.beta_1), t)
        b2p = np.power(f(self.beta_2), t)
        return f(f(self._lr()) * np.sqrt(f(1) - b2p)) / (f(1) - b1p)

    def slots(self, var):
        key = var.data_ptr()
        s = self._slots.get(key)
        if s is None:
            z = lambda: torch.zeros_like(var)   # noqa: E731
            s = {"m": z(), "v": z(), "vhat": z() if self.amsgrad else None}
            self._slots[key] = s
        return s

    def apply_gradients(self, grads_and_vars, constraints=None):
        """One step over every (gradient, variable) pair, then iterations += 1.

        ``constraints``: optional {id(var) or var.data_ptr(): SignedConstraint or a
        positive-mask tensor}; a constrained variable is projected in the same kernel."""
        require_gpu()
        alpha = self.alpha()
        for g, var in grads_and_vars:
            if g is None:
                continue
            if var.dtype != torch.float32 or not var.is_cuda or not var.is_contiguous():
                raise ValueError("variables must be contiguous fp32 device tensors")
            g = g.to(device=var.device, dtype=torch.float32).contiguous()
            if g.shape != var.shape:
                raise ValueError("gradient and variable shapes differ")
            pos = None
            if constraints:
                c = constraints.get(var.data_ptr(), constraints.get(id(var)))
                if c is not None:
                    pos = (c.condition if isinstance(c, SignedConstraint) else torch.as_tensor(c))
                    pos = pos.to(device=var.device, dtype=torch.uint8).contiguous()
            s = self.slots(var)
            with torch.no_grad():
                check(lib().glif_exp_adam(ptr(var), ptr(s["m"]), ptr(s["v"]), ptr(s["vhat"]), ptr(g),
                                          ptr(pos), var.numel(), float(alpha), float(self.beta_1),
                                          float(self.beta_2), float(self.epsilon), stream_ptr(var.device)))
            # the kernel wrote through a raw pointer: mark the tensor modified, so the weight
            # copies the synapse tables keep (keyed on the tensor's version) are refreshed
            torch.autograd.graph.increment_version(var)
        self.iterations += 1


class AdamW:
    """Adam with decoupled weight decay over a fixed list of variables, one launch a step (of up to 64 of them):

    ``m = beta_1 m + (1 - beta_1) g``, ``v = beta_2 v + (1 - beta_2) g^2``,
    ``p = (1 - lr weight_decay) p - lr / (1 - beta_1^t) m / (sqrt(v / (1 - beta_2^t)) + epsilon)``

    ``variables``: contiguous float32, bfloat16 or float16 tensors of one GPU, updated in place (16-bit ones rounded to nearest).
    ``state_bits``: 32, or 8 for moments of a byte each with a float32 scale for every 256: m as ``s (c / 127) |c / 127|`` and v
    as ``s (c / 255)^4``, rounded up or down by words of the Philox stream ``seed`` so that their mean is kept.  A gradient that is
    not finite makes its variable's moments so, in 8 bits those of all 256.  The square of one below some 1e-19 is 0 to v, so
    ``epsilon`` is at least 1e-12.

    The count of steps lies on the device: a captured step that is replayed goes on counting.  It keeps the ``learning_rate``
    that it was captured with; eager steps read the attribute each time."""

    BLOCK = 256

    def __init__(self, variables, learning_rate=0.001, beta_1=0.9, beta_2=0.999, epsilon=1e-8, weight_decay=0.01,
                 state_bits=32, seed=0, name="AdamW"):
        require_gpu()
        self.variables = list(variables)
        if not self.variables:
            raise ValueError("there must be at least one variable")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        for what, b in (("beta_1", beta_1), ("beta_2", beta_2)):
            if not 0.0 <= b < 1.0:
                raise ValueError(f"{what} must be in [0, 1), got {b}")
        for what, b, least in (("epsilon", epsilon, 1e-12), ("weight_decay", weight_decay, 0.0)):
            if not least <= b < math.inf:
                raise ValueError(f"{what} must be >= {least:g} and finite, got {b}")
        dev = getattr(self.variables[0], "device", None)
        for p in self.variables:
            self._check(p)
            if p.device != dev:
                raise ValueError(f"all variables must be on one device, got {dev} and {p.device}")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.variables if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two variables share memory")
        self.learning_rate = learning_rate
        self.beta_1, self.beta_2, self.epsilon, self.weight_decay = float(beta_1), float(beta_2), float(epsilon), float(weight_decay)
        self.state_bits, self.seed, self.name, self.device = int(state_bits), int(seed) & (2 ** 64 - 1), name, dev
        self._types = [p.dtype for p in self.variables]
        self._shapes = [p.shape for p in self.variables]
        self._homes = [0]
        for p in self.variables:
            self._homes.append(self._homes[-1] + -(-p.numel() // self.BLOCK) * self.BLOCK)
        n = self._homes[-1]
        self._strides = [torch.empty(s, device="meta").stride() for s in self._shapes]

        def zeros(n, dtype):
            return torch.zeros(n, dtype=dtype, device=dev)

        if self.state_bits == 32:
            self._first, self._second = zeros(n, torch.float32), zeros(n, torch.float32)
            self._scales = None
        else:
            self._first, self._second = zeros(n, torch.int8), zeros(n, torch.uint8)
            self._scales = zeros(n // self.BLOCK, torch.float32), zeros(n // self.BLOCK, torch.float32)
        self._own = [[self._views(flat, i) for i in range(len(self.variables))] for flat in (self._first, self._second)]
        self._count = zeros(2, torch.int64)      # steps done; the kernel's own
        count = len(self.variables)
        self._sizes = (ctypes.c_int64 * count)(*(p.numel() for p in self.variables))
        self._codes = (ctypes.c_int32 * count)(*(DTYPES[p.dtype] for p in self.variables))
        self._pointers = ctypes.c_void_p * count
        self._ints = ctypes.c_int32 * count

    @staticmethod
    def _check(p):
        if (not isinstance(p, torch.Tensor) or p.layout is not torch.strided or not p.is_cuda or p.dtype not in DTYPES
                or not p.is_contiguous()):
            raise ValueError("variables must be contiguous float32, bfloat16 or float16 tensors on the GPU")

    @property
    def iterations(self) -> int:
        """The steps done (waits for the device)."""
        return int(self._count[0])

    def apply_gradients(self, gradients=None):
        """One step.  ``gradients``: one for each variable, float32 or of its type, None for a variable that stays as it is with
        its moments; by default the variables' ``grad``.  Without any gradient nothing is done or counted."""
        if gradients is None:
            gradients = [p.grad for p in self.variables]
        gradients = list(gradients)
        if len(gradients) != len(self.variables):
            raise ValueError(f"there are {len(self.variables)} variables and {len(gradients)} gradients")
        held, kinds, changed, index = [], [], [], self.device.index
        for g, p, dtype, shape in zip(gradients, self.variables, self._types, self._shapes):
            if p.dtype is not dtype or p.shape != shape or p.get_device() != index or not p.is_contiguous():
                raise ValueError("a variable is not laid out as it was when the optimizer was made")
            if g is None:
                held.append(None)
                kinds.append(0)
                continue
            if not isinstance(g, torch.Tensor) or g.layout is not torch.strided or g.get_device() != index or g.shape != shape or (
                    g.dtype is not dtype and g.dtype is not torch.float32):
                raise ValueError(f"a gradient must be a dense tensor of its variable's shape {tuple(shape)} and device, float32 or of its type")
            if not g.is_contiguous():
                g = g.contiguous()
            held.append(g)
            kinds.append(DTYPES[g.dtype])
            changed.append(p)
        if not changed:
            return
        first_scale, second_scale = self._scales or (None, None)
        with _on(self.device):
            check(lib().glif_adamw(len(held), self._pointers(*(p.data_ptr() for p in self.variables)), self._codes,
                                   self._pointers(*(_p(g) for g in held)), self._ints(*kinds), self._sizes, self.state_bits,
                                   _p(self._first), _p(self._second), _p(first_scale), _p(second_scale), _p(self._count),
                                   float(self.learning_rate), self.beta_1, self.beta_2, self.epsilon, self.weight_decay, self.seed,
                                   stream_ptr(self.device)))
        torch.autograd.graph.increment_version(changed)

    def _views(self, flat, i):
        return flat.as_strided(self._shapes[i], self._strides[i], self._homes[i])

    def moments(self):
        """The first and the second moments as float32 values, a list of each: the state itself where it is held in 32 bits,
        what the codes stand for where in 8."""
        if self.state_bits == 32:
            return list(self._own[0]), list(self._own[1])
        first, second = (torch.empty(self._first.numel(), dtype=torch.float32, device=self.device) for _ in range(2))
        with _on(self.device):
            check(lib().glif_adamw_values(_p(self._first), _p(self._scales[0]), _p(self._second), _p(self._scales[1]), first.numel(),
                                          _p(first), _p(second), stream_ptr(self.device)))
        homes = list(zip(self._shapes, self._strides, self._homes))
        return [first.as_strided(*h) for h in homes], [second.as_strided(*h) for h in homes]

    def _scale_views(self, k, i):
        return self._scales[k][self._homes[i] // self.BLOCK:self._homes[i + 1] // self.BLOCK]

    def _state(self, k, i):
        codes = self._own[k][i]
        return codes if self.state_bits == 32 else (codes, self._scale_views(k, i))

    def state_dict(self):
        """``iterations`` and, for each variable, its ``first`` and ``second`` moments (in 8 bits: the codes and their scales),
        as copies.  The learning rate and the other numbers are the caller's."""
        def copy(s):
            return s.clone() if isinstance(s, torch.Tensor) else tuple(t.clone() for t in s)
        count = range(len(self.variables))
        return dict(iterations=self.iterations, first=[copy(self._state(0, i)) for i in count],
                    second=[copy(self._state(1, i)) for i in count])

    def load_state_dict(self, state):
        """Takes what ``state_dict`` gave for variables of these shapes and the same ``state_bits``."""
        pairs = []
        for k, what in enumerate(("first", "second")):
            if len(state[what]) != len(self.variables):
                raise ValueError(f"{what} has {len(state[what])} moments for {len(self.variables)} variables")
            for i, new in enumerate(state[what]):
                old, new = ([s] if isinstance(s, torch.Tensor) else list(s) for s in (self._state(k, i), new))
                if len(old) != len(new) or any(a.shape != b.shape or a.dtype is not b.dtype for a, b in zip(old, new)):
                    raise ValueError(f"{what}[{i}] does not fit the variable and state_bits = {self.state_bits}")
                pairs += zip(old, new)
        count = int(state["iterations"])
        if count < 0:
            raise ValueError(f"iterations must be >= 0, got {count}")
        for old, new in pairs:
            old.copy_(new)
        self._count.copy_(torch.tensor([count, 0]))
