"""Sequence operators on the GPU: what a readout of the column's activity is made of.

The reference reads its rollouts out with Keras layers (a Dense or a softmax readout, models.py:1138-1209, 1213-1392);
these are the operators of a trained readout over whole training windows and, tick by tick, beside ``V1Column.call``:

* ``layer_norm``                                    over the last axis;
* ``dropout``                                       its mask drawn from the Philox streams of ``inputs`` and never stored;
* ``linear``                                        with bias, activation and residual in one kernel;
* ``gated_linear``                                  both projections of a gated feed-forward block, activation and product;
* ``short_conv``, ``short_conv_step``               a causal convolution of a few ticks per channel;
* ``state_space_scan``, ``state_space_step``        a selective state space;
* ``linear_attention``, ``linear_attention_step``   linear attention with a decay for each head.

Activations are float32, bfloat16 or float16 tensors on the GPU; statistics, sums and states are float32 and every output
is rounded once.  Sequences are time-major ``[T, B, D]`` like the rollouts.  ``lengths`` (int32 ``[B]``, on the device)
gives every batch entry's own number of ticks: those behind it are not read, give zeros and take no part in gradients.
All operators but the steps are differentiable once, backwards; forward-mode derivatives are refused.  Each runs in libglif on the current stream; there is no CPU path.
"""
from __future__ import annotations

import contextlib
import math
from ctypes import byref

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib

__all__ = ["layer_norm", "dropout", "linear", "gated_linear", "short_conv", "short_conv_step", "state_space_scan", "state_space_step",
           "linear_attention", "linear_attention_step"]

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}


# ------------------------------------------------------------------ the arguments ----
def _need(t, name, shape=None, dtype=None, device=None):
    """ValueError unless ``t`` is a device tensor of the wanted shape (None: any size), type and device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        if isinstance(t, torch.Tensor):
            _lib.require_gpu()
        raise ValueError(f"{name} must be a tensor on the GPU")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other arguments are on {device}")
    if dtype is not None and t.dtype is not dtype and t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"{name} must be of type {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape and (
            t.dim() != len(shape) or any(w is not None and w != h for w, h in zip(shape, t.shape))):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _activations(t, name):
    _need(t, name)
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return t


def _params(x, weight, wshape, bias, bshape):
    """The type of the small parameters that are given: float32 or x's, the same for both."""
    w = weight if weight is not None else bias
    if w is None:
        return torch.float32
    kind = w.dtype if isinstance(w, torch.Tensor) else None
    if weight is not None:
        _need(weight, "weight", wshape, (torch.float32, x.dtype), x.device)
    if bias is not None:
        _need(bias, "bias", bshape, (torch.float32, x.dtype), x.device)
        if bias.dtype is not kind:
            raise ValueError("weight and bias must be of one type")
    return kind


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _rows(t, D):
    """t [..., D] as rows of D contiguous elements at one stride, which is returned with it (copied only if it is not laid
    out so)."""
    if t.is_contiguous():
        return t, D
    if t.dim() == 2:
        r = t
    else:
        n = t.numel() // D if D else 0
        try:
            r = t.view(n, D)
        except RuntimeError:
            return t.contiguous(), D
    n, step = r.shape[0], r.stride(0)
    if (D > 1 and r.stride(1) != 1) or (n > 1 and step >= 1 << 24):
        return r.contiguous(), D
    return r, step if n > 1 else D


def _seq(t):
    """t [T, B, ...] with everything behind the first two dimensions contiguous."""
    if t is None or t.is_contiguous():
        return t
    want = 1
    for k in range(t.dim() - 1, 1, -1):
        if t.shape[k] != 1 and t.stride(k) != want:
            return t.contiguous()
        want *= t.shape[k]
    return t


def _lengths(lengths, x, B):
    return None if lengths is None else _dense(_need(lengths, "lengths", (B,), torch.int32, x.device))


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _size(ws):
    return 0 if ws is None else ws.numel()


_HERE = contextlib.nullcontext()


def _on(device):
    """The calls below launch on the current device: make it the tensors'."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _p(t):
    """A tensor's address for a C argument (None: NULL)."""
    return None if t is None else t.data_ptr()


def _stream(device):
    return _lib._raw_stream(device.index)


def _first_only(name):
    """The gradients are computed outside autograd: a graph of them would be wrong without a word."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} is differentiable once: create_graph is not supported")


def _has_tangent(*tensors):
    """Whether a tensor carries a forward-mode derivative, which does not make it require a gradient."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _wants_grad(*tensors):
    """Whether autograd has to see the call: for a gradient, or to refuse a forward-mode derivative."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return _has_tangent(*tensors)


def _refuse_grad(name, *tensors):
    if _has_tangent(*tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")
    if _wants_grad(*tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or use the form for whole sequences")


class _NoCtx:
    """Stands in for the autograd context where no gradient is wanted."""
    needs_input_grad = (False,) * 16

    def save_for_backward(self, *tensors):
        pass

    def set_materialize_grads(self, value):
        pass


def _apply(fn, wants, *args):
    return fn.apply(*args) if wants else fn.forward(_NoCtx(), *args)


# ------------------------------------------------------------------------ layer norm ----
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, pdt):
        D = x.shape[-1]
        xr, xs = _rows(x, D)
        w, b, dev = _dense(weight), _dense(bias), x.device
        y = x.new_empty(x.shape)
        with _on(dev):
            check(lib().glif_layer_norm_fwd(_p(xr), xs, _p(w), _p(b), DTYPES[x.dtype], DTYPES[pdt], x.numel() // D, D, eps,
                                            _p(y), _stream(dev)))
        ctx.save_for_backward(x, weight)
        ctx.eps, ctx.pdt = eps, pdt
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_only("layer_norm")
        x, weight = ctx.saved_tensors
        D, dev, dt, L = x.shape[-1], x.device, DTYPES[x.dtype], lib()
        xr, xs = _rows(x, D)
        gr, gs = _rows(dy, D)
        wx, ww, wb = ctx.needs_input_grad[:3]
        dx = x.new_empty(x.shape) if wx else None
        dw = torch.empty(D, dtype=ctx.pdt, device=dev) if ww else None
        db = torch.empty(D, dtype=ctx.pdt, device=dev) if wb else None
        rows = x.numel() // D
        n = L.glif_layer_norm_bwd_workspace(rows, D, dt, ww or wb)
        ws, w = _workspace(n, dev), _dense(weight)
        with _on(dev):
            check(L.glif_layer_norm_bwd(_p(gr), gs, _p(xr), xs, _p(w), dt, DTYPES[ctx.pdt], rows, D, ctx.eps, _p(dx), _p(dw),
                                        _p(db), _p(ws), n, _stream(dev)))
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis; ``weight`` and ``bias`` [D] float32 or of x's
    type, or None."""
    _activations(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one element in its last axis")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    D = x.shape[-1]
    pdt = _params(x, weight, (D,), bias, (D,))
    return _apply(_LayerNorm, _wants_grad(x, weight, bias), x, weight, bias, float(eps), pdt)


# --------------------------------------------------------------------------- dropout ----
def _dropout(x, residual, p, seed, offset):
    x, residual = _dense(x), _dense(residual)
    y = x.new_empty(x.shape)
    with _on(x.device):
        check(lib().glif_dropout(_p(x), _p(residual), DTYPES[x.dtype], x.numel(), p, seed, offset, _p(y), _stream(x.device)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.draw = (p, seed, offset)
        return _dropout(x, residual, p, seed, offset)

    @staticmethod
    def backward(ctx, dy):
        _first_only("dropout")
        dx = _dropout(dy, None, *ctx.draw) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0, residual=None) -> torch.Tensor:
    """``where(u >= p, x / (1 - p), 0) + residual``: element i (in row-major order) is dropped where the uniform of word
    ``offset + i`` of the Philox stream ``seed`` is below ``p``, as ``inputs.bernoulli`` sets it.  Calls with offsets that
    are x.numel() apart continue one stream; the gradient draws the same mask again."""
    _activations(x, "x")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if int(offset) < 0 or int(offset) >= 2 ** 63:
        raise ValueError(f"offset must be in [0, 2^63), got {offset}")
    if residual is not None:
        _need(residual, "residual", x.shape, x.dtype, x.device)
    return _apply(_Dropout, _wants_grad(x, residual), x, residual, float(p), int(seed) & (2 ** 64 - 1), int(offset))


# ---------------------------------------------------------------------------- linear ----
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, bdt):
        N, K = weight.shape
        dt = DTYPES[x.dtype]
        M = math.prod(x.shape[:-1])
        xr, ldx = _rows(x, K) if K else (x, 0)
        wr, ldw = _rows(weight, K) if K else (weight, 0)
        rr, ldr = _rows(residual, N) if residual is not None else (None, 0)
        b = _dense(bias)
        y = x.new_empty((*x.shape[:-1], N))
        pre = torch.empty((M, N), dtype=torch.float32, device=x.device) if act and any(ctx.needs_input_grad[:3]) else None
        L, dev = lib(), x.device
        n = L.glif_linear_fwd_workspace(dt, M, N, K)
        ws = _workspace(n, dev)
        with _on(dev):
            check(L.glif_linear_fwd(_p(xr), ldx, _p(wr), ldw, _p(b), _p(rr), ldr, dt, DTYPES[bdt], M, N, K, act, _p(y),
                                    _p(pre), _p(ws), n, _stream(dev)))
        ctx.save_for_backward(x, weight, pre)
        ctx.act, ctx.bdt, ctx.M = act, bdt, M
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_only("linear")
        x, weight, pre = ctx.saved_tensors
        N, K = weight.shape
        M, dt, dev = ctx.M, DTYPES[x.dtype], x.device
        xr, ldx = _rows(x, K) if K else (x, 0)
        wr, ldw = _rows(weight, K) if K else (weight, 0)
        gr, ldg = _rows(dy, N) if N else (dy, 0)
        wx, ww, wb, wr_ = ctx.needs_input_grad[:4]
        dx = x.new_empty(x.shape) if wx else None
        dw = x.new_empty((N, K)) if ww else None
        db = torch.empty(N, dtype=ctx.bdt, device=dev) if wb else None
        if wx or ww or wb:
            L, V = lib(), 16 // x.element_size()
            px, pw, pg = xr.data_ptr(), wr.data_ptr(), gr.data_ptr()
            odd = (ldx % V or ldw % V or ldg % V or N % V or K % V or (px | pw | pg) % 16) != 0
            n = L.glif_linear_bwd_workspace(dt, M, N, K, ctx.act, odd)
            ws = _workspace(n, dev)
            with _on(dev):
                check(L.glif_linear_bwd(pg, ldg, _p(pre), px, ldx, pw, ldw, dt, DTYPES[ctx.bdt], M, N, K, ctx.act, _p(dx),
                                        _p(dw), _p(db), _p(ws), n, _stream(dev)))
        return dx, dw, db, dy if wr_ else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias=None, activation=None, residual=None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: x [..., K], weight [N, K] of x's type, bias [N] float32 or of x's type,
    residual [..., N]; ``activation``: None, "relu", "gelu" (the error function's) or "silu".

    For the gradient of an activation its argument is kept in float32.  The gradient behind the activation is rounded to x's
    type for the products that give the gradients of x and weight (the matrix cores take no wider operands beside 16-bit
    ones); the bias's is summed from its float32 values."""
    _activations(x, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS]}, got {activation!r}")
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    _need(weight, "weight", (None, x.shape[-1]), x.dtype, x.device)
    N = weight.shape[0]
    bdt = _params(x, None, None, bias, (N,))
    if residual is not None:
        _need(residual, "residual", (*x.shape[:-1], N), x.dtype, x.device)
    return _apply(_Linear, _wants_grad(x, weight, bias, residual), x, weight, bias, residual, ACTIVATIONS[activation], bdt)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, bdt):
        N, K = weight.shape[0] // 2, weight.shape[1]
        dt = DTYPES[x.dtype]
        M = math.prod(x.shape[:-1])
        xr, ldx = _rows(x, K) if K else (x, 0)
        wr, ldw = _rows(weight, K) if K else (weight, 0)
        b = _dense(bias)
        y = x.new_empty((*x.shape[:-1], N))
        pre = torch.empty((M, 2 * N), dtype=torch.float32, device=x.device) if any(ctx.needs_input_grad[:3]) else None
        L, dev = lib(), x.device
        n = L.glif_gated_linear_fwd_workspace(dt, M, N, K)
        ws = _workspace(n, dev)
        with _on(dev):
            check(L.glif_gated_linear_fwd(_p(xr), ldx, _p(wr), ldw, _p(b), dt, DTYPES[bdt], M, N, K, act, _p(y), _p(pre), _p(ws), n,
                                          _stream(dev)))
        ctx.save_for_backward(x, weight, pre)
        ctx.act, ctx.bdt, ctx.M = act, bdt, M
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_only("gated_linear")
        x, weight, pre = ctx.saved_tensors
        N, K = weight.shape[0] // 2, weight.shape[1]
        M, dt, dev = ctx.M, DTYPES[x.dtype], x.device
        xr, ldx = _rows(x, K) if K else (x, 0)
        wr, ldw = _rows(weight, K) if K else (weight, 0)
        gr, ldg = _rows(dy, N) if N else (dy, 0)
        wx, ww, wb = ctx.needs_input_grad[:3]
        dx = x.new_empty(x.shape) if wx else None
        dw = x.new_empty((2 * N, K)) if ww else None
        db = torch.empty(2 * N, dtype=ctx.bdt, device=dev) if wb else None
        L, V = lib(), 16 // x.element_size()
        px, pw = xr.data_ptr(), wr.data_ptr()
        odd = (ldx % V or ldw % V or K % V or (px | pw) % 16) != 0
        n = L.glif_gated_linear_bwd_workspace(dt, M, N, K, odd)
        ws = _workspace(n, dev)
        with _on(dev):
            check(L.glif_gated_linear_bwd(_p(gr), ldg, _p(pre), px, ldx, pw, ldw, dt, DTYPES[ctx.bdt], M, N, K, ctx.act, _p(dx),
                                          _p(dw), _p(db), _p(ws), n, _stream(dev)))
        return dx, dw, db, None, None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias=None, activation="silu") -> torch.Tensor:
    """``act(x @ weight[:N].T + bias[:N]) * (x @ weight[N:].T + bias[N:])``: the first half of a gated feed-forward block, whose
    second is a ``linear`` with the residual.  x [..., K], weight [2 N, K] of x's type, bias [2 N] float32 or of x's type;
    ``activation``: None, "relu", "gelu" (the error function's) or "silu".

    For the gradient both products are kept in float32; what reaches them is rounded to x's type for the products that give the
    gradients of x and weight, as in ``linear`` (in bfloat16 they are 2.3e-3 from exact ones, where their own last rounding leaves
    1.7e-3), and summed in float32 for the bias's."""
    _activations(x, "x")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS]}, got {activation!r}")
    if x.dim() < 1:
        raise ValueError("x must have at least one axis")
    _need(weight, "weight", (None, x.shape[-1]), x.dtype, x.device)
    if weight.shape[0] % 2:
        raise ValueError(f"weight must have an even number of rows, got {weight.shape[0]}")
    bdt = _params(x, None, None, bias, (weight.shape[0],))
    return _apply(_GatedLinear, _wants_grad(x, weight, bias), x, weight, bias, ACTIVATIONS[activation], bdt)


# ----------------------------------------------------------------- short convolution ----
class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, pdt):
        T, B, D = x.shape
        W = weight.shape[1]
        ctx.set_materialize_grads(False)
        xs, w, b, st = _seq(x), _dense(weight), _dense(bias), _dense(state)
        y, last = x.new_empty((T, B, D)), x.new_empty((B, W - 1, D))
        with _on(x.device):
            check(lib().glif_short_conv_fwd(_p(xs), xs.stride(0), xs.stride(1), _p(w), _p(b), _p(st), _p(lengths),
                                            DTYPES[x.dtype], DTYPES[pdt], T, B, D, W, silu, _p(y), _p(last),
                                            _stream(x.device)))
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu, ctx.pdt = silu, pdt
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        _first_only("short_conv")
        x, weight, bias, state, lengths = ctx.saved_tensors
        (T, B, D), W, dev = x.shape, weight.shape[1], x.device
        wx, ww, wb, ws_ = ctx.needs_input_grad[:4]
        dy = _seq(dy) if dy is not None else torch.zeros((T, B, D), dtype=x.dtype, device=dev)
        dlast, xs, w, b, st = _dense(dlast), _seq(x), _dense(weight), _dense(bias), _dense(state)
        dx = x.new_empty((T, B, D)) if wx else None
        dw = torch.empty((D, W), dtype=ctx.pdt, device=dev) if ww else None
        db = torch.empty(D, dtype=ctx.pdt, device=dev) if wb else None
        ds = x.new_empty((B, W - 1, D)) if ws_ else None
        n = lib().glif_short_conv_bwd_workspace(DTYPES[x.dtype], T, B, D, W) if ww or wb else 0
        ws = _workspace(n, dev)
        with _on(dev):
            check(lib().glif_short_conv_bwd(_p(dy), dy.stride(0), dy.stride(1), _p(dlast), _p(xs), xs.stride(0), xs.stride(1),
                                            _p(w), _p(b), _p(st), _p(lengths), DTYPES[x.dtype], DTYPES[ctx.pdt], T, B, D, W,
                                            ctx.silu, _p(dx), _p(dw), _p(db), _p(ds), _p(ws), n, _stream(dev)))
        return dx, dw, db, ds, None, None, None


def _conv_args(x, weight, bias, activation):
    if activation not in (None, "none", "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    D = x.shape[-1]
    if D < 1:
        raise ValueError("x must have at least one channel")
    _need(weight, "weight", (D, None))
    W = weight.shape[1]
    if not 1 <= W <= 8:
        raise ValueError(f"weight must have 1 to 8 taps, got {W}")
    return int(activation == "silu"), W, _params(x, weight, (D, W), bias, (D,))


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias=None, activation=None, initial_state=None, lengths=None):
    """``act(bias + sum_k weight[:, k] * x[t - (W - 1) + k])`` per channel: x [T, B, D], weight [D, W] (W <= 8) and bias [D]
    float32 or of x's type, ``activation`` None or "silu".  Returns y [T, B, D] and the state [B, W - 1, D], the last
    inputs of each batch entry, which ``initial_state`` (zeros if None) or ``short_conv_step`` goes on from."""
    _activations(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be [T, B, D], got shape {tuple(x.shape)}")
    T, B, D = x.shape
    silu, W, pdt = _conv_args(x, weight, bias, activation)
    if initial_state is not None:
        _need(initial_state, "initial_state", (B, W - 1, D), x.dtype, x.device)
    lengths = _lengths(lengths, x, B)
    return _apply(_ShortConv, _wants_grad(x, weight, bias, initial_state), x, weight, bias, initial_state, lengths, silu, pdt)


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias=None, activation=None) -> torch.Tensor:
    """One tick of ``short_conv``: x [B, D]; ``state`` [B, W - 1, D] is moved on in place.  No gradient."""
    _activations(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be [B, D], got shape {tuple(x.shape)}")
    B, D = x.shape
    silu, W, pdt = _conv_args(x, weight, bias, activation)
    _need(state, "state", (B, W - 1, D), x.dtype, x.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is written in place")
    _refuse_grad("short_conv_step", x, state, weight, bias)
    x = x if D == 1 or x.stride(1) == 1 else x.contiguous()
    w, b = _dense(weight), _dense(bias)
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    with _on(x.device):
        check(lib().glif_short_conv_step(_p(x), x.stride(0), _p(state), _p(w), _p(b), DTYPES[x.dtype], DTYPES[pdt], B, D, W,
                                         silu, _p(y), _stream(x.device)))
    torch.autograd.graph.increment_version(state)
    return y


# ------------------------------------------------------------------------ state space ----
def _scan_struct(u, delta, A, B_, C_, D, z, bias, state, lengths, softplus, ticks):
    """glif_scan of contiguous-enough tensors (held by the caller)."""
    if ticks:
        strides = [t.stride()[:2] if t is not None else (0, 0) for t in (u, delta, z, B_, C_)]
    else:
        strides = [(0, t.stride(0)) if t is not None else (0, 0) for t in (u, delta, z, B_, C_)]
    return _lib.Scan(_p(u), _p(delta), _p(z), _p(B_), _p(C_), _p(A), _p(D), _p(bias), _p(state), _p(lengths),
                     *(n for pair in strides for n in pair), DTYPES[u.dtype], u.shape[0] if ticks else 1, u.shape[-2], u.shape[-1],
                     B_.shape[-2], A.shape[1], softplus)


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B_, C_, D, z, bias, state, lengths, softplus):
        ctx.set_materialize_grads(False)
        (T, B, Dc), dev = u.shape, u.device
        held = [_seq(u), _seq(delta), _dense(A), _seq(B_), _seq(C_), _dense(D), _seq(z), _dense(bias), _dense(state), lengths]
        s = _scan_struct(*held, softplus, True)
        y = torch.empty((T, B, Dc), dtype=u.dtype, device=dev)
        last = torch.empty((B, Dc, A.shape[1]), dtype=torch.float32, device=dev)
        L = lib()
        keep = _workspace(L.glif_scan_keep_bytes(byref(s)), dev) if any(ctx.needs_input_grad) else None
        ws = _workspace(L.glif_scan_fwd_workspace(byref(s)), dev)
        with _on(dev):
            check(L.glif_scan_fwd(byref(s), _p(y), _p(last), _p(keep), _p(ws), _size(ws), _stream(dev)))
        ctx.save_for_backward(u, delta, A, B_, C_, D, z, bias, state, lengths, keep)
        ctx.softplus = softplus
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        _first_only("state_space_scan")
        u, delta, A, B_, C_, D, z, bias, state, lengths, keep = ctx.saved_tensors
        (T, B, Dc), dev = u.shape, u.device
        held = [_seq(u), _seq(delta), _dense(A), _seq(B_), _seq(C_), _dense(D), _seq(z), _dense(bias), _dense(state), lengths]
        s = _scan_struct(*held, ctx.softplus, True)
        dy = _seq(dy) if dy is not None else torch.zeros((T, B, Dc), dtype=u.dtype, device=dev)
        dlast = _dense(dlast)
        like = (u, delta, A, B_, C_, D, z, bias, state)
        outs = [torch.empty(t.shape, dtype=t.dtype, device=dev) if w else None for t, w in zip(like, ctx.needs_input_grad)]
        g = _lib.ScanGrad()
        g.dy, g.dy_st, g.dy_sb = dy.data_ptr(), dy.stride(0), dy.stride(1)
        g.dlast = dlast.data_ptr() if dlast is not None else None
        g.du, g.ddelta, g.dA, g.dB, g.dC, g.dD, g.dz, g.ddelta_bias, g.dstate = (
            t.data_ptr() if t is not None else None for t in outs)
        L = lib()
        ws = _workspace(L.glif_scan_bwd_workspace(byref(s)), dev)
        with _on(dev):
            check(L.glif_scan_bwd(byref(s), byref(g), _p(keep), _p(ws), _size(ws), _stream(dev)))
        return (*outs, None, None)


def _scan_args(u, delta, A, B_, C_, D, z, bias):
    _activations(u, "u")
    lead, Dc = tuple(u.shape[:-1]), u.shape[-1]
    _need(delta, "delta", u.shape, u.dtype, u.device)
    _need(A, "A", (Dc, None), torch.float32, u.device)
    N = A.shape[1]
    if Dc < 1 or not 1 <= N <= 64:
        raise ValueError(f"A must have at least one channel and 1 to 64 states, got {tuple(A.shape)}")
    _need(B_, "B", (*lead, None, N), u.dtype, u.device)
    G = B_.shape[-2]
    if G < 1 or Dc % G:
        raise ValueError(f"the groups of B ({G}) must divide the channels ({Dc})")
    _need(C_, "C", (*lead, G, N), u.dtype, u.device)
    if D is not None:
        _need(D, "D", (Dc,), torch.float32, u.device)
    if z is not None:
        _need(z, "z", u.shape, u.dtype, u.device)
    if bias is not None:
        _need(bias, "delta_bias", (Dc,), torch.float32, u.device)
    return N


def state_space_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus: bool = True, initial_state=None,
                     lengths=None):
    """A diagonal state space whose step, input and output maps come with every tick:

    ``s = softplus(delta + delta_bias)``, ``h[t] = exp(s * A) * h[t - 1] + s * B[t] * u[t]``,
    ``y[t] = ((C[t] * h[t]).sum(-1) + D * u[t]) * silu(z[t])``

    u, delta, z [T, B, D]; B, C [T, B, G, N] (N <= 64; a group's D / G channels share them); A [D, N], D and delta_bias [D]
    and initial_state [B, D, N] float32.  Returns y and the state [B, D, N] after each batch entry's last tick."""
    if torch.is_tensor(u) and u.dim() != 3:
        raise ValueError(f"u must be [T, B, D], got shape {tuple(u.shape)}")
    N = _scan_args(u, delta, A, B, C, D, z, delta_bias)
    if initial_state is not None:
        _need(initial_state, "initial_state", (u.shape[1], u.shape[2], N), torch.float32, u.device)
    lengths = _lengths(lengths, u, u.shape[1])
    return _apply(_Scan, _wants_grad(u, delta, A, B, C, D, z, delta_bias, initial_state), u, delta, A, B, C, D, z, delta_bias,
                  initial_state, lengths, int(bool(delta_softplus)))


def state_space_step(u, state, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus: bool = True) -> torch.Tensor:
    """One tick of ``state_space_scan``: u, delta, z [B, D], B and C [B, G, N]; ``state`` [B, D, N] is moved on in place.
    No gradient."""
    if torch.is_tensor(u) and u.dim() != 2:
        raise ValueError(f"u must be [B, D], got shape {tuple(u.shape)}")
    N = _scan_args(u, delta, A, B, C, D, z, delta_bias)
    _need(state, "state", (u.shape[0], u.shape[1], N), torch.float32, u.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is written in place")
    _refuse_grad("state_space_step", u, state, delta, A, B, C, D, z, delta_bias)
    held = [_tick(u), _tick(delta), _dense(A), _tick(B), _tick(C), _dense(D), _tick(z), _dense(delta_bias), None, None]
    s = _scan_struct(*held, int(bool(delta_softplus)), False)
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    with _on(u.device):
        check(lib().glif_scan_step(byref(s), _p(y), _p(state), _stream(u.device)))
    torch.autograd.graph.increment_version(state)
    return y


def _tick(t):
    """t [B, ...] with everything behind the batch contiguous."""
    if t is None or t.is_contiguous():
        return t
    return t if t[:1].is_contiguous() else t.contiguous()


# ------------------------------------------------------------------- linear attention ----
def _heads(t):
    """t [..., heads, channels] with the channels contiguous, and ticks less than 2^24 elements apart."""
    if t.is_contiguous() or ((t.shape[-1] == 1 or t.stride(-1) == 1) and (t.dim() < 4 or t.shape[0] == 1 or t.stride(0) < 1 << 24)):
        return t
    return t.contiguous()


def _head_strides(t):
    """The strides of ticks (0 where there is but one: it may be anything then), batch entries and heads."""
    st, sb, sh, _ = t.stride()
    return (st if t.shape[0] > 1 else 0), sb, sh


def _attention_struct(q, k, v, log_decay, state, lengths, scale, dims):
    """glif_attention of tensors with contiguous channels (held by the caller) and ``dims`` ticks, entries, heads, groups and
    channels."""
    return _lib.Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _p(state), _p(lengths), *_head_strides(q),
                          *_head_strides(k), *_head_strides(v), scale, DTYPES[q.dtype], *dims)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        (T, B, H, K), (G, V), dev = q.shape, v.shape[2:], q.device
        held = (_heads(q), _heads(k), _heads(v), _dense(log_decay), _dense(state), lengths)
        s = _attention_struct(*held, scale, (T, B, H, G, K, V))
        y = q.new_empty((T, B, H, V))
        last = torch.empty((B, H, K, V), dtype=torch.float32, device=dev)
        L = lib()
        ws = _workspace(L.glif_attention_fwd_workspace(byref(s)), dev)
        with _on(dev):
            check(L.glif_attention_fwd(byref(s), _p(y), _p(last), _p(ws), _size(ws), _stream(dev)))
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        _first_only("linear_attention")
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        (T, B, H, K), (G, V), dev = q.shape, v.shape[2:], q.device
        held = (_heads(q), _heads(k), _heads(v), _dense(log_decay), _dense(state), lengths)
        s = _attention_struct(*held, ctx.scale, (T, B, H, G, K, V))
        dy = _heads(dy) if dy is not None else torch.zeros((T, B, H, V), dtype=q.dtype, device=dev)
        dlast = _dense(dlast)
        wq, wk, wv, _, ws_, _, _ = ctx.needs_input_grad
        dense = torch.contiguous_format
        dq = torch.empty_like(q, memory_format=dense) if wq else None
        dk = torch.empty_like(k, memory_format=dense) if wk else None
        dv = torch.empty_like(v, memory_format=dense) if wv else None
        dstate = torch.empty_like(state, memory_format=dense) if ws_ else None
        g = _lib.AttentionGrad(_p(dy), *_head_strides(dy), _p(dlast), _p(dq), _p(dk), _p(dv), _p(dstate))
        L = lib()
        ws = _workspace(L.glif_attention_bwd_workspace(byref(s)), dev)
        with _on(dev):
            check(L.glif_attention_bwd(byref(s), byref(g), _p(ws), _size(ws), _stream(dev)))
        return dq, dk, dv, None, dstate, None, None


def _attention_args(q, k, v, log_decay, scale):
    _activations(q, "q")
    lead, (H, K) = tuple(q.shape[:-2]), q.shape[-2:]
    _need(k, "k", (*lead, None, K), q.dtype, q.device)
    G = k.shape[-2]
    _need(v, "v", (*lead, G, None), q.dtype, q.device)
    V = v.shape[-1]
    if not 1 <= K <= 128 or not 1 <= V <= 128:
        raise ValueError(f"q, k and v must have 1 to 128 channels a head, got {K} and {V}")
    if G < 1 or H < 1 or H % G:
        raise ValueError(f"the heads of k and v ({G}) must divide those of q ({H})")
    _need(log_decay, "log_decay", (H,), torch.float32, q.device)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay has no gradient: each head's decay is a constant")
    return float(K ** -0.5 if scale is None else scale)


def linear_attention(q, k, v, log_decay, scale=None, initial_state=None, lengths=None):
    """Attention without a softmax, whose heads forget each at its own rate:

    ``S[t] = exp(log_decay) * S[t - 1] + k[t][:, None] * v[t]``, ``y[t] = scale * q[t] @ S[t]``

    q [T, B, H, K], k [T, B, G, K], v [T, B, G, V] (K and V at most 128; H / G heads share a k and a v); log_decay [H]
    float32, at most 0, -inf for a head that sees only its own tick, a constant without a gradient; ``scale`` K^-0.5 if None;
    initial_state [B, H, K, V] float32 or None.  Returns y [T, B, H, V] and the state [B, H, K, V] after each batch entry's
    last tick.  At most 4096 heads, B H 2^20, and B H V and B H K below 2^24 where there is more than one tick.

    Ticks are taken in chunks, as matrix products.  Those of bfloat16 sequences multiply scores and states as two bfloat16
    values each, 16 bits together (their sums, and the states themselves, are float32); those of float16 ones are float32, as
    states and scores go beyond float16's range.  An infinite value or state makes its channel infinite from there on, or NaN where
    the definition does; what an infinite key makes infinite of the state, or an infinite query of its tick's answer, may be NaN
    instead; likewise in the gradients."""
    if torch.is_tensor(q) and q.dim() != 4:
        raise ValueError(f"q must be [T, B, H, K], got shape {tuple(q.shape)}")
    scale = _attention_args(q, k, v, log_decay, scale)
    if initial_state is not None:
        _need(initial_state, "initial_state", (*q.shape[1:], v.shape[-1]), torch.float32, q.device)
    lengths = _lengths(lengths, q, q.shape[1])
    return _apply(_Attention, _wants_grad(q, k, v, log_decay, initial_state), q, k, v, log_decay, initial_state, lengths, scale)


def linear_attention_step(q, k, v, state, log_decay, scale=None) -> torch.Tensor:
    """One tick of ``linear_attention``: q [B, H, K], k [B, G, K], v [B, G, V]; ``state`` [B, H, K, V] is moved on in place.
    No gradient."""
    if torch.is_tensor(q) and q.dim() != 3:
        raise ValueError(f"q must be [B, H, K], got shape {tuple(q.shape)}")
    scale = _attention_args(q, k, v, log_decay, scale)
    _need(state, "state", (*q.shape, v.shape[-1]), torch.float32, q.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is written in place")
    _refuse_grad("linear_attention_step", q, state, k, v, log_decay)
    q, k, v, log_decay = _heads(q), _heads(k), _heads(v), _dense(log_decay)
    (B, H, K), (G, V) = q.shape, v.shape[1:]
    (q_sb, q_sh, _), (k_sb, k_sh, _), (v_sb, v_sh, _) = q.stride(), k.stride(), v.stride()
    s = _lib.Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), None, None, 0, q_sb, q_sh, 0, k_sb, k_sh, 0,
                       v_sb, v_sh, scale, DTYPES[q.dtype], 1, B, H, G, K, V)
    y = q.new_empty((B, H, V))
    with _on(q.device):
        check(lib().glif_attention_step(byref(s), _p(y), _p(state), _stream(q.device)))
    torch.autograd.graph.increment_version(state)
    return y
