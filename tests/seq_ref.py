"""The sequence operators' definitions in 64 bits, one tick at a time, for tests (autograd gives the formulas' gradients),
and how far a result may be from them.

A result of type T is its sum in float32, rounded once: |out - ref| <= u_T |ref| + 1e-5 S, where u_T is T's unit roundoff
(2^-24, 2^-8 and 2^-11) and S the sum of the absolute values of the terms."""
import math

import torch

F64 = torch.float64
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -24}


def act(p, name):
    if name == "relu":
        return torch.relu(p)
    if name == "gelu":
        return p * 0.5 * torch.erfc(-p / math.sqrt(2.0))
    if name == "silu":
        return p / (1.0 + torch.exp(-p))
    return p


def layer_norm(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    xh = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    return xh * (1.0 if w is None else w) + (0.0 if b is None else b)


def linear(x, w, b, name, residual):
    y = act(x @ w.t() + (0.0 if b is None else b), name)
    return y if residual is None else y + residual


def short_conv(x, w, b, name, state, lengths):
    """y and the last state; ticks from a length on are not looked at."""
    (T, B, D), W = x.shape, w.shape[1]
    mem = torch.zeros(B, W - 1, D, dtype=x.dtype) if state is None else state
    ys, lasts = [], []
    for i in range(B):
        n = T if lengths is None else int(lengths[i].clamp(0, T))
        m, col = mem[i], []
        for t in range(n):
            taps = torch.cat([m, x[t, i][None]])
            col.append(act((taps * w.t()).sum(0) + (0.0 if b is None else b), name))
            m = taps[1:]
        col += [torch.zeros(D, dtype=x.dtype)] * (T - n)
        ys.append(torch.stack(col) if T else torch.zeros(0, D, dtype=x.dtype))
        lasts.append(m)
    return torch.stack(ys, 1), torch.stack(lasts)


def scan(u, delta, A, B, C, D=None, z=None, bias=None, softplus=True, state=None, lengths=None, sums=False):
    """y and the last state.  sums: of non-negative inputs (A and the gates apart), with derivatives that are taken as
    non-negative too, so that autograd gives the sums of the gradients' absolute terms."""
    (T, Bn, Dn), N, G = u.shape, A.shape[1], B.shape[2]
    h0 = torch.zeros(Bn, Dn, N, dtype=u.dtype) if state is None else state
    ys, lasts = [], []
    for i in range(Bn):
        n = T if lengths is None else int(lengths[i].clamp(0, T))
        h, col = h0[i], []
        for t in range(n):
            s = delta[t, i] + (0.0 if bias is None else bias)
            if softplus:
                s = torch.logaddexp(s, torch.zeros_like(s))
            Bt, Ct = (v[t, i].repeat_interleave(Dn // G, 0) for v in (B, C))
            decay = torch.exp(s[:, None] * A)
            if sums:
                sd, Ad = s.detach()[:, None], A.detach()
                decay = decay.detach() * (1.0 + (s[:, None] - sd) * Ad.abs() + sd.abs() * (A - Ad))
            h = decay * h + (s * u[t, i])[:, None] * Bt
            y = (h * Ct).sum(-1) + (0.0 if D is None else D * u[t, i])
            if z is not None:
                gate = act(z[t, i], "silu")
                if sums:
                    zd = z[t, i].detach()
                    q = torch.sigmoid(zd)
                    gate = gate.detach().abs() + q * (1.0 + zd.abs() * (1.0 - q)) * (z[t, i] - zd)
                y = y * gate
            col.append(y)
        col += [torch.zeros(Dn, dtype=u.dtype)] * (T - n)
        ys.append(torch.stack(col) if T else torch.zeros(0, Dn, dtype=u.dtype))
        lasts.append(h)
    return torch.stack(ys, 1), torch.stack(lasts)


def slope(p, name):
    with torch.enable_grad():
        q = p.detach().requires_grad_(True)
        return torch.autograd.grad(act(q, name).sum(), q)[0] if name else torch.ones_like(p)


def f64(t, grad=True):
    """t's values on the host in 64 bits, as a leaf."""
    if t is None:
        return None
    t = t.detach().cpu()
    return t.to(F64).requires_grad_(grad) if t.is_floating_point() else t


def near(out, ref, terms, what, more=0.0):
    """out within its type's bound of ref; terms: S (a tensor like ref, or a number); more: an allowance of its own."""
    assert tuple(out.shape) == tuple(ref.shape), (what, tuple(out.shape), tuple(ref.shape))
    o, r = out.detach().cpu().to(F64), ref.detach()
    bound = UNIT[out.dtype] * r.abs() + 1e-5 * terms + more + TINY[out.dtype]
    over = ((o - r).abs() - bound)
    bad = ~(over <= 0)
    assert not bool(bad.any()), (what, int(bad.sum()), float((o - r).abs().max()), float(over.max()))
