"""AdamW in numpy: in 64 bits, and its 8-bit moments operation by operation in float32."""
import numpy as np

from oracle.sample_ref import words  # noqa: F401  words(n, seed, offset)

F = np.float32
BLOCK = 256


def step(p, g, m, v, t, lr, b1, b2, eps, decay):
    """One step in 64 bits; also how large the terms of m and v are, and the update's absolute terms."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    sm, sv = np.abs(b1 * m) + np.abs((1 - b1) * g), b2 * v + (1 - b2) * g * g
    m = b1 * m + (1 - b1) * g
    root = np.sqrt(sv) / np.sqrt(1 - b2 ** t) + eps
    size = lr / (1 - b1 ** t)
    return p * (1 - lr * decay) - size * m / root, m, sv, sm, size * sm / root


def level(code, top):
    r = (code.astype(F) * F(1.0 / top)).astype(F)
    return r * np.abs(r) if top == 127 else (r * r) * (r * r)


def decode(code, scale, top):
    return level(code, top) * np.repeat(scale, BLOCK)[:code.size].reshape(code.shape)


def encode(x, top, u):
    """x (float32, flat) to codes and scales with the random numbers u (16 bits)."""
    n = x.size
    x = np.pad(x.astype(F).ravel(), (0, -n % BLOCK)).reshape(-1, BLOCK)
    u = np.pad(u[:n], (0, -n % BLOCK)).reshape(-1, BLOCK).astype(F)
    most = np.abs(x).max(1)
    fine = np.isfinite(most) & (most >= np.finfo(F).tiny)
    with np.errstate(all="ignore"):
        part = np.abs(x) * (F(1) / most)[:, None]
        root = np.sqrt(part) if top == 127 else np.sqrt(np.sqrt(part))
        below = np.minimum(np.floor(root * F(top)), F(top - 1))
        a, b = level(below, top), level(below + F(1), top)
        code = below + (u * (b - a) < (part - a) * F(65536))
        if top == 255:
            code = np.where(x > 0, np.maximum(code, 1), code)
        else:
            code = code * np.sign(x)
    code = np.where(fine[:, None], code, 0)
    return code.reshape(-1)[:n].astype(np.int8 if top == 127 else np.uint8), most

