"""GPU tests of what is small in AdamW's steps: decays that are less than a variable's last digit, and moments in 8 bits that move by
less than their codes are apart."""
import numpy as np
import pytest
import torch

from tests import adamw_ref as ref
from tests.test_gpu_adamw import B1, B2, DEV, EPS, U, host, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lr", [2e-6, 1e-5, 1e-4])
def test_a_small_decay_is_not_lost(lr, bits):
    """Variables from 1/2 to 1 are 2^-24 apart, a decay is 2e-8 to 1e-6 of them: each lands on the neighbour that is nearest, but for the
    update's own 24 roundings (of what the step takes off it, not of the variable) and three of the decay's."""
    from v1_glif_model_amd.optim import AdamW
    n = 65536
    p = rnd(1, (n,)).abs().remainder(0.5) + 0.5
    opt = AdamW([p], 0.0, B1, B2, EPS, 0.01, state_bits=bits)
    opt.apply_gradients([rnd(2, (n,))])           # moments of many sizes
    before, (m, v), g = host(p), opt.moments(), rnd(3, (n,))
    m, v, opt.learning_rate = host(m[0]), host(v[0]), lr
    opt.apply_gradients([g])
    want, _, _, _, update = ref.step(before, host(g), m, v, 2, lr, B1, B2, EPS, 0.01)
    half = np.spacing(want.astype(np.float32)).astype(np.float64) / 2
    assert (np.abs(host(p) - want) <= half + U * (24 * update + 3 * lr * 0.01 * before)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_variables_stay(dtype):
    from v1_glif_model_amd.optim import AdamW
    for decay in (0.0, 0.01):
        p = torch.tensor([float("inf"), float("-inf"), 1.0, 3e38, float("nan")], device=DEV).to(dtype)
        AdamW([p], 1e-3, weight_decay=decay).apply_gradients([torch.ones(5, device=DEV)])
        assert p[0] == float("inf") and p[1] == float("-inf") and p[2:4].isfinite().all() and p[4].isnan()


STEPS, KEEP = 300, 0.999


def held_state(n):
    """Blocks whose first element has the scale, 1, and gradients that keep it there; the others' codes are 30 to 60 and their
    gradients 0."""
    g = np.random.default_rng(5)
    codes = [g.integers(30, 61, n) * g.choice([-1, 1], n), g.integers(30, 61, n)]
    for c, top in zip(codes, (127, 255)):
        c[::256] = top
    grad = np.zeros(n, np.float32)
    grad[::256] = 1.0
    return [c.astype(t) for c, t in zip(codes, (np.int8, np.uint8))], grad


def left_of(values, at_first):
    """The share that is left of moments in the mean of their magnitudes, without the elements that hold the scales."""
    rest = np.arange(values.size) % 256 != 0
    return np.abs(values[rest]).mean() / np.abs(at_first[rest]).mean() / KEEP ** STEPS


def test_moments_that_move_by_less_than_a_code():
    """They lose 0.1 % a step where codes are 3 to 14 % apart: 300 steps of 65,280 moments.  One rounding is off by at
    most half the way between two codes (standard deviation), which are 2 (60 / 127) / 127 or 4 (60 / 255)^3 / 255 of the scale apart: the
    mean of all, by sqrt(300 / 65,280) of that.  Six deviations allowed; roundings to the nearest, up and down are all
    outside."""
    from v1_glif_model_amd.optim import AdamW
    n = 65536
    codes, grad = held_state(n)
    p = torch.zeros(n, device=DEV)
    opt = AdamW([p], 0.0, KEEP, KEEP, state_bits=8, seed=11)
    ones = torch.ones(n // 256, device=DEV)
    opt.load_state_dict(dict(iterations=10, first=[(torch.from_numpy(codes[0]).to(DEV), ones)],
                             second=[(torch.from_numpy(codes[1]).to(DEV), ones)]))
    g = torch.from_numpy(grad).to(DEV)
    start = [host(x[0]) for x in opt.moments()]
    for _ in range(STEPS):
        opt.apply_gradients([g])
    end = [host(x[0]) for x in opt.moments()]
    F = np.float32
    for k, (top, step) in enumerate(((127, 2 * 60 / 127 / 127), (255, 4 * (60 / 255) ** 3 / 255))):
        assert end[k][::256] == pytest.approx(1.0, abs=1e-4)
        allowed = 6 * step / 2 * np.sqrt(STEPS / (n - n // 256)) / (np.abs(start[k]).reshape(-1, 256)[:, 1:].mean() * KEEP ** STEPS)
        assert abs(left_of(end[k], start[k]) - 1.0) <= allowed, (top, left_of(end[k], start[k]), allowed)
        for u in (0, 32768, 65535):          # up, to the nearest, down: two blocks are enough
            code, scale = codes[k][:512], np.ones(2, F)
            for _ in range(STEPS):
                x = ref.decode(code, scale, top) * F(KEEP) + (grad[:512] if top == 127 else grad[:512] ** 2) * F(1 - KEEP)
                code, scale = ref.encode(x, top, np.full(512, u))
            assert abs(left_of(ref.decode(code, scale, top), start[k][:512]) - 1.0) > 2 * allowed, (top, u)
