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
