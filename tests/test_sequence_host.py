"""The sequence operators' host logic that needs no GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from v1_glif_model_amd import sequence as seq


def test_forward_mode_derivatives_are_seen():
    """A dual tensor requires no gradient, but a call on it must not go past autograd, whether gradients are on or not."""
    x, plain = torch.randn(3, 4), torch.randn(3, 4)
    assert not seq._wants_grad(x, None, plain)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not dual.requires_grad
        assert seq._wants_grad(None, plain, dual) and not seq._wants_grad(plain, None)
        with torch.no_grad():
            assert seq._wants_grad(dual)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            seq._refuse_grad("step", plain, dual)
        seq._refuse_grad("step", plain, None)
    with pytest.raises(ValueError, match="no gradient"):
        seq._refuse_grad("step", plain.requires_grad_(True))
