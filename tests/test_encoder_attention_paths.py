"""The encoders' attention path off the GPU: what the guards of encoder_attention see, and what patched modules do where the kernels do not apply."""
import pytest
import torch
from torch.autograd import forward_ad

from morphik_core_amd import encoder_attention as ea


def test_tensors_that_autograd_follows_in_either_mode_are_refused():
    x = torch.zeros(3)
    whole = torch.zeros(3, dtype=torch.int32)
    ea._refuse_derivatives(torch, "op", (x, whole))
    with pytest.raises(ValueError, match="no gradient"):
        ea._refuse_derivatives(torch, "op", (whole, x.clone().requires_grad_()))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        ea._refuse_derivatives(torch, "op", (x, whole))
        with pytest.raises(ValueError, match="tangent"):
            ea._refuse_derivatives(torch, "op", (whole, dual))
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # which leaves the forward mode on
            ea._refuse_derivatives(torch, "op", (dual,))
        with torch.inference_mode():
            ea._refuse_derivatives(torch, "op", (dual,))
