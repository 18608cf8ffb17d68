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


def test_what_the_kernel_refuses_goes_the_frameworks_way():
    """Every shape, layout and scale that `attention` would raise for is no call of the attention function's."""

    def x(heads, rows, dim, dtype=torch.bfloat16, batch=2):
        return torch.zeros(batch, heads, rows, dim, dtype=dtype)

    q, k = x(4, 5, 32), x(2, 7, 32)
    assert ea._fits(torch, q, k, k) and ea._fits(torch, q, k, k, 0.3, 30.0) and ea._fits(torch, q.half(), k.half(), k.half())
    wide = torch.empty_strided((2, 2, 3, 32), (64, 32, (1 << 23) + 8, 1), dtype=torch.bfloat16, device="meta")
    far = torch.empty_strided((2, 2, 3, 32), (64, 32, 1 << 23, 1), dtype=torch.bfloat16, device="meta")
    on_meta = q.to("meta")
    assert ea._fits(torch, on_meta, far, far) and not ea._fits(torch, on_meta, wide, far) and not ea._fits(torch, on_meta, far, wide)
    odd = torch.zeros(2, 2, 7, 36, dtype=torch.bfloat16)[..., :32]
    for args in ((q, k, x(2, 7, 64)), (q, x(2, 7, 64), x(2, 7, 64)), (q, k, x(2, 6, 32)), (q, k, x(1, 7, 32)), (q, x(3, 7, 32), x(3, 7, 32)), (q, k[:1], k[:1]), (q, k.half(), k),
                 (q, k, k.float()), (q.float(), k.float(), k.float()), (q, odd, k), (q, k, odd), (x(4, 5, 20), x(2, 7, 20), x(2, 7, 20)), (x(4, 5, 264), x(2, 7, 264), x(2, 7, 264)),
                 (q, k.transpose(2, 3).contiguous().transpose(2, 3), k), (q, k[:, :0], k[:, :0])):
        assert not ea._fits(torch, *args), [tuple(t.shape) for t in args]
    for scaling, cap in ((0.0, 0.0), (-1.0, 0.0), (float("nan"), 0.0), (float("inf"), 0.0), (3e38, 0.0), (1.0, -1.0), (1.0, 3e38), (1.0, float("nan")), (1e-30, 1e30), (3e38, 1e-3)):
        assert not ea._fits(torch, q, k, k, scaling, cap), (scaling, cap)
