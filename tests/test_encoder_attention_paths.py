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


def test_a_softcap_is_kept_where_the_kernel_does_not_apply():
    """Off the GPU, and with a mask of holes: the capped formula in 64 bits, not the framework's uncapped function.  32-bit sums over 16 and 7 terms: 1e-5."""

    class Module(torch.nn.Module):
        num_key_value_groups = 2

    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, h, 7, 16, generator=g) * x for h, x in ((4, 6.0), (2, 2.0), (2, 1.0)))
    bits = torch.rand(2, 1, 7, 7, generator=g) < 0.6
    bits[:, :, 3] = False
    low = torch.where(bits, 0.0, torch.finfo(torch.float32).min)
    below = torch.ones(7, 7, dtype=torch.bool).tril()[None, None].expand(2, 1, 7, 7)
    r = torch.tensor([[[0, 4], [1, 3], [2, 2], [0, 7], [5, 7], [0, 1], [3, 7]]] * 2, dtype=torch.int32)
    at = torch.arange(7)
    runs = ((at >= r[..., :1]) & (at < r[..., 1:]))[:, None]
    for mask, seen, kw in ((None, below, {}), (None, torch.ones_like(below), dict(is_causal=False)), (bits, bits, {}), (low, bits, {}), (r[:, None], runs, {})):
        s = 5.0 * torch.tanh(q.double() @ k.double().repeat_interleave(2, 1).transpose(2, 3) * 0.25 / 5.0)
        s = s.masked_fill(~seen, -torch.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        want = (p @ v.double().repeat_interleave(2, 1)).transpose(1, 2)
        got = ea._interface_attention(Module(), q, k, v, mask, scaling=0.25, softcap=5.0, **kw)[0]
        if mask is low:  # every key of an all-masked row weighs the same there
            got, want = (t[:, [0, 1, 2, 4, 5, 6]] for t in (got, want))
        assert torch.allclose(got.double(), want, rtol=0, atol=1e-5)
    with pytest.raises(ValueError, match="softcap"):
        ea._interface_attention(Module(), q, k, v, None, softcap=5.0, position_bias=low)
    x = q.clone().requires_grad_()
    ea._interface_attention(Module(), x, k, v, bits, softcap=5.0)[0].sum().backward()
    assert bool(torch.isfinite(x.grad).all())
