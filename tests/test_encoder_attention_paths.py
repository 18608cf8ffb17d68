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


def test_parts_of_one_buffer_are_told_from_parts_that_overlap():
    """Against the places themselves: pairs of slices, in the order of a projection and with the heads outside the rows, of one batch entry and several, cut
    along any dimension.  Never apart where an element is in both; heads cut from a buffer apart, in either order of its dimensions."""
    import itertools
    import random

    def places(t):
        index = torch.zeros((), dtype=torch.int64)
        for st, n in zip(t.stride(), t.shape):
            index = index[..., None] + st * torch.arange(n)
        return set((index + t.storage_offset()).flatten().tolist())

    rng = random.Random(1)
    told = 0
    for batch, heads_outside in itertools.product((1, 3), (False, True)):
        rows, heads, dim = 5, 6, 4
        whole = torch.zeros(batch, heads, rows, dim).transpose(1, 2) if heads_outside else torch.zeros(batch, rows, heads, dim)
        q, k, v = whole.split([3, 1, 2], 2)
        for a, b in itertools.permutations((q, k, v), 2):
            assert not ea._share_memory(a, b)
        for _ in range(600):
            parts = []
            for _ in range(2):
                t = whole
                for d in range(4):
                    lo = rng.randrange(t.shape[d])
                    hi = rng.randrange(lo, t.shape[d]) + 1
                    t = t.narrow(d, lo, hi - lo) if rng.random() < 0.6 else t
                parts.append(t)
            meet = bool(places(parts[0]) & places(parts[1]))
            said = ea._share_memory(*parts)
            assert said or not meet
            assert said == ea._share_memory(*parts[::-1])
            told += not meet and not said
    assert told > 300
    flat = torch.zeros(400)
    for _ in range(2000):  # any two strided boxes of one buffer
        parts = [flat.as_strided([rng.randint(1, 3) for _ in range(4)], [rng.randint(0, 40) for _ in range(3)] + [1], rng.randint(0, 60)) for _ in range(2)]
        assert ea._share_memory(*parts) or not places(parts[0]) & places(parts[1])
    near = [flat.as_strided((2, 3, 1, 4), (24, 10, 4, 1), at) for at in (0, 5)]  # the second entry's first row starts 4 behind the first one's last
    assert places(near[0]) & places(near[1]) and ea._share_memory(*near)


def test_asking_for_fused_attention_without_a_gpu_says_so(caplog, monkeypatch):
    from morphik_core_amd.embedding import MI355XColpaliEmbeddingModel

    none = {"rotary": 0, "decoder": 0, "packed": 0}
    monkeypatch.delenv("MV_ENCODER_FUSED_ATTENTION", raising=False)
    assert MI355XColpaliEmbeddingModel(preset="tiny", device="cpu", seed=3, fused_attention=False).fused_attention == none and not caplog.records
    assert MI355XColpaliEmbeddingModel(preset="tiny", device="cpu", seed=3).fused_attention == none and not caplog.records
    assert MI355XColpaliEmbeddingModel(preset="tiny", device="cpu", seed=3, fused_attention=True).fused_attention == none
    assert [r.levelname for r in caplog.records if "fused_attention" in r.message] == ["WARNING"]
    caplog.clear()
    monkeypatch.setenv("MV_ENCODER_FUSED_ATTENTION", "1")  # a setting of the machine, not a request to this model
    assert MI355XColpaliEmbeddingModel(preset="tiny", device="cpu", seed=3).fused_attention == none and not caplog.records
