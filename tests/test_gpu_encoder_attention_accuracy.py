"""Attention against its definition in 64 bits where its own arithmetic is the question: caps of every size, fp16 weights
far below a row's largest, operands that are not finite.

Tolerance per element, in terms of the row: p_j its weights, a = sum_j p_j |v_j|, e the largest sum_d |q_d k_d| * scale, n its keys, u half a step of the type
(bf16 2^-8, fp16 2^-11).
  result                      u |o|  (fp16 below 2^-14: 2^-25)
  weights as operands         u a  (bf16 has the exponents of fp32; of an fp16 weight at most 2^-36 of the row's sum is lost: 2^-36 sum_j |v_j|)
  scores, off by d each       2 d a: the numerators are off by at most d relative, and so is their sum
    the dot product           d = (dim + 16) 2^-23 e
    the cap                   d = 2^-20 |s| (a relative error of the capped score) or, up to caps of 100, 2^-21 cap at most: 100 * 2^-21 = 2^-14.3
  sums and exponentials       (n + 64) 2^-23 a"""
import math

import math

import pytest
import torch

from tests.test_gpu_encoder_attention import DT, ea, gen, make  # noqa: F401  (ea: the fixture)
from tests.test_gpu_encoder_attention import oracle as ranges_oracle

pytestmark = pytest.mark.gpu


def oracle(q, k, v, lo=None, hi=None, scale=None, softcap=0.0):
    """-> (result, tolerance); one range of keys for all rows."""
    batch, rows, heads, dim = q.shape
    kv = k.shape[2]
    k, v = k[:, lo:hi], v[:, lo:hi]
    scale = dim**-0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(batch, rows, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(batch):
        for h in range(heads):
            qq, kk, vv = q[b, :, h].double(), k[b, :, h // (heads // kv)].double(), v[b, :, h // (heads // kv)].double()
            s = (qq @ kk.t().contiguous()) * scale
            d = (dim + 16) * 2.0**-23 * ((qq.abs() @ kk.abs().t().contiguous()) * scale).amax(-1, keepdim=True)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                d = d + torch.clamp(2.0**-20 * s.abs().amax(-1, keepdim=True), min=2.0**-21 * softcap if softcap <= 100 else 0.0)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o, a = p @ vv, p @ vv.abs()
            out[b, :, h] = o
            tol[b, :, h] = u * o.abs() + u * a + (2 * d + (vv.shape[0] + 64) * 2.0**-23) * a + ((2.0**-25 + 2.0**-36 * vv.abs().sum(0)) if q.dtype == torch.float16 else 0.0)
    return out, tol


def check(got, want, tol, what):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"{what}: {float(off.max()):.3e} off, {float((off - tol).max()):.3e} more than allowed"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [0.5, 5.0, 30.0, 50.0, 100.0, 101.0, 1e3, 1e4, 1e6, 1e9, 1e20, 1e30, 2e38])
def test_caps_of_every_size(ea, dtype, cap):  # noqa: F811
    """A cap far above the scores leaves them as they are, whatever its size; scores around and above it are bent."""
    g = gen(40)
    for dim, rows, keys, heads, kv, spread in ((64, 33, 1000, 2, 1, 2.0), (128, 3, 700, 8, 2, 1.0), (256, 20, 90, 4, 2, 2.0), (72, 40, 200, 2, 2, 2.0), (32, 2, 4000, 2, 1, 3.0)):
        q = make(g, 1, rows, heads, dim, DT[dtype], "split", spread)
        k, v = make(g, 1, keys, kv, dim, DT[dtype], "split"), make(g, 1, keys, kv, dim, DT[dtype], "split")
        check(ea.attention(q, k, v, softcap=cap), *oracle(q, k, v, softcap=cap), what=(dim, "scores of a few"))
        if cap <= 1e4:  # scores a few times 0.05 times the factor: from far below to far above half the cap
            for factor in (20.0, cap):
                args = dict(softcap=cap, scale=factor / dim**0.5)
                check(ea.attention(q * 0.05, k, v, **args), *oracle(q * 0.05, k, v, **args), what=(dim, factor))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,keys", [(1, 300), (40, 8464), (300, 8464), (1, 20001), (2, 131072)])
def test_thousands_of_weak_keys_beside_a_strong_one(ea, dtype, rows, keys):  # noqa: F811
    """One key (first, in the middle or last) takes nearly all of the softmax and holds zeros, the others, 5 ... 22 below it, hold ones and twos: the result is
    their share, in one piece and cut along the keys."""
    dim = 64
    for at in (0, keys // 2, keys - 1):
        for gap in (5.0, 12.0, 17.0, 17.5, 18.0, 20.0, 22.0):
            q = torch.zeros(1, rows, 2, dim, device="cuda")
            k = torch.zeros(1, keys, 1, dim, device="cuda")
            v = torch.ones(1, keys, 1, dim, device="cuda")
            q[..., 0], q[:, :, 1, 1] = 8.0, 1.0
            k[:, at, :, 0] = gap  # 8 * gap / sqrt(64)
            k[:, :, 0, 1] = torch.linspace(-2, 2, keys, device="cuda")
            v[..., 1::2], v[:, at] = 2.0, 0.0
            q, k, v = (t.to(DT[dtype]) for t in (q, k, v))
            check(ea.attention(q, k, v), *oracle(q, k, v), what=(at, gap))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [40, 72, 80, 128, 256])
@pytest.mark.parametrize("rows,keys", [(70, 200), (3, 2500), (600, 600)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_and_no_others(ea, dtype, dim, rows, keys):  # noqa: F811
    """Infinite and NaN values at a few keys, rows with ranges of their own: where a row sees them, the columns that hold them are what the sum is (an infinity
    of one sign, else NaN) and the other columns stay; rows that do not see them stay altogether.  The keys' scores are near each other, so that no weight
    is rounded to 0."""
    g = gen(dim + keys)
    q, k, v = (make(g, 1, n, h, dim, DT[dtype], "heads", x) for n, h, x in ((rows, 4, 0.3), (keys, 2, 1.0), (keys, 2, 1.0)))
    lo = torch.randint(0, keys, (1, rows), generator=g, device="cuda")
    hi = torch.maximum(lo, torch.randint(0, keys + 1, (1, rows), generator=g, device="cuda"))
    r = torch.stack([lo, hi], -1).to(torch.int32)
    r[:, ::5] = torch.tensor([0, keys], dtype=torch.int32, device="cuda")
    want, tol = ranges_oracle(q, k, v, r)
    held = {keys // 3: (0, math.inf), keys // 3 + 1: (1, -math.inf), keys // 2: (dim - 1, math.nan), keys // 2 + 9: (0, -math.inf), keys - 2: (7, math.inf)}
    v2, seen = v.clone(), {}
    for at, (col, x) in held.items():
        v2[:, at, :, col] = x
        sees = (r[0, :, 0] <= at) & (at < r[0, :, 1])
        seen.setdefault(col, []).append((x, sees))
    got = ea.attention(q, k, v2, key_ranges=r)
    for col, marks in seen.items():
        total = sum(torch.where(s, x, 0.0) for x, s in marks)  # inf - inf and NaN come out as they do in the row's own sum
        odd = ~torch.isfinite(total)
        assert torch.equal(got[0, odd, :, col].float().nan_to_num(7.0, 8.0, 9.0), total[odd, None].expand(-1, 4).float().nan_to_num(7.0, 8.0, 9.0))
        got[0, odd, :, col], want[0, odd, :, col] = 0, 0
    check(got, want, tol, "the others")


@pytest.mark.parametrize("dim", [72, 80, 128, 256])
def test_a_value_that_is_not_finite_does_not_hold_up_the_call(ea, dim):  # noqa: F811
    """A page whose activations overflowed takes up to a few times as long (measured: 1.0 ... 4.5 times, 17 where the heads are narrower than the kernel and K is
    infinite in its first columns), not hundreds of times (161 ... 253 in the form that took every such row again key by key)."""
    g = gen(dim)
    rows = 2048
    q, k, v = (make(g, 1, rows, h, dim, torch.float16, "split") for h in (8, 8, 8))
    full = torch.full((1,), rows, dtype=torch.int32, device="cuda")
    causal = ea.padded_ranges(torch.zeros_like(full), full, rows, prefix=0)
    pages = ea.document_ranges(torch.tensor([0, 700, 1000, rows], dtype=torch.int32, device="cuda"), rows)

    def us(q, k, v, r):
        events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        for _ in range(2):
            events[0].record()
            out = ea.attention(q, k, v, key_ranges=r)
            events[1].record()
            events[1].synchronize()
        return events[0].elapsed_time(events[1]) * 1e3, out

    for name, r in (("all", None), ("causal", causal), ("pages", pages)):
        clean = min(us(q, k, v, r)[0] for _ in range(3))
        for what in ("q", "k", "v"):
            for x in (math.inf, math.nan):
                bad = [t.clone() for t in (q, k, v)]
                bad["qkv".index(what)][:, 900, :, 5] = x
                took, out = us(*bad, r)
                print(f"{dim} {name} {what} {x}: {took / clean:.2f} of {clean:.0f} us")
                assert not bool(torch.isfinite(out[:, 950]).all()) or what == "q"
                assert took <= (12 if dim != 72 else 40) * clean + 100, (name, what, x, took, clean)


def test_forward_mode_tangents_are_refused(ea):  # noqa: F811
    from torch.autograd import forward_ad

    g = gen(43)
    q, k, v = (make(g, 1, 4, 2, 16, torch.bfloat16, "split") for _ in range(3))
    table, pos = ea.RotaryTable.with_sections(16, [8]), torch.zeros(4, dtype=torch.int64, device="cuda")
    cos = torch.ones(1, 4, 8, device="cuda")
    with forward_ad.dual_level():
        for bad in range(3):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == bad else t for i, t in enumerate((q, k, v))]
            with pytest.raises(ValueError, match="tangent"):
                ea.attention(*args)
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(ValueError, match="tangent"):
            ea.rotary(q, dual, pos, table)
        with pytest.raises(ValueError, match="tangent"):
            ea.rotary_tables(q, k, cos, forward_ad.make_dual(cos, torch.ones_like(cos)))
        assert ea.attention(q, k, v).shape == q.shape and ea.rotary(q, k, pos, table)[0].shape == q.shape


def test_heads_of_one_buffer_outside_the_rows_turn_in_place(ea):  # noqa: F811
    """q and k as parts of one [batch, heads, rows, dim] buffer: the bits of a new tensor, the heads behind them as they were."""
    g = gen(44)
    whole = torch.randn(3, 8, 11, 64, generator=g, device="cuda").to(torch.bfloat16)
    keep = whole.clone()
    q, k = whole[:, :4].transpose(1, 2), whole[:, 4:6].transpose(1, 2)
    table, pos = ea.RotaryTable.with_sections(64, [32]), torch.arange(11, device="cuda")
    want = ea.rotary(q, k, pos, table)
    a, b = ea.rotary(q, k, pos, table, in_place=True)
    assert a is q and b is k and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(whole[:, 6:], keep[:, 6:])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [72, 128])
@pytest.mark.parametrize("rows,keys", [(3, 1), (40, 70), (4, 2501), (64, 128)])
def test_an_infinite_value_at_the_last_key_is_infinite(ea, dtype, dim, rows, keys):  # noqa: F811
    """The last key of a call that ends inside a tile: its column is infinite in the rows that see it, not NaN, and no row's other columns change."""
    g = gen(keys)
    q, k, v = (make(g, 1, n, 2, dim, DT[dtype], "split", x) for n, x in ((rows, 0.3), (keys, 1.0), (keys, 1.0)))
    r = torch.tensor([0, keys], dtype=torch.int32, device="cuda").repeat(1, rows, 1)
    r[:, 1::2, 1] -= 1  # every other row ends in front of it
    want, tol = ranges_oracle(q, k, v, r)
    for x in (math.inf, -math.inf):
        v2 = v.clone()
        v2[:, -1, :, 3] = x
        got = ea.attention(q, k, v2, key_ranges=r)
        assert bool((got[:, ::2, :, 3] == x).all())
        got[:, ::2, :, 3] = want[:, ::2, :, 3].to(got.dtype)
        check(got, want, tol + 2.0**-7 * want.abs(), x)
