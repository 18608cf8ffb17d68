"""The HIP rotary and attention operators against their formulas in 64 bits.

Tolerances of attention, per element, with u half a step of the type relative to the value (bf16 2^-8, fp16 2^-11), a = sum_j p_j |v_j| of the row and
column, e the largest sum_d |q_d k_d| * scale of the row: u |o| for the result's rounding, u a for the weights' (each is off by u at most), and for
32-bit arithmetic 2 (dim + 16) 2^-23 e a (scores; once in the numerator, once in the sum) + (keys + 64) 2^-23 a (sums, exponentials), doubled for a cap
(its tanh is 3 cap 2^-22 off at most: added to e).  fp16 results below 2^-14 are rounded to 2^-25: added too.
Rotation: u |result| for the result's rounding plus 2^-21 (|x| + |y|) for angles, cosines and two 32-bit products."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ea():
    from morphik_core_amd import encoder_attention

    assert torch.cuda.is_available()
    yield encoder_attention
    torch.cuda.empty_cache()  # the tests behind fill the card with their slabs


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(g, batch, rows, heads, dim, dtype, layout, spread=1.0):
    x = (torch.randn(batch, rows, heads, dim, generator=g, device="cuda") * spread).to(dtype)
    if layout == "heads":  # [batch, heads, rows, dim] in memory
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "fused":  # inside wider rows, with something on either side
        wide = torch.full((batch, rows, heads * dim + 24), 1e4, device="cuda").to(dtype)
        wide[..., 8 : 8 + heads * dim] = x.flatten(2)
        return wide[..., 8 : 8 + heads * dim].view(batch, rows, heads, dim)
    return x


def oracle(q, k, v, ranges=None, scale=None, softcap=0.0):
    """-> (result, tolerance) in 64 bits, from the definition, one head at a time; keys outside a row's range are not touched at all."""
    batch, rows, heads, dim = q.shape
    keys, kv = k.shape[1], k.shape[2]
    scale = dim**-0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(batch, rows, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if keys == 0 or rows == 0:
        return out, tol
    if ranges is None:
        lo = torch.zeros(batch, rows, dtype=torch.int64, device=q.device)
        hi = torch.full_like(lo, keys)
    else:
        r = ranges.long().expand(batch, rows, 2)
        lo, hi = r[..., 0].clamp(0, keys), r[..., 1].clamp(0, keys)
    j = torch.arange(keys, device=q.device)
    for b in range(batch):
        seen = (j >= lo[b, :, None]) & (j < hi[b, :, None])
        live = seen.any(-1)
        used = seen.any(0)[:, None]
        for h in range(heads):
            kk = torch.where(used, k[b, :, h // (heads // kv)].double(), 0.0)
            vv = torch.where(used, v[b, :, h // (heads // kv)].double(), 0.0)
            qq = q[b, :, h].double()
            s = (qq @ kk.t().contiguous()) * scale
            e = torch.where(seen, (qq.abs() @ kk.abs().t().contiguous()) * scale, 0.0).amax(-1, keepdim=True)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                e = 2 * e + 3 * softcap
            s = torch.where(seen, s, -math.inf)
            p = torch.where(seen, torch.exp(s - torch.where(live, s.amax(-1), 0.0)[:, None]), 0.0)
            p = p / torch.where(live, p.sum(-1), 1.0)[:, None]
            o, a = p @ vv, p @ vv.abs()
            out[b, :, h] = o
            n = seen.sum(-1, keepdim=True)
            tol[b, :, h] = u * o.abs() + u * a + (2 * (dim + 16) * e + n + 64) * 2.0**-23 * a + (2.0**-25 if q.dtype == torch.float16 else 0.0)
    return out, tol


def check(got, want, tol, what=""):
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), what
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0 if got.numel() else True, f"{what}: {float((got.double() - want).abs().max()):.3e} off, {float(over.max()):.3e} more than allowed"


def some_ranges(g, batch, rows, keys):
    """Random runs: empty ones, single keys, whole rows, ends beyond what there is."""
    a = torch.randint(-3, keys + 4, (batch, rows), generator=g, device="cuda")
    b = torch.randint(-3, keys + 4, (batch, rows), generator=g, device="cuda")
    kind = torch.randint(0, 8, (batch, rows), generator=g, device="cuda")
    lo, hi = torch.minimum(a, b), torch.maximum(a, b)
    hi = torch.where(kind == 0, lo, hi)  # empty
    hi = torch.where(kind == 1, lo + 1, hi)  # one key
    lo, hi = torch.where(kind == 2, 0, lo), torch.where(kind == 2, keys, hi)
    lo, hi = torch.where(kind == 3, hi, lo), torch.where(kind == 3, lo, hi)  # back to front: empty
    return torch.stack([lo, hi], -1).to(torch.int32)


# --------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 104, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_every_head_width_and_type(ea, dtype, dim, softcap):
    g = gen(dim)
    for rows, keys, heads, kv, layout in ((37, 37, 4, 2, "split"), (70, 201, 6, 1, "heads"), (1, 130, 3, 3, "fused"), (129, 1, 2, 2, "split")):
        q = make(g, 2, rows, heads, dim, DT[dtype], layout, 2.0)
        k, v = make(g, 2, keys, kv, dim, DT[dtype], layout), make(g, 2, keys, kv, dim, DT[dtype], layout)
        check(ea.attention(q, k, v, softcap=softcap), *oracle(q, k, v, softcap=softcap), what=(rows, keys, "all"))
        r = some_ranges(g, 2, rows, keys)
        check(ea.attention(q, k, v, key_ranges=r, softcap=softcap), *oracle(q, k, v, r, softcap=softcap), what=(rows, keys, "ranges"))


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 1030])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_sizes_around_the_tiles(ea, rows, group):
    g = gen(rows * 10 + group)
    for keys in (1, 31, 32, 33, 64, 65, 127, 128, 300):
        q, k, v = make(g, 1, rows, 2 * group, 32, DT["bf16"], "split"), make(g, 1, keys, 2, 32, DT["bf16"], "split"), make(g, 1, keys, 2, 32, DT["bf16"], "split")
        check(ea.attention(q, k, v), *oracle(q, k, v), what=keys)
        r = some_ranges(g, 1, rows, keys)
        check(ea.attention(q, k, v, key_ranges=r), *oracle(q, k, v, r), what=keys)


@pytest.mark.parametrize("rows,keys", [(1, 20000), (3, 4097), (16, 9001), (40, 2500)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_few_rows_over_many_keys(ea, rows, keys, dtype):
    g = gen(keys)
    for batch, heads, kv, dim in ((1, 1, 1, 64), (2, 16, 2, 128), (1, 8, 1, 256), (5, 4, 4, 72)):
        q, k, v = make(g, batch, rows, heads, dim, DT[dtype], "heads", 3.0), make(g, batch, keys, kv, dim, DT[dtype], "heads"), make(g, batch, keys, kv, dim, DT[dtype], "heads")
        check(ea.attention(q, k, v), *oracle(q, k, v))
        ends = torch.randint(0, keys + 1, (batch,), generator=g, device="cuda").to(torch.int32)
        ends[0] = keys
        r = ea.padded_ranges(torch.zeros_like(ends), ends, rows, prefix=0, row_offset=keys - rows)
        check(ea.attention(q, k, v, key_ranges=r, softcap=30.0), *oracle(q, k, v, r, softcap=30.0))
        r = some_ranges(g, batch, rows, keys)
        check(ea.attention(q, k, v, key_ranges=r), *oracle(q, k, v, r))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [16, 64, 80, 104, 128, 200, 256])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_small_and_large_blocks_of_every_width(ea, dtype, dim, softcap):
    """Short calls (rows spread over more, smaller blocks, with and without a cut along the keys), long keys, and more short problems than the card holds."""
    g = gen(dim + 1)
    for batch, rows, keys, heads, kv in ((1, 20, 500, 8, 1), (2, 130, 480, 2, 2), (2, 500, 500, 6, 1), (1, 300, 1100, 6, 2), (300, 70, 40, 2, 2)):
        q, k, v = (make(g, batch, n, h, dim, DT[dtype], "heads", x) for n, h, x in ((rows, heads, 2.0), (keys, kv, 1.0), (keys, kv, 1.0)))
        check(ea.attention(q, k, v, softcap=softcap), *oracle(q, k, v, softcap=softcap), what=(rows, keys, "all"))
        r = some_ranges(g, batch, rows, keys)
        check(ea.attention(q, k, v, key_ranges=r, softcap=softcap), *oracle(q, k, v, r, softcap=softcap), what=(rows, keys, "ranges"))
        last = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
        r = ea.padded_ranges(last // 5, last - 3, rows, prefix=0, row_offset=max(keys - rows, 0))
        check(ea.attention(q, k, v, key_ranges=r, softcap=softcap), *oracle(q, k, v, r, softcap=softcap), what=(rows, keys, "causal"))


@pytest.mark.parametrize("dim", [64, 80, 256])
def test_masks_of_the_encoders(ea, dim):
    """Causal, prefix and two-sided padding on either side; packed documents of one to many rows, some of none; one range row for a whole batch."""
    g = gen(7)
    batch, rows = 3, 333
    q, k, v = (make(g, batch, rows, h, dim, DT["bf16"], "heads") for h in (4, 2, 2))
    starts = torch.tensor([0, 100, 333], dtype=torch.int32, device="cuda")  # the last one holds nothing
    ends = torch.tensor([200, 333, 333], dtype=torch.int32, device="cuda")
    for prefix in (None, 0, 17, 1000, torch.tensor([5, 60, 1], dtype=torch.int32, device="cuda")):
        r = ea.padded_ranges(starts, ends, rows, prefix=prefix)
        got = ea.attention(q, k, v, key_ranges=r)
        check(got, *oracle(q, k, v, r), what=prefix)
        assert not bool(got[2].any()) and not bool(got[0, 200:].any()) and not bool(got[1, :100].any())
    lengths = [1, 64, 0, 63, 65, 1, 0, 130, 2]
    offsets = torch.tensor([3] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    for prefix in (None, 0, 30):
        r = ea.document_ranges(offsets, rows, prefix=prefix)
        got = ea.attention(q[0], k[0], v[0], key_ranges=r)
        want, tol = oracle(q[:1], k[:1], v[:1], r)
        check(got[None], want, tol)
        assert not bool(got[:3].any()) and not bool(got[329:].any())  # in front of the first, behind the last document
        check(ea.attention(q, k, v, key_ranges=r), *oracle(q, k, v, r))  # the same ranges for every batch entry


def test_ranges_say_what_the_definition_says(ea):
    starts, ends = [0, 2, 5, 9], [4, 9, 5, 40]
    prefixes = [2, 0, 3, -4]
    s, e, p = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, ends, prefixes))

    def row(start, end, at, prefix):
        if not start <= at < end:
            return [0, 0]
        return [start, end] if prefix is None else [start, max(at + 1, min(start + max(prefix, 0), end))]

    for offset in (0, 6):
        for prefix in (None, 0, 3, p):
            got = ea.padded_ranges(s, e, 11, prefix=prefix, row_offset=offset).tolist()
            pf = prefixes if prefix is p else [prefix] * 4
            assert got == [[row(starts[b], ends[b], i + offset, pf[b]) for i in range(11)] for b in range(4)]
    spans = torch.stack([s, e], 1)  # strided starts and ends
    assert torch.equal(ea.padded_ranges(spans[:, 0], spans[:, 1], 11), ea.padded_ranges(s, e, 11))
    offsets = [1, 1, 4, 4, 9, 10]
    o = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    p = torch.tensor([9, 2, 9, 3, 0], dtype=torch.int32, device="cuda")
    for prefix in (None, 0, 2, p):
        want = []
        for i in range(14):
            doc = [d for d in range(5) if offsets[d] <= i < offsets[d + 1]]
            want.append(row(offsets[doc[0]], offsets[doc[0] + 1], i, int(p[doc[0]]) if prefix is p else prefix) if doc else [0, 0])
        assert ea.document_ranges(o, 14, prefix=prefix).tolist() == [want]
    assert ea.document_ranges(o[:1], 3).tolist() == [[[0, 0]] * 3]
    assert ea.document_ranges(o, 0).shape == (1, 0, 2) and ea.padded_ranges(s[:0], e[:0], 5).shape == (0, 5, 2)
    m = torch.zeros(1, 6, 50, dtype=torch.bool, device="cuda")
    r = some_ranges(gen(3), 1, 6, 50)
    for i, (a, b) in enumerate(r[0].tolist()):
        m[0, i, max(a, 0) : max(b, 0)] = True
    got, ok = ea.ranges_from_mask(m)
    assert bool(ok)
    q, k, v = (make(gen(4), 1, n, 2, 16, DT["bf16"], "split") for n in (6, 50, 50))
    assert torch.equal(ea.attention(q, k, v, key_ranges=got), ea.attention(q, k, v, key_ranges=r))


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [40, 128, 256])
@pytest.mark.parametrize("rows,keys", [(90, 90), (4, 3000)])
def test_what_masked_keys_hold_reaches_no_row(ea, poison, dim, rows, keys):
    """NaN and infinities in keys and values that a row does not see -- though its neighbours in the tile do -- leave the row's result as it was."""
    g = gen(int(dim + rows))
    q, k, v = (make(g, 2, n, h, dim, DT["bf16"], "split") for n, h in ((rows, 4), (keys, 2), (keys, 2)))
    starts = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    ends = torch.tensor([keys - 5, keys], dtype=torch.int32, device="cuda")
    r = ea.padded_ranges(starts, ends, rows, prefix=0, row_offset=keys - rows)
    want, tol = oracle(q, k, v, r)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[0, keys - 5 :] = poison
        t[1, :10] = poison
    check(ea.attention(q, k2, v2, key_ranges=r), want, tol, "padding")
    # one poisoned key in the middle: rows that see it are not finite, the others keep their values
    at = keys - rows // 2
    v2 = v.clone()
    v2[:, at] = poison
    got = ea.attention(q, k, v2, key_ranges=r)
    sees = ((r[..., 0] <= at) & (at < r[..., 1]))[:, :, None, None].expand_as(got)
    assert not bool(torch.isfinite(got[sees]).any())
    check(torch.where(sees, 0, got), torch.where(sees, 0, want), tol, "neighbours")


def test_scores_of_extreme_size(ea):
    """Weights of one key only, scores far apart and all equal: the running maximum has to move and the sums to hold."""
    g = gen(5)
    q, k, v = (make(g, 1, n, 2, 64, DT["bf16"], "split") for n in (65, 700, 700))
    for factor in (0.0, 1e-3, 30.0, 300.0):
        check(ea.attention(q * factor, k, v), *oracle(q * factor, k, v), what=factor)
        check(ea.attention(q * factor, k, v, softcap=50.0), *oracle(q * factor, k, v, softcap=50.0), what=factor)
    order = (q[:, :1].float() * k.float()).sum(-1).argsort(1)  # rising scores: every tile moves the maximum
    k = torch.gather(k, 1, order[..., None].expand_as(k)).contiguous()
    check(ea.attention(q * 20, k, v), *oracle(q * 20, k, v))
    check(ea.attention(q, k, v, scale=3.0), *oracle(q, k, v, scale=3.0))


@pytest.mark.parametrize("rows,keys", [(3, 40), (40, 70), (1, 3000), (4, 3000)])
@pytest.mark.parametrize("dim", [40, 128])
def test_scores_of_minus_infinity(ea, dim, rows, keys):
    """Keys whose scores are -infinity weigh nothing; a row that sees no other key is 0 / 0 by the formula, whether or not it is cut along the keys; a row
    that sees no key at all is zero."""
    g = gen(dim + keys)
    q, k, v = (make(g, 1, n, h, dim, DT["bf16"], "split") for n, h in ((rows, 2), (keys, 1), (keys, 1)))
    q[..., 0] = 1.0
    half = keys // 2
    k[:, :half, :, 0] = -math.inf
    cut = torch.tensor([half, keys], dtype=torch.int32, device="cuda").expand(1, rows, 2).contiguous()
    check(ea.attention(q, k, v), *oracle(q, k, v, cut))
    ranges = torch.tensor([0, half], dtype=torch.int32, device="cuda").repeat(1, rows, 1)
    ranges[:, 0] = half
    got = ea.attention(q, k, v, key_ranges=ranges)
    assert not bool(got[:, 0].any()) and bool(got[:, 1:].isnan().all())
    k[:, :, :, 0] = -math.inf
    assert bool(ea.attention(q, k, v).isnan().all())


def test_sizes_of_nothing(ea):
    q, k, v = (make(gen(1), 2, 5, h, 16, DT["fp16"], "split") for h in (4, 2, 2))
    assert not bool(ea.attention(q, k[:, :0], v[:, :0]).any())
    assert ea.attention(q[:, :0], k, v).shape == (2, 0, 4, 16) and ea.attention(q[:0], k[:0], v[:0]).shape == (0, 5, 4, 16)
    assert ea.attention(q[0], k[0], v[0]).shape == (5, 4, 16)
    assert not bool(ea.attention(q, k, v, key_ranges=torch.zeros(1, 5, 2, dtype=torch.int32, device="cuda")).any())


def test_strides_of_one_entry_do_not_matter(ea):
    """A dimension of one entry may have any stride (slices of wider tensors have odd ones)."""
    g = gen(2)
    q, k, v = (make(g, 1, 9, 1, 16, DT["bf16"], "split") for _ in range(3))
    odd = torch.zeros(1, 9, 1, 16 * 9 + 3, dtype=torch.bfloat16, device="cuda")
    q2 = odd.as_strided((1, 9, 1, 16), (9 * 147 + 1, 16, 7, 1))
    q2.copy_(q)
    assert torch.equal(ea.attention(q2, k, v), ea.attention(q, k, v))


def test_one_key_has_no_step(ea):
    """Rows of k and v may be at most 2^23 elements apart, but one row is apart from nothing."""
    g = gen(6)
    q, k, v = (make(g, 1, n, 1, 16, DT["bf16"], "split") for n in (9, 1, 1))
    far = (1 << 25, 1 << 24, 16, 1)
    assert torch.equal(ea.attention(q, k.as_strided(k.shape, far), v.as_strided(v.shape, far)), v.expand(1, 9, 1, 16))


def test_offsets_past_32_bits(ea):
    """Rows, keys and values more than 2^31 elements into their tensors."""
    dim, keys = 256, (1 << 23) + 1000
    k = torch.zeros(1, keys, 1, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(9)
    tail = 300
    for t in (k, v):
        t[:, -tail:] = make(g, 1, tail, 1, dim, DT["bf16"], "split")
    q = make(g, 1, 4, 2, dim, DT["bf16"], "split")
    r = torch.tensor([[[keys - 300, keys - 1], [keys - 40, keys + 9], [keys - 1, keys], [keys, keys]]], dtype=torch.int32, device="cuda")
    want, tol = oracle(q, k[:, -tail:], v[:, -tail:], r - (keys - tail))
    check(ea.attention(q, k, v, key_ranges=r), want, tol)
    batch = k.view(2, keys // 2, 1, dim)  # the second entry starts past 2^30 elements, its end past 2^31
    wide = v.view(2, keys // 2, 1, dim)
    r2 = torch.tensor([[[0, 0]] * 4, (r[0] - keys // 2).clamp(0, keys // 2).tolist()], dtype=torch.int32, device="cuda")
    got = ea.attention(q.expand(2, -1, -1, -1), batch, wide, key_ranges=r2)
    check(got[1:], want, tol)
    # as many rows: a query tensor of more than 2^31 elements, of which the last rows are live
    r3 = torch.zeros(1, keys, 2, dtype=torch.int32, device="cuda")
    r3[0, -tail:] = torch.tensor([keys - tail, keys], dtype=torch.int32, device="cuda")
    got = ea.attention(k, k, v, key_ranges=r3)
    want, tol = oracle(k[:, -tail:], k[:, -tail:], v[:, -tail:])
    check(got[:, -tail:], want, tol)
    assert not bool(got[:, : keys - tail].any())


def test_the_same_bits_every_time_on_any_stream(ea):
    g = gen(11)
    cases = []
    for batch, rows, keys, heads, kv, dim in ((2, 300, 300, 8, 2, 128), (1, 1, 9000, 8, 1, 256), (3, 20, 20, 4, 4, 72)):
        q, k, v = (make(g, batch, n, h, dim, DT["bf16"], "split") for n, h in ((rows, heads), (keys, kv), (keys, kv)))
        cases.append((q, k, v, some_ranges(g, batch, rows, keys)))
    want = [ea.attention(q, k, v, key_ranges=r) for q, k, v, r in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([ea.attention(q, k, v, key_ranges=r) for q, k, v, r in cases])
    torch.cuda.synchronize()
    for one in got:
        for a, b in zip(one, want):
            assert torch.equal(a, b)


def test_two_captured_graphs_replay_side_by_side(ea):
    """Rotation and attention captured together, twice, with new inputs copied in and eager work between the replays."""
    g = gen(12)
    table = ea.RotaryTable.with_sections(128, [24, 20, 20], theta=1e6)
    graphs = []
    for rows, keys in ((65, 65), (1, 5000)):
        q = make(g, 1, rows, 8, 128, DT["bf16"], "split")
        k, v = make(g, 1, keys, 2, 128, DT["bf16"], "split"), make(g, 1, keys, 2, 128, DT["bf16"], "split")
        pos = torch.randint(0, 9999, (3, 1, rows), generator=g, device="cuda")
        ends = torch.full((1,), keys, dtype=torch.int32, device="cuda")

        def body(q=q, k=k, v=v, pos=pos, ends=ends, rows=rows, keys=keys):
            r = ea.padded_ranges(torch.zeros_like(ends), ends, rows, prefix=0, row_offset=keys - rows)
            return ea.attention(ea.rotary(q, None, pos, table)[0], k, v, key_ranges=r)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            body()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body()
        graphs.append((graph, body, out, q, k, v, ends, keys))
    for turn in range(4):
        wants = []
        for graph, body, out, q, k, v, ends, keys in graphs:
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            ends.fill_(keys - turn)
            wants.append(body())
        torch.cuda.synchronize()
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (graph, body, out, *_), want in zip(graphs, wants):
            assert torch.equal(out, want), turn


# --------------------------------------------------------------------------- rotation
def rotary_oracle(x, cos, sin, pairing, scale=1.0):
    """x [batch, rows, heads, dim], cos / sin [batch, rows, pairs] in 64 bits -> (result, tolerance)"""
    pairs = cos.shape[-1]
    w = x.double()
    i = torch.arange(pairs, device=x.device)
    a, b = (i, i + pairs) if pairing == "halves" else (2 * i, 2 * i + 1)
    c, s = cos[:, :, None] * scale, sin[:, :, None] * scale
    out, tol = w.clone(), torch.zeros_like(w)
    out[..., a] = w[..., a] * c - w[..., b] * s
    out[..., b] = w[..., b] * c + w[..., a] * s
    t = 2.0**-21 * scale * (w[..., a].abs() + w[..., b].abs())
    tol[..., a], tol[..., b] = t, t
    u = torch.finfo(x.dtype).eps / 2
    tol += u * out.abs() + (2.0**-25 if x.dtype == torch.float16 else 0.0)
    tol[..., 2 * pairs :] = 0
    return out, tol


def angles(positions, table):
    a = positions[table.axis.long()].permute(1, 2, 0).double() * table.inv_freq
    return a.cos(), a.sin()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dim,sections", [(128, [22, 21, 21]), (80, [20, 20]), (16, [8]), (256, [30, 20, 14]), (72, [5, 4]), (6, [1, 2]), (10, [3]), (2, [1])])
def test_rotation_of_every_width_type_and_layout(ea, dtype, pairing, dim, sections):
    g = gen(dim)
    for batch, rows, heads, kv, layout, span, interleaved in ((2, 37, 4, 2, "split", 100, False), (1, 1, 12, 1, "heads", 10, True), (3, 130, 3, 3, "fused", 1000000, True)):
        table = ea.RotaryTable.with_sections(dim, sections, theta=1e6, rot_dim=2 * sum(sections), interleaved=interleaved, pairing=pairing, scale=1.0 if heads == 4 else 0.75)
        q, k = make(g, batch, rows, heads, dim, DT[dtype], layout), make(g, batch, rows, kv, dim, DT[dtype], layout)
        for ptype in (torch.int64, torch.int32):
            pos = torch.randint(-5, span, (len(sections), batch, rows), generator=g, device="cuda").to(ptype)
            cos, sin = angles(pos, table)
            before = q.clone()
            got = ea.rotary(q, k, pos, table)
            for x, y in zip((q, k), got):
                check(y, *rotary_oracle(x, cos, sin, pairing, table.scale), what=(layout, ptype))
                assert y.is_contiguous()
            assert torch.equal(q, before)
        only_q, none = ea.rotary(q, None, pos, table)
        none2, only_k = ea.rotary(None, k, pos, table)
        assert none is None and none2 is None and torch.equal(only_q, got[0]) and torch.equal(only_k, got[1])
        a, b = ea.rotary(q, k, pos, table, in_place=True)
        assert a is q and b is k and torch.equal(q, got[0]) and torch.equal(k, got[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dim,pairs", [(72, 36), (72, 13), (40, 20), (23, 11), (17, 1), (9, 4), (24, 12), (130, 65)])
def test_rotation_at_any_alignment_leaves_its_neighbours(ea, dtype, pairing, dim, pairs):
    """Heads that start anywhere in 16 bytes, three elements between heads, five between rows: the elements between stay, in place gives the same bits."""
    g, heads, rows = gen(dim + pairs), 3, 41
    table = ea.RotaryTable.with_sections(dim, [pairs], rot_dim=2 * pairs, pairing=pairing)
    pos = torch.randint(0, 1000, (1, 1, rows), generator=g, device="cuda")
    cos, sin = angles(pos, table)
    for offset in (0, 1, 2, 5):
        row = heads * (dim + 3) + 5
        flat = torch.randn(offset + rows * row, generator=g, device="cuda").to(DT[dtype])
        before = flat.clone()
        q = flat.as_strided((1, rows, heads, dim), (rows * row, row, dim + 3, 1), offset)
        got = ea.rotary(q, None, pos, table)[0]
        check(got, *rotary_oracle(q, cos, sin, pairing))
        assert torch.equal(flat, before)
        ea.rotary(q, None, pos, table, in_place=True)
        assert torch.equal(q, got)
        before.as_strided(q.shape, q.stride(), offset).copy_(got)
        assert torch.equal(flat, before)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
def test_rotation_by_tables(ea, dtype, pairing):
    g = gen(21)
    for dim, pairs, batch, rows in ((80, 40, 1, 333), (128, 32, 3, 17), (24, 5, 2, 9)):
        q, k = make(g, batch, rows, 4, dim, DT[dtype], "fused"), make(g, batch, rows, 2, dim, DT[dtype], "split")
        angle = torch.rand(batch, rows, pairs, generator=g, device="cuda") * 9
        for cos, sin in ((angle.cos(), angle.sin()), (angle.cos()[:1], angle.sin()[:1]), tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (angle.cos(), angle.sin()))):
            got = ea.rotary_tables(q, k, cos, sin, pairing=pairing)
            for x, y in zip((q, k), got):
                check(y, *rotary_oracle(x, cos.double().expand(batch, -1, -1), sin.double().expand(batch, -1, -1), pairing))
        packed = ea.rotary_tables(q[0], k[0], angle.cos()[0], angle.sin()[0], pairing=pairing)
        assert packed[0].shape == q[0].shape and torch.equal(packed[0], ea.rotary_tables(q, k, angle.cos(), angle.sin(), pairing=pairing)[0][0])


def test_positions_of_fewer_dimensions(ea):
    g = gen(22)
    one, three = ea.RotaryTable.with_sections(32, [16]), ea.RotaryTable.with_sections(32, [6, 5, 5])
    q, k = make(g, 2, 7, 2, 32, DT["fp32"], "split"), make(g, 2, 7, 1, 32, DT["fp32"], "split")
    pos = torch.randint(0, 99, (3, 2, 7), generator=g, device="cuda")
    full = ea.rotary(q, k, pos[:1], one)[0]
    assert torch.equal(ea.rotary(q, k, pos[0], one)[0], full)  # [batch, rows]
    assert torch.equal(ea.rotary(q, k, pos[0, 0], one)[0], ea.rotary(q, k, pos[:1, :1].expand(1, 2, 7), one)[0])  # [rows]
    assert torch.equal(ea.rotary(q, k, pos[:, :1], three)[0], ea.rotary(q, k, pos[:, :1].expand(3, 2, 7), three)[0])  # one batch entry for all
    assert torch.equal(ea.rotary(q[1], k[1], pos[:, 1], three)[0], ea.rotary(q, k, pos, three)[0][1])  # [axes, rows] of packed rows
    assert ea.rotary(q[:, :0], k[:, :0], pos[:, :, :0], three)[0].shape == (2, 0, 2, 32)
    # a fused projection's views, turned in place, leave its values alone
    whole = torch.randn(2, 7, 4 * 32, generator=g, device="cuda")
    keep = whole.clone()
    a, b, c = (t.view(2, 7, -1, 32) for t in whole.split([64, 32, 32], -1))
    want = ea.rotary(a, b, pos, three)
    ea.rotary(a, b, pos, three, in_place=True)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(c.flatten(2), keep[..., 96:])


def test_rotation_of_offsets_past_32_bits(ea):
    rows = (1 << 24) + 7
    q = torch.zeros(1, rows, 1, 128, dtype=torch.bfloat16, device="cuda")
    q[0, -3:] = 1.0
    pos = torch.arange(rows, device="cuda")[None]
    table = ea.RotaryTable.with_sections(128, [64])
    want, tol = rotary_oracle(q[:, -3:], *angles(pos[None, :, -3:], table), "halves")
    check(ea.rotary(q, None, pos, table)[0][:, -3:], want, tol)
    ea.rotary(q, None, pos, table, in_place=True)
    check(q[:, -3:], want, tol)


# --------------------------------------------------------------------------- one behind the other, refusals on the device
def test_rotation_then_attention_as_a_block_uses_them(ea):
    """A decoder block's middle: fused projection -> three-axis rotation in place -> attention over a padded prefix, against 64 bits throughout.  The
    rotated operands are compared first; attention is then held to the oracle on those same operands."""
    g = gen(30)
    batch, rows, heads, kv, dim = 2, 150, 6, 2, 64
    whole = make(g, batch, rows, 1, (heads + 2 * kv) * dim, DT["bf16"], "split").view(batch, rows, -1)
    q, k, v = (t.view(batch, rows, -1, dim) for t in whole.split([heads * dim, kv * dim, kv * dim], -1))
    table = ea.RotaryTable.with_sections(dim, [12, 10, 10], theta=1e6)
    pos = torch.randint(0, 200, (3, batch, rows), generator=g, device="cuda")
    wq, wk = (rotary_oracle(x, *angles(pos, table), "halves") for x in (q, k))
    ea.rotary(q, k, pos, table, in_place=True)
    check(q, *wq), check(k, *wk)
    r = ea.padded_ranges(torch.tensor([0, 30], dtype=torch.int32, device="cuda"), torch.tensor([140, 150], dtype=torch.int32, device="cuda"), rows, prefix=100)
    check(ea.attention(q, k, v, key_ranges=r), *oracle(q, k, v, r))


def test_refusals_on_the_device(ea):
    q, k, v = (make(gen(1), 1, 4, 2, 16, DT["bf16"], "split") for _ in range(3))
    with pytest.raises(ValueError, match="different devices"):
        ea.attention(q, k, v.cpu())
    with pytest.raises(ValueError, match="different devices"):
        ea.attention(q, k, v, key_ranges=torch.zeros(1, 4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="different devices"):
        ea.rotary(q, k, torch.zeros(4, dtype=torch.int64), ea.RotaryTable.with_sections(16, [8]))
    with torch.enable_grad():
        with pytest.raises(ValueError, match="no gradient"):
            ea.attention(q.clone().requires_grad_(), k, v)
        with pytest.raises(ValueError, match="no gradient"):
            ea.rotary(q.clone().requires_grad_(), k, torch.zeros(4, dtype=torch.int64, device="cuda"), ea.RotaryTable.with_sections(16, [8]))
    with torch.no_grad():
        ea.attention(q.clone().requires_grad_(), k, v)


@pytest.mark.parametrize("rows,keys", [(1, 1), (77, 77), (5, 300), (300, 5), (200, 450)])
def test_causal_without_ranges(ea, rows, keys):
    g = gen(rows + keys)
    q, k, v = (make(g, 2, n, h, 72, DT["bf16"], "split") for n, h in ((rows, 6), (keys, 2), (keys, 2)))
    full = torch.full((2,), keys, dtype=torch.int32, device="cuda")
    at = torch.arange(rows, device="cuda", dtype=torch.int32) + keys - rows
    r = torch.stack([torch.zeros_like(at), (at + 1).clamp_min(0)], -1)[None]
    got = ea.attention(q, k, v, causal=True)
    check(got, *oracle(q, k, v, r))
    if rows <= keys:
        assert torch.equal(got, ea.attention(q, k, v, key_ranges=ea.padded_ranges(torch.zeros_like(full), full, rows, prefix=0, row_offset=keys - rows)))


# --------------------------------------------------------------------------- the encoders
def _encoder(kind):
    """A small random model of an encoder family with heads that the kernels take, in bf16 on the GPU, and batches for it: text of one length, padded
    text, images."""
    import numpy as np

    from tests import offline_assets as oa

    g = torch.Generator().manual_seed(7)
    if kind == "colpali":
        from transformers import ColPaliConfig, ColPaliForRetrieval, PaliGemmaConfig
        from transformers.models.gemma import GemmaConfig
        from transformers.models.siglip import SiglipVisionConfig

        vis = SiglipVisionConfig(vision_use_head=False, hidden_size=144, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2, image_size=56, patch_size=14)
        txt = GemmaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=1, head_dim=256, vocab_size=300)
        cfg = ColPaliConfig(vlm_config=PaliGemmaConfig(vision_config=vis, text_config=txt, image_token_index=299, projection_dim=256, hidden_size=256, vocab_size=300), embedding_dim=128)
        torch.manual_seed(5)
        model = ColPaliForRetrieval(cfg).to(torch.bfloat16).cuda().eval()
        images = dict(input_ids=torch.tensor([[299] * 16 + [1, 4, 2]] * 2), attention_mask=torch.ones(2, 19, dtype=torch.long), pixel_values=torch.rand(2, 3, 56, 56, generator=g).to(torch.bfloat16))
    else:
        from morphik_core_amd import colqwen_embedding as cq

        base = cq.PRESETS["tiny-2.5" if kind == "colqwen2.5" else "tiny"]
        widths = dict(hidden_size=160, out_hidden_size=256) if kind == "colqwen2.5" else dict(embed_dim=160, hidden_size=256)
        cq.PRESETS["_test"] = dict(base, vision={**base["vision"], **widths, "num_heads": 2},
                                   text={**base["text"], "hidden_size": 256, "num_attention_heads": 2, "num_key_value_heads": 1})
        proc, tokens = oa.colqwen2_processor()
        try:
            model = cq.build_random_colqwen2("_test", tokens, "cuda", torch.bfloat16)
        finally:
            del cq.PRESETS["_test"]
        rng = np.random.default_rng(0)
        b = proc(images=[oa.page_image(rng, 60, 60), oa.page_image(rng, 112, 84), oa.page_image(rng, 200, 140)], return_tensors="pt")
        images = {k: b[k].to(torch.bfloat16) if k == "pixel_values" else b[k] for k in ("input_ids", "attention_mask", "pixel_values", "image_grid_thw")}
    ids = torch.randint(1, 50, (3, 21), generator=g)
    padded = torch.ones_like(ids)
    padded[1, 13:] = 0
    padded[2, 1:] = 0
    batches = [dict(input_ids=ids, attention_mask=torch.ones_like(ids)), dict(input_ids=ids, attention_mask=padded), images]
    return model, [{k: v.cuda() for k, v in b.items()} for b in batches]


@pytest.mark.parametrize("kind", ["colpali", "colqwen2", "colqwen2.5"])
def test_encoders_with_patched_attention_embed_as_before(ea, kind, monkeypatch):
    """The patched model against itself in float32: no further off than the unpatched bf16 model is (its own roundings set the scale: half as far again,
    and a floor of four bf16 steps of a unit vector's rows), with the kernels running and nothing falling back; then unpatched, its own results again."""
    import copy

    model, batches = _encoder(kind)
    wide = copy.deepcopy(model).float()

    def embed(m, cast=False):
        out = []
        with torch.inference_mode():
            for b in batches:
                b = {k: v.float() if cast and v.is_floating_point() else v for k, v in b.items()}
                out.append(m(**b).embeddings.float().clone())
        return out

    exact, before = embed(wide, True), embed(model)
    calls = {"attention": 0, "turned": 0}
    attention, launch = ea.attention, ea._launch_rotary
    monkeypatch.setattr(ea, "attention", lambda *a, **k: (calls.__setitem__("attention", calls["attention"] + 1), attention(*a, **k))[1])
    monkeypatch.setattr(ea, "_launch_rotary", lambda *a, **k: (calls.__setitem__("turned", calls["turned"] + 1), launch(*a, **k))[1])
    counts = ea.patch_attention(model)
    got = embed(model)
    layers = len([m for m in model.modules() if type(m).__name__ in ("GemmaAttention", "Qwen2VLAttention", "Qwen2_5_VLAttention")])
    vision = len([m for m in model.modules() if type(m).__name__ in ("SiglipAttention", "VisionAttention", "Qwen2_5_VLVisionAttention")])
    assert counts["rotary"] == 1 and counts["decoder"] == layers and counts["packed"] == (0 if kind == "colpali" else vision)
    assert calls["attention"] == 3 * layers + vision and calls["turned"] == 3 * layers + counts["packed"]
    for b, x, y, z in zip(batches, exact, before, got):
        valid = b["attention_mask"].bool()
        off, base = (z - x)[valid].norm(dim=-1), (y - x)[valid].norm(dim=-1)
        print(f"{kind}: off the float32 model by {float(off.max()):.4f} (unpatched {float(base.max()):.4f})")
        assert float(off.max()) <= 1.5 * float(base.max()) + 4 * 2.0**-8 and bool(torch.isfinite(z).all())
    with torch.enable_grad():  # autograd on: the modules' own forwards
        n = dict(calls)
        assert model(**batches[0]).embeddings.requires_grad and calls == n
    ea.unpatch_attention(model)
    assert all(torch.equal(a, b) for a, b in zip(embed(model), before))


def test_embedding_model_with_fused_attention(ea):
    """The option of the embedding class, end to end: pages and queries, as many rows as without it and nearly the same directions."""
    import asyncio

    from morphik_core_amd.embedding import MI355XColpaliEmbeddingModel

    plain = MI355XColpaliEmbeddingModel(preset="tiny", device="cuda", seed=1)
    fused = MI355XColpaliEmbeddingModel(preset="tiny", device="cuda", seed=1, fused_attention=True)
    assert plain.fused_attention == {"rotary": 0, "decoder": 0, "packed": 0} and fused.fused_attention == {"rotary": 1, "decoder": 2, "packed": 0}
    for text in ("revenue", "what is the total revenue of the second quarter"):
        a, b = (asyncio.run(m.embed_for_query(text)) for m in (plain, fused))
        assert a.shape == b.shape and float((a * b).sum(-1).min()) > 0.99
