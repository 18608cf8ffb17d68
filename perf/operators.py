"""The encoder's attention operators, as cases to time and to check: multi-axis rotary positions and attention over key ranges
(documents, prefixes, padding, capped scores), in plain torch operations (`own` false) or through the framework's entry points
(`own` true).  Every case is a dict of plain values; `prepare` makes its inputs from a seed, `run` is one call."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 1000000.0


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a search query of 20 tokens through one decoder layer: the smallest call, latency counts (8 heads over one K/V head of 256)
        dict(name="query_text", op="attention", form="padded", batch=1, rows=20, keys=20, heads=8, kv_heads=1, dim=256, dtype="bf16",
             mask="prefix", prefix=8, pad="right", softcap=0.0, layout="heads", lengths="full", shape_seed=0),
        # 32 queries of different lengths in one padded batch, causal decoder, 12 heads over 2 K/V heads
        dict(name="query_batch", op="attention", form="padded", batch=32, rows=39, keys=39, heads=12, kv_heads=2, dim=128, dtype="bf16",
             mask="causal", prefix=0, pad="left", softcap=0.0, layout="heads", lengths="ragged", shape_seed=1),
        # eight 448-pixel pages in the vision tower: 1024 patches, 16 heads of 72, every patch sees its page
        dict(name="page_vision", op="attention", form="padded", batch=8, rows=1024, keys=1024, heads=16, kv_heads=16, dim=72, dtype="bf16",
             mask="full", prefix=0, pad="right", softcap=0.0, layout="split", lengths="full", shape_seed=2),
        # the same pages behind it in the decoder: 1024 patch tokens that see each other, then a causal prompt; shorter pages padded
        dict(name="page_text", op="attention", form="padded", batch=8, rows=1030, keys=1030, heads=8, kv_heads=1, dim=256, dtype="bf16",
             mask="prefix", prefix=1024, pad="right", softcap=0.0, layout="heads", lengths="ragged", shape_seed=3),
        # windowed layers of a dynamic-resolution vision tower: eight pages packed, windows of 64 patches and the ragged ones at page borders
        dict(name="vision_windows", op="attention", form="documents", docs="windows", pages=8, page=46 * 34, heads=16, kv_heads=16, dim=80,
             dtype="bf16", mask="full", prefix=0, softcap=0.0, layout="fused", shape_seed=4),
        # its full-attention layers: pages of very different resolution packed one behind the other, a 16-patch one among them; the largest
        dict(name="vision_pages", op="attention", form="documents", docs="pages", pages=6, page=8464, heads=16, kv_heads=16, dim=80,
             dtype="fp16", mask="full", prefix=0, softcap=0.0, layout="fused", shape_seed=5),
        # a causal decoder with capped scores over left-padded text, one request of the batch empty
        dict(name="text_capped", op="attention", form="padded", batch=5, rows=733, keys=733, heads=16, kv_heads=2, dim=128, dtype="fp16",
             mask="causal", prefix=0, pad="left", softcap=50.0, layout="split", lengths="one_empty", shape_seed=6),
        # one more token behind long texts: a single row for each, thousands of keys
        dict(name="next_token", op="attention", form="padded", batch=3, rows=1, keys=16001, heads=16, kv_heads=2, dim=128, dtype="bf16",
             mask="causal", prefix=0, pad="left", softcap=0.0, layout="heads", lengths="ragged", shape_seed=7),
        # positions of one query (time, height, width equal on text): latency
        dict(name="rotary_query", op="rotary", batch=1, rows=20, heads=12, kv_heads=2, dim=128, rot_dim=128, axes=3, sections="blocks",
             pairing="halves", dtype="bf16", layout="heads", span=20, source="positions", shape_seed=8),
        # positions of eight pages of about 1100 tokens in the decoder
        dict(name="rotary_pages", op="rotary", batch=8, rows=1101, heads=16, kv_heads=2, dim=128, rot_dim=128, axes=3, sections="blocks",
             pairing="halves", dtype="bf16", layout="heads", span=1101, source="positions", shape_seed=9),
        # the vision tower's packed patches, q and k inside the fused projection, angles given as cosines and sines
        dict(name="rotary_patches", op="rotary", batch=1, rows=8 * 46 * 34, heads=16, kv_heads=16, dim=80, rot_dim=80, axes=2, sections="grid",
             pairing="halves", dtype="bf16", layout="fused", span=92, source="tables", shape_seed=10),
        # a long video in 32 bits: times far from zero, axes interleaved, half of each head rotated, neighbouring elements as pairs
        dict(name="rotary_video", op="rotary", batch=2, rows=4001, heads=8, kv_heads=1, dim=256, rot_dim=128, axes=3, sections="interleaved",
             pairing="adjacent", dtype="fp32", layout="split", span=1000000, source="positions", shape_seed=11),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    kv = rng.choice([1, 1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 6, 8] if kv < 8 else [1, 2])
    layout = rng.choice(["split", "heads", "fused"])
    shape_seed = rng.randrange(1 << 30)
    if rng.random() < 0.35:
        dim = 8 * _log_int(rng, 2, 32)
        source = rng.choice(["positions", "positions", "tables"])
        return dict(op="rotary", batch=_log_int(rng, 1, 8), rows=_log_int(rng, 1, 4100), heads=heads, kv_heads=kv, dim=dim,
                    rot_dim=dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2), axes=rng.choice([1, 2, 3]),
                    sections=rng.choice(["blocks", "interleaved", "grid"]), pairing=rng.choice(["halves", "adjacent"]),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), layout=layout, span=_log_int(rng, 32, 1000000), source=source,
                    shape_seed=shape_seed)
    dim = rng.choice([64, 72, 80, 96, 128, 256, 8 * rng.randint(2, 32)])
    mask = rng.choice(["full", "causal", "prefix"])
    softcap = rng.choice([0.0, 0.0, 30.0, 50.0])
    common = dict(op="attention", heads=heads, kv_heads=kv, dim=dim, dtype=dtype, mask=mask, softcap=softcap, layout=layout, shape_seed=shape_seed)
    kind = rng.random()
    if kind < 0.3:
        docs = rng.choice(["windows", "pages"])
        page = _log_int(rng, 16, 3000)
        return dict(common, form="documents", docs=docs, pages=_log_int(rng, 1, 8), page=page, prefix=_log_int(rng, 1, page) if mask == "prefix" else 0)
    if kind < 0.5:  # few rows behind many keys
        rows = _log_int(rng, 1, 32)
        keys = rows + _log_int(rng, 1, 16000)
        batch = _log_int(rng, 1, 4)
        lengths = rng.choice(["full", "ragged"])
        pad = "left"
    else:
        rows = keys = _log_int(rng, 1, 2000)
        batch = _log_int(rng, 1, 8)
        lengths = rng.choice(["full", "ragged", "ragged", "one_empty"] if batch > 1 else ["full", "ragged"])
        pad = rng.choice(["left", "right"])
    return dict(common, form="padded", batch=batch, rows=rows, keys=keys, prefix=_log_int(rng, 1, keys) if mask == "prefix" else 0, pad=pad, lengths=lengths)


# --------------------------------------------------------------------------- shapes that follow from a case alone
def _documents(case):
    """Lengths of the packed documents."""
    rng = random.Random(case["shape_seed"])
    if case["docs"] == "windows":  # windows of 64 patches; what is left over at a page's border comes in shorter ones
        out = []
        for _ in range(case["pages"]):
            left = case["page"]
            while left > 0:
                n = min(left, 64 if rng.random() < 0.75 else rng.choice([16, 32, 48, rng.randint(1, 63)]))
                out.append(n)
                left -= n
        return out
    return [case["page"]] + [max(1, int(case["page"] * rng.random() ** 2)) for _ in range(case["pages"] - 1)]


def _spans(case):
    """(first valid key, end of the valid keys) of every sequence of a padded batch."""
    rng = random.Random(case["shape_seed"])
    n, out = case["keys"], []
    for b in range(case["batch"]):
        if case["lengths"] == "full" or (b == 0 and case["lengths"] == "ragged"):
            ln = n
        elif case["lengths"] == "one_empty" and b == case["batch"] - 1:
            ln = 0
        else:
            ln = rng.randint(1, n)
        out.append((n - ln, n) if case["pad"] == "left" else (0, ln))
    return out


def _row_range(case, start, end, position):
    """The keys [lo, hi) that the row at `position` sees; nothing where the row itself is padding."""
    if not start <= position < end:
        return 0, 0
    if case["mask"] == "full":
        return start, end
    return start, max(position + 1, min(start + case["prefix"], end))


def _sequences(case):
    """For each sequence: (its batch entry, first row, rows, position of the first row, start, end)."""
    if case["form"] == "documents":
        out, at = [], 0
        for n in _documents(case):
            out.append((0, at, n, at, at, at + n))
            at += n
        return out
    shift = case["keys"] - case["rows"]
    return [(b, 0, case["rows"], shift, s, e) for b, (s, e) in enumerate(_spans(case))]


def _dims(case):
    if case["form"] == "documents":
        t = sum(_documents(case))
        return 1, t, t
    return case["batch"], case["rows"], case["keys"]


def _sections(case):
    """-> for each pair its axis, for each pair its frequency."""
    pairs, axes = case["rot_dim"] // 2, case["axes"]
    if case["sections"] == "interleaved":
        axis = [j % axes for j in range(pairs)]
    else:
        part = pairs // axes
        bounds = [pairs - (axes - 1) * part] + [part] * (axes - 1)  # the first axis takes what does not divide
        axis = [a for a, n in enumerate(bounds) for _ in range(n)]
    if case["sections"] == "grid":  # every axis runs through the frequencies from the start
        seen, freq = {}, []
        for a in axis:
            i = seen.get(a, 0)
            seen[a] = i + 1
            freq.append(10000.0 ** (-i / max(1, axis.count(a))))
    else:
        freq = [THETA ** (-j / pairs) for j in range(pairs)]
    return axis, freq


# --------------------------------------------------------------------------- inputs
def _heads(gen, case, batch, rows, heads, dtype, spread):
    x = torch.randn(batch, rows, heads, case["dim"], generator=gen, device="cuda")
    if spread:  # heads differ in how sharply they attend
        x *= torch.rand(heads, 1, generator=gen, device="cuda") * 2 + 0.5
    return x.to(dtype)


def _laid_out(case, parts):
    """The tensors [batch, rows, heads, dim] as a program holds them: each by itself, heads outside rows, or inside one fused projection."""
    if case["layout"] == "heads":
        return [p.transpose(1, 2).contiguous().transpose(1, 2) for p in parts]
    if case["layout"] == "fused" and all(p.shape[:2] == parts[0].shape[:2] for p in parts):
        whole = torch.cat(parts, 2).contiguous()
        return list(whole.split([p.shape[2] for p in parts], 2))
    return [p.contiguous() for p in parts]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "attention":
        batch, rows, keys = _dims(case)
        q = _heads(gen, case, batch, rows, case["heads"], dtype, True)
        k = _heads(gen, case, batch, keys, case["kv_heads"], dtype, False)
        v = _heads(gen, case, batch, keys, case["kv_heads"], dtype, False)
        q, k, v = _laid_out(case, [q, k, v])
        return dict(case=case, q=q, k=k, v=v)
    batch, rows = case["batch"], case["rows"]
    q = _heads(gen, case, batch, rows, case["heads"], dtype, False)
    k = _heads(gen, case, batch, rows, case["kv_heads"], dtype, False)
    v = _heads(gen, case, batch, rows, case["kv_heads"], dtype, False)
    q, k, _ = _laid_out(case, [q, k, v])
    positions = torch.randint(0, case["span"] + 1, (case["axes"], batch, rows), generator=gen, device="cuda")
    positions[0] = positions[0].sort(-1).values  # time runs on, height and width come and go
    axis, freq = _sections(case)
    state = dict(case=case, q=q, k=k, positions=positions, axis=torch.tensor(axis, device="cuda"), freq=torch.tensor(freq, dtype=torch.float64, device="cuda"))
    if case["source"] == "tables":
        angle = positions[state["axis"]].permute(1, 2, 0).double() * state["freq"]
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def prepare(case, seed):
    """The inputs and, for the framework's own kernels, the plan of a forward: the key ranges, the table of frequencies."""
    state = _inputs(case, seed)
    if not own:
        return state
    from morphik_core_amd import encoder_attention as ea

    if case["op"] == "rotary":
        if case["source"] == "positions":
            state["table"] = ea.RotaryTable(state["freq"], state["axis"], head_dim=case["dim"], pairing=case["pairing"])
        return state
    _, rows, keys = _dims(case)
    prefix = None if case["mask"] == "full" else case["prefix"]
    state["ranges"] = None  # every row sees every key
    if case["form"] == "documents":
        ends = torch.tensor([0] + _documents(case), dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        state["ranges"] = ea.document_ranges(ends, rows, prefix=prefix)
    elif prefix is not None or case["lengths"] != "full":
        spans = torch.tensor(_spans(case), dtype=torch.int32).cuda()
        state["ranges"] = ea.padded_ranges(spans[:, 0], spans[:, 1], rows, prefix=prefix, row_offset=keys - rows)
    return state


# --------------------------------------------------------------------------- one call
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        if not own:
            return _plain_attention(state)
        from morphik_core_amd import encoder_attention as ea

        return ea.attention(state["q"], state["k"], state["v"], key_ranges=state["ranges"], softcap=case["softcap"])
    if not own:
        return _plain_rotary(state)
    from morphik_core_amd import encoder_attention as ea

    if case["source"] == "tables":
        return ea.rotary_tables(state["q"], state["k"], state["cos"], state["sin"], pairing=case["pairing"])
    return ea.rotary(state["q"], state["k"], state["positions"], state["table"])


def _plain_attention(state):
    """Scores, cap, mask, softmax by exp and sum, product with the values, in 32 bits; documents of one length go together."""
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    batch, rows, heads, dim = q.shape
    if case["form"] == "documents":
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
        starts, at = {}, 0
        for n in _documents(case):
            starts.setdefault(n, []).append(at)
            at += n
        for n, first in starts.items():
            index = torch.tensor(first, device=q.device)[:, None] + torch.arange(n, device=q.device)
            seen = None
            if case["mask"] != "full":
                i = torch.arange(n, device=q.device)
                seen = ((i[None] <= i[:, None]) | (i[None] < case["prefix"]))[None]
            out[index] = _plain_block(case, q[0, index], k[0, index], v[0, index], seen)
        return out[None]
    seen = None
    if case["mask"] != "full" or case["lengths"] != "full":
        spans = torch.tensor(_spans(case), device=q.device)
        start, end = spans[:, 0, None, None], spans[:, 1, None, None]
        at = torch.arange(case["keys"] - rows, case["keys"], device=q.device)[None, :, None]
        key = torch.arange(case["keys"], device=q.device)[None, None]
        seen = (at >= start) & (at < end) & (key >= start) & (key < end)
        if case["mask"] != "full":
            seen = seen & ((key <= at) | (key < start + case["prefix"]))
    return _plain_block(case, q, k, v, seen)


def _plain_block(case, q, k, v, seen):
    """[entries, rows, heads, dim] over [entries, keys, kv heads, dim]; `seen` [entries, rows, keys] or None."""
    entries, rows, heads, dim = q.shape
    keys, kv = k.shape[1], k.shape[2]
    out = torch.empty(entries, rows, heads, dim, dtype=q.dtype, device=q.device)
    ks = k.float().permute(0, 2, 3, 1).contiguous()  # [entries, kv heads, dim, keys]
    vs = v.float().transpose(1, 2).contiguous()
    step = max(1, (1 << 30) // (entries * heads * keys))
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        qs = q[:, r0:r1].float().permute(0, 2, 1, 3).reshape(entries, kv, (heads // kv) * (r1 - r0), dim)
        s = torch.matmul(qs, ks).view(entries, heads, r1 - r0, keys) / math.sqrt(dim)
        if case["softcap"]:
            s = torch.tanh(s / case["softcap"]) * case["softcap"]
        if seen is not None:
            s = s.masked_fill(~(seen[:, r0:r1] if seen.shape[1] == rows else seen)[:, None], float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, torch.ones_like(total), total)
        o = torch.matmul(p.view(entries, kv, -1, keys), vs)
        out[:, r0:r1] = o.view(entries, heads, r1 - r0, dim).transpose(1, 2).to(q.dtype)
    return out


def _plain_rotary(state):
    case = state["case"]
    if case["source"] == "tables":
        cos, sin = state["cos"], state["sin"]
    else:  # angles in 64 bits: a product of a far position and its frequency loses its fraction in 32
        angle = state["positions"][state["axis"]].permute(1, 2, 0).double() * state["freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
    cos, sin = cos[:, :, None], sin[:, :, None]
    pairs = case["rot_dim"] // 2
    out = []
    for x in (state["q"], state["k"]):
        w = x.float()
        if case["pairing"] == "halves":
            a, b = w[..., :pairs], w[..., pairs : 2 * pairs]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin, w[..., 2 * pairs :]], -1)
        else:
            a, b = w[..., 0 : 2 * pairs : 2], w[..., 1 : 2 * pairs : 2]
            r = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), w[..., 2 * pairs :]], -1)
        out.append(r.to(x.dtype))
    return tuple(out)


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    return _exact_attention(case, state)


def _exact_attention(case, state):
    """Row by row of the definition: every row has its key range [lo, hi); blocks of rows share one product over the keys they reach."""
    q, k, v = state["q"], state["k"], state["v"]
    batch, rows, heads, dim = q.shape
    out = torch.zeros(batch, rows, heads, dim, dtype=torch.float64, device=q.device)
    lo = torch.zeros(batch, rows, dtype=torch.int64)
    hi = torch.zeros(batch, rows, dtype=torch.int64)
    for b, first, n, position, start, end in _sequences(case):
        for i in range(n):
            lo[b, first + i], hi[b, first + i] = _row_range(case, start, end, position + i)
    for b in range(batch):
        r0 = 0
        while r0 < rows:
            r1 = min(rows, r0 + 512)
            live = hi[b, r0:r1] > lo[b, r0:r1]
            if bool(live.any()):
                k0, k1 = int(lo[b, r0:r1][live].min()), int(hi[b, r0:r1][live].max())
                key = torch.arange(k0, k1, device=q.device)
                seen = (key >= lo[b, r0:r1, None].to(q.device)) & (key < hi[b, r0:r1, None].to(q.device))
                none = ~seen.any(-1)
                for h in range(heads):
                    g = h // (heads // k.shape[2])
                    s = (q[b, r0:r1, h].double() @ k[b, k0:k1, g].double().t().contiguous()) * dim**-0.5
                    if case["softcap"]:
                        s = case["softcap"] * torch.tanh(s / case["softcap"])
                    w = torch.where(seen, s, torch.full_like(s, -1e300))
                    w = torch.where(seen, torch.exp(w - w.amax(-1, keepdim=True)), torch.zeros_like(w))
                    o = (w @ v[b, k0:k1, g].double()) / w.sum(-1, keepdim=True)
                    out[b, r0:r1, h] = torch.where(none[:, None], torch.zeros_like(o), o)
            r0 = r1
    return out


def _exact_rotary(case, state):
    """Each pair as a complex number, turned by exp(i angle)."""
    if case["source"] == "tables":
        turn = torch.complex(state["cos"].double(), state["sin"].double())
    else:
        angle = torch.stack([state["positions"][a].double() * f for a, f in zip(state["axis"].tolist(), state["freq"].tolist())], -1)
        turn = torch.complex(torch.cos(angle), torch.sin(angle))
    pairs, out = case["rot_dim"] // 2, []
    first = torch.arange(pairs, device="cuda") * (1 if case["pairing"] == "halves" else 2)
    second = first + (pairs if case["pairing"] == "halves" else 1)
    for x in (state["q"], state["k"]):
        w = x.double()
        z = torch.complex(w[..., first], w[..., second]) * turn[:, :, None]
        r = w.clone()
        r[..., first], r[..., second] = z.real, z.imag
        out.append(r)
    return tuple(out)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "rotary":
        tokens = case["batch"] * case["rows"]
        values = tokens * (case["heads"] + case["kv_heads"])
        angles = tokens * (case["axes"] * 8 if case["source"] == "positions" else case["rot_dim"] * 4)
        return {"bytes": 2 * values * case["dim"] * size + angles, "flops": values * case["rot_dim"] * 3}
    batch, rows, _ = _dims(case)
    pairs = seen_rows = seen_keys = 0
    for _b, _first, n, position, start, end in _sequences(case):
        furthest = 0
        for i in range(n):
            lo, hi = _row_range(case, start, end, position + i)
            pairs += hi - lo
            seen_rows += hi > lo
            furthest = max(furthest, hi - lo)
        seen_keys += furthest
    moved = (seen_rows + batch * rows) * case["heads"] + 2 * seen_keys * case["kv_heads"]
    return {"bytes": moved * case["dim"] * size + (8 * batch * rows if case["mask"] != "full" or case["form"] == "documents" or case["lengths"] != "full" else 0),
            "flops": 4 * case["dim"] * case["heads"] * pairs}
