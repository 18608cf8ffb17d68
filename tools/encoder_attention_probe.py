#!/usr/bin/env python3
"""The encoders' rotary positions and attention (morphik_core_amd/encoder_attention.py) beside what the framework runs without them.

  python tools/encoder_attention_probe.py kernels            attention against scaled_dot_product_attention on the same tensors, us a call (device time)
  python tools/encoder_attention_probe.py encoders           whole forwards, fused_attention off and on in turn: ColPali-v1.2 (16 pages, one query), ColQwen2 and
                                                             ColQwen2.5-3B (eight small pages); random weights of the full architectures
  python tools/encoder_attention_probe.py one B L H HK D dtype   one attention call, 20 times: the workload of a counter pass
One JSON object on stdout."""
import json
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from morphik_core_amd import encoder_attention as ea

# batch, rows, heads, K/V heads, head width, type: the blocks of the two encoder families at their working sizes, and round ones of each width
SHAPES = [(8, 1024, 16, 16, 72, "bf16"), (8, 1030, 8, 1, 256, "bf16"), (1, 8464, 16, 16, 80, "bf16"), (1, 8464, 16, 16, 80, "fp16"), (8, 1101, 12, 2, 128, "bf16"),
          (8, 1101, 16, 2, 128, "bf16"), (2, 4096, 16, 16, 64, "bf16"), (2, 4096, 16, 16, 128, "bf16"), (4, 2048, 8, 1, 256, "bf16")]
CAUSAL = {(8, 1101, 12, 2, 128, "bf16"), (8, 1101, 16, 2, 128, "bf16")}


def qkv(batch, rows, heads, kv, dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(batch, rows, h, dim, generator=g, device="cuda").to({"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]) for h in (heads, kv, kv)]


def us(fn, calls=20, rounds=5):
    for _ in range(3):
        fn()
    best = float("inf")
    for _ in range(rounds):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(calls):
            fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) / calls * 1e3)
    return best


def kernels():
    out = {}
    for shape in SHAPES:
        batch, rows, heads, kv, dim, dtype = shape
        q, k, v = qkv(*shape)
        causal = shape in CAUSAL
        flops = 4 * batch * heads * rows * rows * dim / (2 if causal else 1)
        with torch.inference_mode():
            ours = us(lambda: ea.attention(q, k, v, causal=causal))
            heads_first = [t.transpose(1, 2).contiguous() for t in (q, k, v)]
            sdpa = us(lambda: torch.nn.functional.scaled_dot_product_attention(*heads_first, is_causal=causal, enable_gqa=heads != kv))
        out[f"{batch} x {rows} rows, {heads} heads over {kv}, {dim} wide, {dtype}" + (", causal" if causal else "")] = {
            "attention_us": round(ours, 1), "PFLOPs": round(flops / ours / 1e9, 3), "sdpa_us": round(sdpa, 1)}
    return out


def timed(fn, calls):
    fn()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(calls):
        fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / calls


def in_turn(model, forwards, rounds=3, calls=6):
    """ms of each forward without and with the kernels, best of some rounds of both in turn."""
    best = {}
    with torch.inference_mode():
        for _ in range(rounds):
            for kind in ("without", "with"):
                if kind == "with":
                    ea.patch_attention(model)
                for name, fn in forwards.items():
                    ms = timed(fn, calls) * 1e3
                    best.setdefault(name, {})[kind] = min(ms, best.get(name, {}).get(kind, ms))
                ea.unpatch_attention(model)
    return {name: {k: round(x, 2) for k, x in both.items()} for name, both in best.items()}


def encoders():
    import asyncio

    import numpy as np

    from morphik_core_amd.colqwen_embedding import build_random_colqwen2
    from morphik_core_amd.embedding import MI355XColpaliEmbeddingModel
    from tests import offline_assets as oa

    out = {}
    emb = MI355XColpaliEmbeddingModel(preset="colpali-v1.2", device="cuda:0", fused_attention=False)
    n = emb.n_image_tokens
    g = torch.Generator().manual_seed(0)
    image_token = int(emb.model.config.vlm_config.image_token_index if hasattr(emb.model.config.vlm_config, "image_token_index") else emb.model.config.vlm_config.image_token_id)
    pages = dict(input_ids=torch.tensor([[image_token] * n + [2, 9, 11, 14, 15, 16]] * 16), attention_mask=torch.ones(16, n + 6, dtype=torch.long),
                 pixel_values=torch.rand(16, 3, emb.image_size, emb.image_size, generator=g).to(torch.bfloat16))
    pages = {k: v.cuda() for k, v in pages.items()}
    res = in_turn(emb.model, {"16 pages, ms": lambda: emb.model(**pages),
                              "one query (text to rows on the host), ms": lambda: asyncio.run(emb.embed_for_query("what is the total revenue of the second quarter"))})
    res["16 pages, pages/s"] = {k: round(16e3 / ms, 1) for k, ms in res["16 pages, ms"].items()}
    out["colpali-v1.2"] = res
    del emb
    torch.cuda.empty_cache()
    for preset in ("colqwen2-v1.0", "colqwen2.5-3b"):
        proc, ids = oa.colqwen2_processor(min_tokens=64, max_tokens=768)
        model = build_random_colqwen2(preset, ids, "cuda:0", torch.bfloat16)
        rng = np.random.default_rng(8)
        b = proc(images=[oa.page_image(rng, h, w) for h, w in ((448, 448), (560, 420), (336, 672), (784, 588), (448, 448), (280, 280), (700, 500), (644, 476))], return_tensors="pt")
        small = {k: (b[k].to(torch.bfloat16) if k == "pixel_values" else b[k]).cuda() for k in ("input_ids", "attention_mask", "pixel_values", "image_grid_thw")}
        out[preset] = in_turn(model, {"eight small pages, ms": lambda: model(**small)})
        del model
        torch.cuda.empty_cache()
    return out


def main():
    what = sys.argv[1]
    if what == "one":
        shape = (*(int(x) for x in sys.argv[2:7]), sys.argv[7])
        q, k, v = qkv(*shape)
        with torch.inference_mode():
            for _ in range(20):
                ea.attention(q, k, v)
        torch.cuda.synchronize()
        return
    print(json.dumps({"device": torch.cuda.get_device_name(0), "torch": torch.__version__, what: kernels() if what == "kernels" else encoders()}, indent=1))


if __name__ == "__main__":
    main()
