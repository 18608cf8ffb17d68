"""Multi-axis rotary positions and attention over key ranges: what the entry points refuse, without a GPU (every refusal comes before anything is
launched), and the plan objects that live on the host."""
import ctypes as C
import math
import os
import shutil
import subprocess
import sys

import pytest
import torch

from morphik_core_amd import _lib
from morphik_core_amd import encoder_attention as ea

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def qkv(batch=2, rows=5, keys=5, heads=4, kv=2, dim=16, dtype=torch.bfloat16):
    return (torch.zeros(batch, rows, heads, dim, dtype=dtype), torch.zeros(batch, keys, kv, dim, dtype=dtype), torch.zeros(batch, keys, kv, dim, dtype=dtype))


def test_attention_refuses_what_it_cannot_do():
    q, k, v = qkv()
    with pytest.raises(ValueError, match="on a GPU"):
        ea.attention(q, k, v)
    for dtype in (torch.float32, torch.float64, torch.int16):
        with pytest.raises(ValueError, match="dtype"):
            ea.attention(*qkv(dtype=dtype))
    with pytest.raises(ValueError, match="differ in type"):
        ea.attention(q, k.half(), v)
    with pytest.raises(ValueError, match="do not fit"):
        ea.attention(q, k, v[:, :4])
    with pytest.raises(ValueError, match="do not fit"):
        ea.attention(q[:1], k, v)
    with pytest.raises(ValueError, match="do not fit"):
        ea.attention(q, k[..., :8], v[..., :8])
    with pytest.raises(ValueError, match="multiple"):
        ea.attention(*qkv(heads=3, kv=2))
    with pytest.raises(ValueError, match="multiple"):
        ea.attention(*qkv(heads=0, kv=2))
    for dim in (4, 12, 264):
        with pytest.raises(ValueError, match="multiples of 8 up to 256"):
            ea.attention(*qkv(dim=dim))
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ea.attention(q, k, v, scale=scale)
    for cap in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="softcap"):
            ea.attention(q, k, v, softcap=cap)
    with pytest.raises(ValueError, match="causal goes without"):
        ea.attention(q, k, v, causal=True, key_ranges=torch.zeros(2, 5, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="batch, rows, heads, dim"):
        ea.attention(q[0, 0], k, v)
    with pytest.raises(ValueError, match="side by side"):
        ea.attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v)
    wide = torch.zeros(2, 5, 4, 20, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="side by side"):
        ea.attention(wide[..., :16], k, v)  # heads every 20 elements
    shifted = torch.zeros(2 * 5 * 4 * 16 + 8, dtype=torch.bfloat16)[4:-4].view(2, 5, 4, 16)
    with pytest.raises(ValueError, match="side by side"):
        ea.attention(shifted, k, v)  # 8 bytes off
    for bad in (torch.zeros(2, 5, 2), torch.zeros(3, 5, 2, dtype=torch.int32), torch.zeros(2, 4, 2, dtype=torch.int32), torch.zeros(2, 5, dtype=torch.int32),
                torch.zeros(2, 5, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="key_ranges"):
            ea.attention(q, k, v, key_ranges=bad)


def test_rotary_refuses_what_it_cannot_do():
    q, k, _ = qkv()
    table = ea.RotaryTable.with_sections(16, [4, 2, 2], device="cpu")
    pos = torch.zeros(3, 2, 5, dtype=torch.int64)
    with pytest.raises(ValueError, match="on a GPU"):
        ea.rotary(q, k, pos, table)
    with pytest.raises(ValueError, match="RotaryTable"):
        ea.rotary(q, k, pos, (1, 2))
    with pytest.raises(ValueError, match="neither"):
        ea.rotary(None, None, pos, table)
    with pytest.raises(ValueError, match="dtype"):
        ea.rotary(q.double(), k.double(), pos, table)
    with pytest.raises(ValueError, match="differ"):
        ea.rotary(q, k.half(), pos, table)
    with pytest.raises(ValueError, match="differ"):
        ea.rotary(q, k[:, :3], pos, table)
    with pytest.raises(ValueError, match="int32 or int64"):
        ea.rotary(q, k, pos.float(), table)
    for bad in (pos[:, :, :4], pos[:, :1].expand(3, 3, 5), pos[None]):
        with pytest.raises(ValueError, match="do not fit"):
            ea.rotary(q, k, bad, table)
    with pytest.raises(ValueError, match="axes"):
        ea.rotary(q, k, pos[:2], table)
    with pytest.raises(ValueError, match="heads of 16"):
        ea.rotary(q, k, pos, ea.RotaryTable.with_sections(32, [16], device="cpu"))
    with pytest.raises(ValueError, match="next to each other"):
        ea.rotary(q.transpose(1, 3).contiguous().transpose(1, 3), k, pos, table)
    with pytest.raises(ValueError, match="share memory"):
        ea.rotary(q[:, :, :1].expand(-1, -1, 4, -1), k, pos, table, in_place=True)
    with pytest.raises(ValueError, match="share memory"):
        ea.rotary(q, q[:, :, 1:3], pos, table, in_place=True)
    cos = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError, match="on a GPU"):
        ea.rotary_tables(q, k, cos, cos)
    with pytest.raises(ValueError, match="float32"):
        ea.rotary_tables(q, k, cos.half(), cos.half())
    with pytest.raises(ValueError, match="differ"):
        ea.rotary_tables(q, k, cos, cos[:1])
    for bad in (torch.zeros(2, 5, 9), torch.zeros(2, 4, 8), torch.zeros(3, 5, 8), torch.zeros(8)):
        with pytest.raises(ValueError, match="does not fit"):
            ea.rotary_tables(q, k, bad, bad)
    with pytest.raises(ValueError, match="pairing"):
        ea.rotary_tables(q, k, cos, cos, pairing="neighbours")


def test_views_of_a_fused_projection_may_be_turned_in_place():
    """The guard against shared memory lets the views through that a fused projection gives."""
    whole = torch.zeros(2, 5, 8 * 16)
    q, k, v = (t.view(2, 5, -1, 16) for t in whole.split([4 * 16, 2 * 16, 2 * 16], -1))
    assert not ea._overlaps(q) and not ea._share_memory(q, k) and not ea._share_memory(k, q) and not ea._share_memory(k, v)
    assert ea._share_memory(q, whole.view(2, 5, 8, 16)[:, :, 3:5])
    assert not ea._share_memory(q.contiguous(), k.contiguous())
    assert ea._overlaps(q[:, :, :1].expand(-1, -1, 4, -1)) and not ea._overlaps(q.transpose(1, 2))


def test_ranges_refuse_what_they_cannot_do():
    s = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="on a GPU"):
        ea.padded_ranges(s, s, 4)
    with pytest.raises(ValueError, match="int32"):
        ea.padded_ranges(s.long(), s, 4)
    with pytest.raises(ValueError, match="int32"):
        ea.padded_ranges(s, s[:2], 4)
    with pytest.raises(ValueError, match="negative"):
        ea.padded_ranges(s, s, -1)
    with pytest.raises(ValueError, match="negative"):
        ea.padded_ranges(s, s, 4, row_offset=-1)
    with pytest.raises(ValueError, match="negative"):
        ea.padded_ranges(s, s, 4, prefix=-2)
    with pytest.raises(ValueError, match="prefix"):
        ea.padded_ranges(s, s, 4, prefix=s[:2])
    with pytest.raises(ValueError, match="on a GPU"):
        ea.document_ranges(s, 4)
    with pytest.raises(ValueError, match="int32"):
        ea.document_ranges(s[:0], 4)
    with pytest.raises(ValueError, match="int32"):
        ea.document_ranges(s.long(), 4)
    with pytest.raises(ValueError, match="prefix"):
        ea.document_ranges(s, 4, prefix=s)  # three offsets are two documents
    with pytest.raises(ValueError, match="boolean"):
        ea.ranges_from_mask(torch.zeros(2, 3, 4))


def test_ranges_from_mask_says_when_a_row_is_not_one_run():
    m = torch.zeros(2, 4, 6, dtype=torch.bool)
    m[0, 0, 2:5] = True
    m[0, 1, :] = True
    m[1, 2, 5] = True
    r, ok = ea.ranges_from_mask(m)
    assert bool(ok) and r.dtype == torch.int32
    assert r[0].tolist() == [[2, 5], [0, 6], [0, 0], [0, 0]] and r[1].tolist() == [[0, 0], [0, 0], [5, 6], [0, 0]]
    m[1, 3, 0] = m[1, 3, 2] = True
    assert not bool(ea.ranges_from_mask(m)[1])
    assert ea.ranges_from_mask(m[:, :, :0])[0].tolist() == [[[0, 0]] * 4] * 2


def test_rotary_table_of_sections_and_of_a_grid():
    t = ea.RotaryTable.with_sections(16, [4, 2, 2], theta=100.0, device="cpu")
    assert t.axis.tolist() == [0, 0, 0, 0, 1, 1, 2, 2] and t.axes == 3 and t.pairs == 8
    assert torch.equal(t.inv_freq, torch.tensor([100.0 ** (-j / 8) for j in range(8)], dtype=torch.float64))
    assert ea.RotaryTable.with_sections(16, [4, 2, 2], interleaved=True, device="cpu").axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    g = ea.RotaryTable.grid(16, 2, theta=100.0, device="cpu")
    assert g.axis.tolist() == [0] * 4 + [1] * 4 and g.inv_freq.tolist() == [100.0 ** (-j / 4) for j in range(4)] * 2
    p = ea.RotaryTable.with_sections(16, [3], rot_dim=6, device="cpu")
    assert p.pairs == 3 and p.head_dim == 16
    with pytest.raises(ValueError, match="add up"):
        ea.RotaryTable.with_sections(16, [4, 4, 4], device="cpu")
    with pytest.raises(ValueError, match="divide"):
        ea.RotaryTable.grid(12, 4, device="cpu")
    with pytest.raises(ValueError, match="fit a head"):
        ea.RotaryTable([1.0] * 9, head_dim=16, device="cpu")
    with pytest.raises(ValueError, match="below 0"):
        ea.RotaryTable([1.0, 1.0], [0, -1], head_dim=16, device="cpu")
    with pytest.raises(ValueError, match="axes of shape"):
        ea.RotaryTable([1.0, 1.0], [0], head_dim=16, device="cpu")
    with pytest.raises(ValueError, match="pairing"):
        ea.RotaryTable([1.0], head_dim=16, pairing="x", device="cpu")
    with pytest.raises(ValueError, match="finite"):
        ea.RotaryTable([1.0], head_dim=16, scale=math.nan, device="cpu")


def test_the_c_entries_refuse_bad_structs_before_any_launch():
    """MV_ERR_INVALID and a message, with no device in reach: sizes, types, alignment and missing pointers are checked on the host."""
    L = _lib.lib()

    def attn(**kw):
        p = _lib.AttnC()
        base = dict(q=16, k=16, v=16, out=16, dtype=_lib.MV_BF16, batch=1, rows=1, keys=1, heads=2, kv_heads=1, dim=16, scale=0.25)
        for n, x in {**base, **kw}.items():
            setattr(p, n, x)
        return L.mv_enc_attention(0, C.byref(p), None), L.mv_last_error().decode()

    assert attn(batch=0)[0] == 0 and attn(rows=0)[0] == 0  # nothing to do is no error
    for kw in (dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(batch=-1), dict(keys=-1), dict(keys=0x7FFFF001), dict(dtype=_lib.MV_F32), dict(dim=20),
               dict(dim=0), dict(dim=264), dict(scale=0.0), dict(scale=math.inf), dict(softcap=-1.0), dict(q=0), dict(k=8), dict(out=20),
               dict(q_row=4), dict(v_head=12), dict(ranges=4), dict(ranges=8, ranges_batch=3), dict(rows=0x7FFFFFFF, heads=4096, kv_heads=1)):
        rc, msg = attn(**kw)
        assert rc == -1 and msg.startswith("mv_enc_attention"), (kw, rc, msg)
    assert L.mv_enc_attention(0, None, None) == -1

    def rot(**kw):
        p = _lib.RotaryC()
        base = dict(q=16, k=16, q_out=16, k_out=16, dtype=_lib.MV_BF16, batch=1, rows=1, heads=2, kv_heads=1, dim=16, pairs=8, positions=16, inv_freq=16, axis=16)
        for n, x in {**base, **kw}.items():
            setattr(p, n, x)
        return L.mv_enc_rotary(0, C.byref(p), None), L.mv_last_error().decode()

    assert rot(rows=0)[0] == 0 and rot(heads=0, kv_heads=0)[0] == 0
    for kw in (dict(pairs=9), dict(pairs=-1), dict(dim=0), dict(dim=8192), dict(dtype=7), dict(q=0), dict(k_out=0), dict(positions=0), dict(inv_freq=0),
               dict(axis=0), dict(cos=16), dict(cos=16, sin=16), dict(q=17), dict(rows=0x7FFFFFFF, batch=0x7FFFFFFF, heads=64)):
        rc, msg = rot(**kw)
        assert rc == -1 and msg.startswith("mv_enc_rotary"), (kw, rc, msg)
    assert L.mv_enc_rotary(0, None, None) == -1
    assert L.mv_enc_padded_ranges(0, None, 1, None, 1, None, -1, 2, 3, 0, None, None) == -1
    assert L.mv_enc_padded_ranges(0, None, 1, None, 1, None, -1, 0, 3, 0, None, None) == 0
    assert L.mv_enc_document_ranges(0, None, 1, None, -1, 3, None, None) == -1
    assert L.mv_enc_document_ranges(0, None, 1, None, -1, 0, None, None) == 0


def test_calls_of_more_threads_than_a_launch_holds_are_refused():
    """2^32 threads and more: a refusal of the entry's own, not the launch's error."""
    L = _lib.lib()
    p = _lib.AttnC(q=16, k=16, v=16, out=16, dtype=_lib.MV_BF16, batch=65536, rows=1, keys=1, heads=128, kv_heads=128, dim=8, scale=1.0)
    assert L.mv_enc_attention(0, C.byref(p), None) == -1 and "too many rows" in L.mv_last_error().decode()
    r = _lib.RotaryC(q=16, k=16, q_out=16, k_out=16, dtype=_lib.MV_BF16, batch=2, rows=0x7FFFFFFF, heads=2, kv_heads=1, dim=16, pairs=8, positions=16, inv_freq=16, axis=16)
    assert L.mv_enc_rotary(0, C.byref(r), None) == -1 and "too many tokens" in L.mv_last_error().decode()
    assert L.mv_enc_padded_ranges(0, 16, 1, 16, 1, None, -1, 3, 0x7FFFFFFF, 0, 16, None) == -1 and "too many rows" in L.mv_last_error().decode()


def test_scales_that_leave_32_bits_are_refused():
    q, k, v = qkv()
    with pytest.raises(ValueError, match="scale"):
        ea.attention(q, k, v, scale=1e39)
    with pytest.raises(ValueError, match="softcap"):
        ea.attention(q, k, v, softcap=1e39)
    with pytest.raises(ValueError, match="finite"):
        ea.RotaryTable([1.0], head_dim=16, scale=1e39, device="cpu")
    for scale, cap in ((3e38, 0.0), (3e38, 1e-3), (1e-30, 1e30), (1.0, 3e38)):  # in range themselves, but not scale * log2(e), scale / cap or cap * log2(e)
        p = _lib.AttnC(q=16, k=16, v=16, out=16, dtype=_lib.MV_BF16, batch=1, rows=1, keys=1, heads=2, kv_heads=1, dim=16, scale=scale, softcap=cap)
        assert _lib.lib().mv_enc_attention(0, C.byref(p), None) == -1 and "32 bits" in _lib.lib().mv_last_error().decode()


def test_the_structs_are_laid_out_as_the_header_declares_them(tmp_path):
    """sizeof and the last field's offset, from a C compiler over include/mvmaxsim.h."""
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mvmaxsim.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(mv_attn), '
                   "offsetof(mv_attn, softcap), offsetof(mv_attn, dtype), sizeof(mv_rotary), offsetof(mv_rotary, pairs), offsetof(mv_rotary, scale));return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    A, R = _lib.AttnC, _lib.RotaryC
    assert got == [C.sizeof(A), A.softcap.offset, A.dtype.offset, C.sizeof(R), R.pairs.offset, R.scale.offset]


HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_the_attention_kernels_keep_the_wait_states_of_their_matrix_results(tmp_path):
    """The listing of csrc/mv_attention.hip under its own build flags: along no path does a VALU instruction touch an MFMA's result fewer than 7 issue
    slots behind it (tools/mfma_hazard_scan.py), and none of the packed fp32 instructions is there."""
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import mfma_hazard_scan as hz

    csrc = os.path.join(ROOT, "morphik-core_amd", "csrc")
    out = str(tmp_path / "mv_attention.s")
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-ffp-contract=off", "-fno-fast-math", "-I" + os.path.join(ROOT, "include"),
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form=1"]
    subprocess.run([HIPCC] + flags + ["-S", "--offload-device-only", os.path.join(csrc, "mv_attention.hip"), "-o", out], check=True, capture_output=True, timeout=900)
    kernels = hz.parse(out)
    found = [(ws, m, c) for ins in kernels.values() for ws, m, c in hz.scan(ins)]
    assert found
    for ws, mfma, consumer in found:
        assert ws >= 7, f"`{consumer}` reads the result of `{mfma}` {ws} issue slots behind it"
    text = open(out).read()
    for name in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"):
        assert name not in text
    shutil.rmtree(tmp_path, ignore_errors=True)


def _outputs(model, batches):
    with torch.inference_mode():
        return [model(**b).embeddings.clone() for b in batches]


@pytest.mark.parametrize("preset", ["colpali", "tiny", "tiny-2.5"])
def test_patched_attention_leaves_a_model_without_a_gpu_exactly_as_it_was(preset):
    """patch_attention on a CPU model: every rotary, decoder and packed module is found, and each falls back to its own forward (the attention function to
    the framework's): bit-identical outputs, before, between and after; patching twice does nothing."""
    ids = torch.tensor([[1, 5, 9, 3, 2], [1, 7, 0, 0, 0]])
    batches = [dict(input_ids=ids, attention_mask=torch.ones_like(ids)), dict(input_ids=ids, attention_mask=(ids > 0).long())]
    if preset == "colpali":
        from morphik_core_amd.embedding import MI355XColpaliEmbeddingModel

        emb = MI355XColpaliEmbeddingModel(preset="tiny", device="cpu", seed=3)
        assert emb.fused_attention == {"rotary": 0, "decoder": 0, "packed": 0}  # never without a GPU
        model, want_counts = emb.model, {"rotary": 1, "decoder": 2, "packed": 0}
        pv = torch.rand(1, 3, 56, 56, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        batches.append(dict(input_ids=torch.tensor([[1023] * 16 + [1, 4, 2]]), attention_mask=torch.ones(1, 19, dtype=torch.long), pixel_values=pv))
    else:
        import numpy as np

        from morphik_core_amd.colqwen_embedding import build_random_colqwen2
        from tests import offline_assets as oa

        proc, tokens = oa.colqwen2_processor()
        model, want_counts = build_random_colqwen2(preset, tokens, "cpu", torch.bfloat16), {"rotary": 1, "decoder": 2, "packed": 2}
        rng = np.random.default_rng(0)
        b = proc(images=[oa.page_image(rng, 60, 60), oa.page_image(rng, 112, 84)], return_tensors="pt")
        batches.append({k: b[k].to(torch.bfloat16) if k == "pixel_values" else b[k] for k in ("input_ids", "attention_mask", "pixel_values", "image_grid_thw")})
    before = [name for _, name in ea._implementations(model)]
    want = _outputs(model, batches)
    assert ea.patch_attention(model) == want_counts
    assert ea.patch_attention(model) == {"rotary": 0, "decoder": 0, "packed": 0}
    assert {name for _, name in ea._implementations(model)} == {"mv_key_ranges"}
    assert all(torch.equal(a, b) for a, b in zip(_outputs(model, batches), want))
    ea.unpatch_attention(model)
    assert [name for _, name in ea._implementations(model)] == before and not any(hasattr(m, "_mv_attn_forward") or hasattr(m, "_mv_rotary_table") for m in model.modules())
    assert all(torch.equal(a, b) for a, b in zip(_outputs(model, batches), want))
    ea.unpatch_attention(model)


def test_the_attention_function_turns_ranges_back_into_a_mask_where_the_kernel_does_not_apply():
    class Module(torch.nn.Module):
        is_causal = True
        num_key_value_groups = 2

    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(2, h, 5, 16, generator=g) for h in (4, 2, 2))
    r = torch.tensor([[[0, 1], [0, 2], [0, 3], [1, 4], [0, 5]], [[2, 5], [2, 3], [0, 5], [0, 5], [4, 5]]], dtype=torch.int32)
    m = torch.zeros(2, 1, 5, 5, dtype=torch.bool)
    for b in range(2):
        for i, (lo, hi) in enumerate(r[b].tolist()):
            m[b, 0, i, lo:hi] = True
    from transformers import AttentionInterface

    want = AttentionInterface()["sdpa"](Module(), q, k, v, m, scaling=0.25, dropout=0.0)[0]
    got = ea._interface_attention(Module(), q, k, v, r[:, None], scaling=0.25)[0]
    assert torch.equal(got, want)
