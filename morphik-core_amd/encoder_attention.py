"""The attention half of the encoder blocks as hand-written HIP kernels (csrc/mv_rotary.hip, csrc/mv_attention.hip): rotary positions with
several axes and attention over key ranges, which the SigLIP / Gemma (ColPali) and Qwen2-VL / Qwen2.5-VL (ColQwen2) blocks use one behind the
other.  The reference formulation is `model(**processor(x))` under bf16 autocast (core/embedding/colpali_embedding_model.py:251-262, 275-305).

  table = RotaryTable.with_sections(128, [22, 21, 21], theta=1e6)     # once per model: frequency and axis of every pair
  q, k = rotary(q, k, positions, table)                               # positions [3, batch, rows]: time, height, width
  ranges = padded_ranges(starts, ends, rows, prefix=1024)             # once per forward: the keys that each row sees
  out = attention(q, k, v, key_ranges=ranges)                         # [batch, rows, heads, dim]

Every mask these encoders use is a range of keys per row -- padding on either side, causal, a prefix that sees itself, documents or
windows packed one behind the other -- so that is the one form of mask here: `padded_ranges` and `document_ranges` make the usual ones on the
device, `ranges_from_mask` takes a boolean mask.  A row whose range is empty gets zeros, and what keys outside a row's range hold (NaN and
infinity included) does not reach the row.

Everything is enqueued on torch's current stream of the tensors' device, allocates through torch only, keeps nothing between calls and may be
captured into a graph.  These are inference operators, as the encoders run them: nothing here has a gradient, and tensors that would need one
are refused.  There is no CPU path: tensors off the GPU are refused.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from typing import Any, Optional, Sequence, Tuple

from . import _lib

_PAIRINGS = ("halves", "adjacent")
_FORMATS = {C.c_void_p: "P", C.c_int64: "q", C.c_int32: "i", C.c_float: "f"}


def _packer(cls) -> struct.Struct:
    """The C struct's layout as a struct.Struct (a call packs its operands in one go: setting them field by field costs as long as a small kernel)."""
    return struct.Struct("@" + "".join(_FORMATS[t] for _, t in cls._fields_))


_PACK_ATTN, _PACK_ROTARY = _packer(_lib.AttnC), _packer(_lib.RotaryC)
_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


def _dtype_code(torch, dtype, what: str, fp32: bool) -> int:
    if dtype is torch.bfloat16:
        return _lib.MV_BF16
    if dtype is torch.float16:
        return _lib.MV_F16
    if fp32 and dtype is torch.float32:
        return _lib.MV_F32
    raise ValueError(f"{what}: dtype {dtype} (bfloat16{', float16 or float32' if fp32 else ' or float16'})")


def _device_index(torch, what: str, *tensors: Any) -> int:
    """All on one GPU, none that autograd would follow.  -> its index"""
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a GPU (there is no CPU path)")
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t.device != device:
            raise ValueError(f"{what}: tensors on different devices ({device}, {t.device})")
        if grad and t.requires_grad:
            raise ValueError(f"{what}: has no gradient (run it under torch.inference_mode() or torch.no_grad())")
    return device.index


def _stream(torch, index: int) -> int:
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle without the Stream object around it (1 us less)
    return raw(index) if raw is not None else torch.cuda.current_stream(index).cuda_stream


def _heads4(t: Any, what: str, name: str) -> Any:
    """[batch, rows, heads, dim]; [rows, heads, dim] counts as one batch entry."""
    n = t.dim()
    if n == 4:
        return t
    if n == 3:
        return t.unsqueeze(0)
    raise ValueError(f"{what}: {name} must be [batch, rows, heads, dim] or [rows, heads, dim], not {tuple(t.shape)}")


# --------------------------------------------------------------------------- rotary positions
class RotaryTable:
    """Frequency and axis of every pair of a head: what stays the same from call to call.

    inv_freq [pairs] (any float type, kept in 64 bits), axes [pairs] whole numbers (None: one axis for all), head_dim the width of a head, of
    which the first 2 * pairs elements turn; pairing "halves": elements (j, j + pairs) are a pair, "adjacent": (2 j, 2 j + 1); scale multiplies the
    turned elements (the attention factor of some long-context schemes)."""

    def __init__(self, inv_freq: Any, axes: Any = None, *, head_dim: int, pairing: str = "halves", scale: float = 1.0, device: Any = None):
        torch = _torch()
        freq = inv_freq if torch.is_tensor(inv_freq) else torch.tensor(inv_freq, dtype=torch.float64)
        if freq.dim() != 1:
            raise ValueError(f"RotaryTable: inv_freq must be one row of frequencies, not {tuple(freq.shape)}")
        if device is None:
            device = freq.device if freq.is_cuda else torch.device("cuda", torch.cuda.current_device())
        pairs = int(freq.shape[0])
        host = torch.zeros(pairs, dtype=torch.int64) if axes is None else torch.as_tensor(axes).to("cpu", torch.int64)
        if host.shape != (pairs,):
            raise ValueError(f"RotaryTable: {pairs} frequencies but axes of shape {tuple(host.shape)}")
        if pairs and int(host.min()) < 0:
            raise ValueError("RotaryTable: an axis below 0")
        if not 1 <= head_dim <= 4096 or 2 * pairs > head_dim:
            raise ValueError(f"RotaryTable: {pairs} pairs do not fit a head of {head_dim} (at most 4096)")
        if pairing not in _PAIRINGS:
            raise ValueError(f"RotaryTable: pairing {pairing!r} (one of {_PAIRINGS})")
        if not math.isfinite(scale):
            raise ValueError("RotaryTable: scale must be finite")
        self.head_dim, self.pairs, self.pairing, self.scale = int(head_dim), pairs, pairing, float(scale)
        self.axes = int(host.max()) + 1 if pairs else 0  # axes that positions must have at least
        self.inv_freq = freq.to(device=device, dtype=torch.float64).contiguous()
        self.axis = host.to(device=device, dtype=torch.int32)

    @classmethod
    def with_sections(cls, head_dim: int, sections: Sequence[int], *, theta: float = 10000.0, rot_dim: Optional[int] = None, interleaved: bool = False,
                      **kwargs: Any) -> "RotaryTable":
        """One run of frequencies theta^(-j / pairs) over rot_dim (default: head_dim); sections = pairs of each axis, one after the other, or dealt out
        in turn (`interleaved`: 0, 1, 2, 0, 1, 2, ... until an axis has its share)."""
        pairs = (head_dim if rot_dim is None else rot_dim) // 2
        sections = [int(s) for s in sections]
        if min(sections, default=0) < 0 or sum(sections) != pairs:
            raise ValueError(f"RotaryTable: sections {sections} must add up to {pairs} pairs")
        if interleaved:
            left, axes = list(sections), []
            while len(axes) < pairs:
                for a, n in enumerate(left):
                    if n:
                        axes.append(a)
                        left[a] = n - 1
        else:
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
        return cls([theta ** (-j / pairs) for j in range(pairs)], axes, head_dim=head_dim, **kwargs)

    @classmethod
    def grid(cls, head_dim: int, axes: int = 2, *, theta: float = 10000.0, **kwargs: Any) -> "RotaryTable":
        """Vision towers: every axis (height, width) runs through its own frequencies from the start, over an equal share of the pairs."""
        pairs = head_dim // 2
        if axes < 1 or pairs % axes:
            raise ValueError(f"RotaryTable: {pairs} pairs do not divide by {axes} axes")
        share = pairs // axes
        return cls([theta ** (-j / share) for j in range(share)] * axes, [a for a in range(axes) for _ in range(share)], head_dim=head_dim, **kwargs)


def _rotary_operands(torch, what, q, k, in_place):
    """-> (q and k as [batch, rows, heads, dim] or None, outputs in that form, outputs as the caller shaped them)"""
    first = q if q is not None else k
    if first is None:
        raise ValueError(f"{what}: neither q nor k")
    ins, outs, shaped = [], [], []
    for n, t in (("q", q), ("k", k)):
        if t is None:
            ins.append(None), outs.append(None), shaped.append(None)
            continue
        x = _heads4(t, what, n)
        st = x.stride()
        if st[3] != 1 and x.shape[3] > 1 and x.numel():
            raise ValueError(f"{what}: the elements of a head of {n} must lie next to each other")
        if in_place:
            if _overlaps(x):
                raise ValueError(f"{what}: {n} cannot be turned in place, its heads or rows share memory")
            out = x
        else:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        ins.append(x), outs.append(out), shaped.append(t if in_place else out if x is t else out.view(t.shape))
    if q is not None and k is not None:
        a, b = ins[0].shape, ins[1].shape
        if q.dtype is not k.dtype or a[:2] != b[:2] or a[3] != b[3]:
            raise ValueError(f"{what}: q and k differ in type, batch, rows or head width ({tuple(a)} {q.dtype}, {tuple(b)} {k.dtype})")
        if in_place and _share_memory(*ins):
            raise ValueError(f"{what}: q and k cannot be turned in place, they share memory")
    return ins, outs, tuple(shaped)


_NO_STRIDES = (0, 0, 0)


def _launch_rotary(torch, what, ins, outs, first, index, pos, pos_strides, freq, axis, cos, sin, table_strides, scale, adjacent, pairs):
    (q, k), (qo, ko) = ins, outs
    batch, rows, _, dim = first.shape
    code = _dtype_code(torch, first.dtype, what, fp32=True)
    packed = _PACK_ROTARY.pack(
        *(0 if t is None else t.data_ptr() for t in (q, k, qo, ko)),
        *(st for t in (q, k, qo, ko) for st in (_NO_STRIDES if t is None else t.stride()[:3])),
        0 if pos is None else pos.data_ptr(), *pos_strides, freq, axis, cos, sin, *table_strides, scale, code,
        int(pos is not None and pos.dtype is torch.int64), adjacent, batch, rows, 0 if q is None else q.shape[2], 0 if k is None else k.shape[2], dim, pairs)
    _lib.check(_lib.lib().mv_enc_rotary(index, packed, _stream(torch, index)))


def _extent(x) -> Tuple[int, int]:
    n = x.element_size() * (1 + sum((s - 1) * st for s, st in zip(x.shape, x.stride())))
    return x.data_ptr(), x.data_ptr() + n


def _overlaps(x) -> bool:
    """Whether two elements of x can share memory: sorted by stride, every dimension must step past all that lies below it."""
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(x.stride(), x.shape) if n > 1):
        if st <= reach:
            return True
        reach += st * (n - 1)
    return False


def _share_memory(a, b) -> bool:
    """Conservative but for views of one buffer whose heads lie side by side in its rows (a fused projection)."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.stride()[:2] == b.stride()[:2]:
        # the same rows of one buffer: apart if their windows within a row's step do not meet, seen from the lower one
        size = a.element_size()
        lo, hi = (a, b) if a0 <= b0 else (b, a)
        gap = (hi.data_ptr() - lo.data_ptr()) // size
        width = [1 + sum((n - 1) * st for n, st in zip(x.shape[2:], x.stride()[2:])) for x in (lo, hi)]
        step = min((st for st, n in zip(a.stride()[:2], a.shape[:2]) if n > 1), default=None)
        if gap >= width[0] and (step is None or gap + width[1] <= step):
            return False
    return True


def rotary(q: Any, k: Any, positions: Any, table: RotaryTable, *, in_place: bool = False) -> Tuple[Any, Any]:
    """Turn q [batch, rows, heads, dim] and k [batch, rows, kv_heads, dim] (or [rows, heads, dim]; either may be None) to their positions:
    pair j by positions[axis_j] * inv_freq_j.  positions: whole numbers, int32 or int64, [axes, batch, rows] (axes and batch may be left out where
    there is one of them; a batch of 1 serves all).  float32, bfloat16 or float16, any strides with the elements of a head side by side.
    -> (q, k): new contiguous tensors, or the inputs themselves with `in_place`."""
    torch = _torch()
    what = "rotary"
    if not isinstance(table, RotaryTable):
        raise ValueError(f"{what}: table must be a RotaryTable")
    ins, outs, shaped = _rotary_operands(torch, what, q, k, in_place)
    first = ins[0] if ins[0] is not None else ins[1]
    _dtype_code(torch, first.dtype, what, fp32=True)
    batch, rows, _, dim = first.shape
    if dim != table.head_dim:
        raise ValueError(f"{what}: heads of {dim}, the table is for {table.head_dim}")
    if positions.dtype is not torch.int64 and positions.dtype is not torch.int32:
        raise ValueError(f"{what}: positions must be int32 or int64, not {positions.dtype}")
    n = positions.dim()
    if n == 3:
        pos = positions
    elif n == 2:  # [axes, rows] of packed rows where q has no batch, [batch, rows] of one axis where it has
        pos = positions[:, None] if (q if q is not None else k).dim() == 3 else positions[None]
    else:
        pos = positions[None, None] if n == 1 else positions
    if pos.dim() != 3 or pos.shape[1] not in (1, batch) or pos.shape[2] != rows:
        raise ValueError(f"{what}: positions {tuple(positions.shape)} do not fit {batch} x {rows} rows")
    if pos.shape[0] < table.axes:
        raise ValueError(f"{what}: positions have {pos.shape[0]} axes, the table needs {table.axes}")
    index = _device_index(torch, what, first, *([ins[1]] if ins[1] is not None else []), pos, table.inv_freq)
    st = pos.stride()
    _launch_rotary(torch, what, ins, outs, first, index, pos, (st[0], st[1] if pos.shape[1] == batch else 0, st[2]), table.inv_freq.data_ptr(),
                   table.axis.data_ptr(), 0, 0, _NO_STRIDES, table.scale, int(table.pairing == "adjacent"), table.pairs)
    return shaped


def rotary_tables(q: Any, k: Any, cos: Any, sin: Any, *, pairing: str = "halves", in_place: bool = False) -> Tuple[Any, Any]:
    """`rotary` with the angles given as cosines and sines, float32 [batch, rows, pairs] (batch may be left out or 1; any strides), as a model
    computes them once for all its blocks."""
    torch = _torch()
    what = "rotary_tables"
    if pairing not in _PAIRINGS:
        raise ValueError(f"{what}: pairing {pairing!r} (one of {_PAIRINGS})")
    ins, outs, shaped = _rotary_operands(torch, what, q, k, in_place)
    first = ins[0] if ins[0] is not None else ins[1]
    _dtype_code(torch, first.dtype, what, fp32=True)
    batch, rows, _, dim = first.shape
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f"{what}: cos and sin must be float32")
    if cos.shape != sin.shape or cos.stride() != sin.stride():
        raise ValueError(f"{what}: cos and sin differ in shape or strides")
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    if cos.dim() != 3 or cos.shape[0] not in (1, batch) or cos.shape[1] != rows or not 0 < 2 * cos.shape[2] <= dim <= 4096:
        raise ValueError(f"{what}: cos of {tuple(cos.shape)} does not fit {batch} x {rows} rows of heads of {dim} (at most 4096)")
    index = _device_index(torch, what, first, *([ins[1]] if ins[1] is not None else []), cos, sin)
    st = cos.stride()
    _launch_rotary(torch, what, ins, outs, first, index, None, _NO_STRIDES, 0, 0, cos.data_ptr(), sin.data_ptr(),
                   (st[0] if cos.shape[0] == batch else 0, st[1], st[2]), 1.0, int(pairing == "adjacent"), cos.shape[2])
    return shaped


# --------------------------------------------------------------------------- key ranges
def _prefix(torch, what, prefix, n, device):
    """-> (pointer or None, scalar)"""
    if prefix is None:
        return None, -1
    if isinstance(prefix, int):
        if prefix < 0:
            raise ValueError(f"{what}: prefix must not be negative (None: rows see their whole sequence)")
        return None, min(prefix, 0x7FFFFFFF)
    if prefix.dtype != torch.int32 or prefix.shape != (n,) or prefix.device != device or not prefix.is_contiguous():
        raise ValueError(f"{what}: prefix must be a number or contiguous int32 [{n}] on {device}")
    return prefix.data_ptr(), 0


def padded_ranges(starts: Any, ends: Any, rows: int, *, prefix: Any = None, row_offset: int = 0) -> Any:
    """Key ranges of a padded batch: entry b's sequence is the keys [starts[b], ends[b]) (int32 on the GPU); row i stands at i + row_offset (keys in
    front of the rows: a cache).  prefix None: a row sees its whole sequence; a number or int32 [batch]: the first `prefix` keys of it and those up to
    itself (0: causal).  Rows outside their sequence see nothing.  -> int32 [batch, rows, 2] for `attention`."""
    torch = _torch()
    what = "padded_ranges"
    if starts.dtype != torch.int32 or ends.dtype != torch.int32 or starts.dim() != 1 or starts.shape != ends.shape:
        raise ValueError(f"{what}: starts and ends must be int32, one entry per sequence")
    if not 0 <= rows <= 0x7FFFFFFF or row_offset < 0:
        raise ValueError(f"{what}: rows and row_offset must not be negative")
    ptr, scalar = _prefix(torch, what, prefix, starts.shape[0], starts.device)
    index = _device_index(torch, what, starts, ends)
    out = torch.empty((starts.shape[0], rows, 2), dtype=torch.int32, device=starts.device)
    _lib.check(_lib.lib().mv_enc_padded_ranges(index, starts.data_ptr(), starts.stride(0), ends.data_ptr(), ends.stride(0), ptr, scalar, starts.shape[0],
                                               rows, row_offset, out.data_ptr(), _stream(torch, index)))
    return out


def document_ranges(offsets: Any, rows: int, *, prefix: Any = None) -> Any:
    """Key ranges of documents packed one behind the other: document s is the rows [offsets[s], offsets[s + 1]), offsets int32 [documents + 1] on
    the GPU, ascending; rows before the first or behind the last document see nothing.  prefix as in `padded_ranges`, per document.
    -> int32 [1, rows, 2] for `attention`."""
    torch = _torch()
    what = "document_ranges"
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous():
        raise ValueError(f"{what}: offsets must be contiguous int32 [documents + 1]")
    if not 0 <= rows <= 0x7FFFFFFF:
        raise ValueError(f"{what}: rows must not be negative")
    docs = offsets.shape[0] - 1
    ptr, scalar = _prefix(torch, what, prefix, docs, offsets.device)
    index = _device_index(torch, what, offsets)
    out = torch.empty((1, rows, 2), dtype=torch.int32, device=offsets.device)
    _lib.check(_lib.lib().mv_enc_document_ranges(index, offsets.data_ptr(), docs, ptr, scalar, rows, out.data_ptr(), _stream(torch, index)))
    return out


def ranges_from_mask(mask: Any) -> Tuple[Any, Any]:
    """Boolean mask [batch, rows, keys] (True: the row sees the key) -> (int32 ranges [batch, rows, 2], a truth value on the device: whether every
    row's keys are one run, so that the ranges say the same as the mask)."""
    torch = _torch()
    if mask.dtype != torch.bool or mask.dim() != 3:
        raise ValueError(f"ranges_from_mask: a boolean [batch, rows, keys], not {mask.dtype} {tuple(mask.shape)}")
    batch, rows, keys = mask.shape
    if keys == 0:
        return torch.zeros((batch, rows, 2), dtype=torch.int32, device=mask.device), torch.ones((), dtype=torch.bool, device=mask.device)
    bits = mask.to(torch.uint8)
    lo = bits.argmax(-1).to(torch.int32)
    hi = keys - bits.flip(-1).argmax(-1).to(torch.int32)
    count = mask.sum(-1, dtype=torch.int32)
    seen = count > 0
    lo, hi = torch.where(seen, lo, 0), torch.where(seen, hi, 0)
    return torch.stack([lo, hi], -1), (hi - lo == count).all()


# --------------------------------------------------------------------------- attention
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index: int, *sizes: int) -> int:
    n = _lib.lib().mv_enc_attention_workspace_bytes(index, *sizes)
    if n < 0:
        _lib.check(int(n))
    return int(n)


def attention(q: Any, k: Any, v: Any, *, key_ranges: Any = None, scale: Optional[float] = None, softcap: float = 0.0) -> Any:
    """Softmax attention of q [batch, rows, heads, dim] over k, v [batch, keys, kv_heads, dim] (or [rows, heads, dim] of packed documents), heads
    a multiple of kv_heads.  key_ranges int32 [batch or 1, rows, 2]: row i sees the keys [lo, hi), cut to what there is; an empty range gives
    zeros; None: every key.  scale defaults to dim ** -0.5; softcap c > 0 caps scores to c * tanh(score / c).  bfloat16 or float16; dim a multiple
    of 8 up to 256; any strides that are multiples of 8 with the elements of a head side by side, 16-byte aligned.
    -> new contiguous tensor of q's shape."""
    torch = _torch()
    what = "attention"
    shape = q.shape
    code = _dtype_code(torch, q.dtype, what, fp32=False)
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"{what}: q, k and v differ in type ({q.dtype}, {k.dtype}, {v.dtype})")
    q, k, v = _heads4(q, what, "q"), _heads4(k, what, "k"), _heads4(v, what, "v")
    batch, rows, heads, dim = q.shape
    k_shape = k.shape
    k_batch, keys, kv_heads, k_dim = k_shape
    if k_shape != v.shape or k_batch != batch or k_dim != dim:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k_shape)} and v {tuple(v.shape)} do not fit")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{what}: {heads} heads over {kv_heads} K/V heads (a multiple)")
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError(f"{what}: heads of {dim} (multiples of 8 up to 256)")
    scale = dim**-0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite")
    if not (softcap >= 0 and math.isfinite(softcap)):
        raise ValueError(f"{what}: softcap must not be negative (0: no cap)")
    pointers, strides = [], []
    for name, t, sizes in (("q", q, q.shape), ("k", k, k_shape), ("v", v, k_shape)):
        st, at = t.stride(), t.data_ptr()
        if (st[3] != 1 or at & 15 or (st[0] | st[1] | st[2]) & 7) and t.numel():
            # a dimension of one entry has no step
            st = tuple(0 if n == 1 else x for n, x in zip(sizes, st[:3])) + (st[3],)
            if st[3] != 1 or at & 15 or (st[0] | st[1] | st[2]) & 7:
                raise ValueError(f"{what}: {name} must be 16-byte aligned, strides multiples of 8, the elements of a head side by side")
        pointers.append(at)
        strides += st[:3]
    if key_ranges is not None:
        if key_ranges.dtype is not torch.int32 or key_ranges.dim() != 3 or key_ranges.shape[0] not in (1, batch) or tuple(key_ranges.shape[1:]) != (rows, 2):
            raise ValueError(f"{what}: key_ranges must be int32 [{batch} or 1, {rows}, 2], not {key_ranges.dtype} {tuple(key_ranges.shape)}")
        index = _device_index(torch, what, q, k, v, key_ranges)
        if not key_ranges.is_contiguous() or key_ranges.data_ptr() & 7:
            key_ranges = key_ranges.clone(memory_format=torch.contiguous_format)
        ranges, ranges_batch = key_ranges.data_ptr(), 0 if key_ranges.shape[0] == 1 else 2 * rows
    else:
        index = _device_index(torch, what, q, k, v)
        ranges = ranges_batch = 0
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if batch and rows:
        need = _workspace_bytes(index, batch, rows, keys, heads, kv_heads, dim)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None  # torch's own reuse rules keep it this call's on this stream
        packed = _PACK_ATTN.pack(*pointers, out.data_ptr(), ranges, *strides, ranges_batch, work.data_ptr() if need else 0, need, code, batch, rows, keys, heads, kv_heads, dim, scale, softcap)
        _lib.check(_lib.lib().mv_enc_attention(index, packed, _stream(torch, index)))
    return out if len(shape) == 4 else out.view(shape)
