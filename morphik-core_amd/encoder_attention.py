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
(in either mode of autograd) are refused.  There is no CPU path: tensors off the GPU are refused.
"""
from __future__ import annotations

import ctypes as C
import functools
import logging
import math
import os
import struct
import types
from typing import Any, Dict, Optional, Sequence, Tuple

from . import _lib

logger = logging.getLogger(__name__)

_PAIRINGS = ("halves", "adjacent")
_FP32_MAX = 2.0**128 - 2.0**104
_MAX_ROW_STRIDE = 1 << 23  # of k and v, in elements
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
    index = tensors[0].get_device()
    if index < 0:
        raise ValueError(f"{what}: tensors must be on a GPU (there is no CPU path)")
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"{what}: tensors on different devices ({tensors[0].device}, {t.device})")
    _refuse_derivatives(torch, what, tensors)
    return index


def _refuse_derivatives(torch, what: str, tensors: Sequence[Any]) -> None:
    """Neither mode of autograd follows these operators: a tensor that it would follow is refused, not dropped from the derivative."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise ValueError(f"{what}: has no gradient (run it under torch.inference_mode() or torch.no_grad())")
    forward = torch.autograd.forward_ad
    if getattr(forward, "_current_level", 0) >= 0 and torch._C._is_fwd_grad_enabled():  # inside a dual level only: asking costs 1 us a tensor
        for t in tensors:
            if forward.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what}: has no gradient (an operand carries a forward-mode tangent)")


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
        if not abs(scale) < _FP32_MAX:
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


def _rotary_operands(what, q, k, in_place):
    """-> (q, k as [batch, rows, heads, dim] or None, their outputs, the outputs as the caller shaped them, the first of q and k)"""
    torch = _torch()
    x = x_out = q_out = y = y_out = k_out = None
    if q is not None:
        x, x_out, q_out = _rotary_operand(torch, what, "q", q, in_place)
    if k is not None:
        y, y_out, k_out = _rotary_operand(torch, what, "k", k, in_place)
        if x is not None:
            a, b = x.shape, y.shape
            if x.dtype is not y.dtype or a[0] != b[0] or a[1] != b[1] or a[3] != b[3]:
                raise ValueError(f"{what}: q and k differ in type, batch, rows or head width ({tuple(a)} {x.dtype}, {tuple(b)} {y.dtype})")
            if in_place and _share_memory(x, y):
                raise ValueError(f"{what}: q and k cannot be turned in place, they share memory")
    elif x is None:
        raise ValueError(f"{what}: neither q nor k")
    return x, y, x_out, y_out, (q_out, k_out), y if x is None else x


def _rotary_operand(torch, what, name, t, in_place):
    x = t if t.dim() == 4 else _heads4(t, what, name)
    if x.stride(3) != 1 and x.shape[3] > 1 and x.numel():
        raise ValueError(f"{what}: the elements of a head of {name} must lie next to each other")
    if not in_place:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        return x, out, out if x is t else out.view(t.shape)
    if _overlaps(x):
        raise ValueError(f"{what}: {name} cannot be turned in place, its heads or rows share memory")
    return x, x, t


_NO_STRIDES = (0, 0, 0)


def _launch_rotary(torch, what, q, k, qo, ko, index, code, positions, pos_strides, freq, axis, cos, sin, table_strides, scale, wide_positions, adjacent, pairs):
    heads = kv_heads = at_q = at_k = at_qo = at_ko = q0 = q1 = q2 = k0 = k1 = k2 = qo0 = qo1 = qo2 = ko0 = ko1 = ko2 = 0
    if q is not None:
        batch, rows, heads, dim = q.shape
        at_q, (q0, q1, q2, _) = q.data_ptr(), q.stride()
        at_qo, (qo0, qo1, qo2, _) = (at_q, (q0, q1, q2, 1)) if qo is q else (qo.data_ptr(), qo.stride())
    if k is not None:
        batch, rows, kv_heads, dim = k.shape
        at_k, (k0, k1, k2, _) = k.data_ptr(), k.stride()
        at_ko, (ko0, ko1, ko2, _) = (at_k, (k0, k1, k2, 1)) if ko is k else (ko.data_ptr(), ko.stride())
    p0, p1, p2 = pos_strides
    t0, t1, t2 = table_strides
    packed = _PACK_ROTARY.pack(at_q, at_k, at_qo, at_ko, q0, q1, q2, k0, k1, k2, qo0, qo1, qo2, ko0, ko1, ko2, positions, p0, p1, p2, freq, axis, cos, sin, t0, t1, t2, scale,
                               code, wide_positions, adjacent, batch, rows, heads, kv_heads, dim, pairs)
    _lib.check(_lib.lib().mv_enc_rotary(index, packed, _stream(torch, index)))


def _extent(x) -> Tuple[int, int]:
    at = x.data_ptr()
    n = x.numel() if x.is_contiguous() else 1 + sum((s - 1) * st for s, st in zip(x.shape, x.stride()))
    return at, at + n * x.element_size()


def _overlaps(x) -> bool:
    """Whether two elements of x can share memory: sorted by stride, every dimension must step past all that lies below it."""
    if x.is_contiguous():
        return False
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(x.stride(), x.shape) if n > 1):
        if st <= reach:
            return True
        reach += st * (n - 1)
    return False


def _share_memory(a, b) -> bool:
    """Conservative, but not for parts of one buffer: heads side by side in its rows (a fused projection), whatever the order of its dimensions."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a1 <= b0 or b1 <= a0:
        return False
    lo, hi = (a, b) if a0 <= b0 else (b, a)
    gap, rest = divmod(hi.data_ptr() - lo.data_ptr(), a.element_size())
    if rest:
        return True
    if a.stride()[:2] == b.stride()[:2] and a.shape[:2] == b.shape[:2]:
        # the same rows of one buffer: apart if their windows within a row's step do not meet, seen from the lower one
        width = [1 + sum((n - 1) * st for n, st in zip(x.shape[2:], x.stride()[2:])) for x in (lo, hi)]
        outer = sorted((st, n) for st, n in zip(a.stride()[:2], a.shape[:2]) if n > 1)
        nearest = min((st for st, _ in outer), default=None)  # of two rows' starts
        if len(outer) == 2:
            nearest = min(nearest, outer[1][0] - outer[0][0] * (outer[0][1] - 1))
        if gap >= width[0] and (nearest is None or gap + width[1] <= nearest):
            return False
    # boxes of one grid: with the same steps, `hi` starts some whole steps from `lo` in each dimension; where the box that holds both steps past itself, two
    # elements share memory only if all their places are the same, so one dimension in which the boxes do not meet is enough
    steps = []
    for st_l, n_l, st_h, n_h in zip(lo.stride(), lo.shape, hi.stride(), hi.shape):
        if n_l > 1 and n_h > 1 and st_l != st_h:
            return True
        if max(n_l, n_h) > 1:
            steps.append((st_l if n_l > 1 else st_h, n_l, n_h))
    reach, apart, left = 0, False, gap
    boxes = []
    for st, n_l, n_h in sorted(steps, reverse=True):
        at, left = divmod(left, st) if st else (0, left)
        boxes.append((st, max(n_l, at + n_h)))
        apart |= at >= n_l
    for st, n in reversed(boxes):
        if n > 1 and st <= reach:
            return True
        reach += st * (n - 1)
    return left != 0 or not apart


def rotary(q: Any, k: Any, positions: Any, table: RotaryTable, *, in_place: bool = False) -> Tuple[Any, Any]:
    """Turn q [batch, rows, heads, dim] and k [batch, rows, kv_heads, dim] (or [rows, heads, dim]; either may be None) to their positions:
    pair j by positions[axis_j] * inv_freq_j.  positions: whole numbers, int32 or int64, [axes, batch, rows] (axes and batch may be left out where
    there is one of them; a batch of 1 serves all).  float32, bfloat16 or float16, any strides with the elements of a head side by side.
    -> (q, k): new contiguous tensors, or the inputs themselves with `in_place`."""
    torch = _torch()
    what = "rotary"
    if not isinstance(table, RotaryTable):
        raise ValueError(f"{what}: table must be a RotaryTable")
    x, y, xo, yo, shaped, first = _rotary_operands(what, q, k, in_place)
    code = _dtype_code(torch, first.dtype, what, fp32=True)
    batch, rows, _, dim = first.shape
    if dim != table.head_dim:
        raise ValueError(f"{what}: heads of {dim}, the table is for {table.head_dim}")
    if positions.dtype is not torch.int64 and positions.dtype is not torch.int32:
        raise ValueError(f"{what}: positions must be int32 or int64, not {positions.dtype}")
    n = positions.dim()
    if n == 3:
        pos = positions
    elif n == 2:  # [axes, rows] of packed rows where q has no batch, [batch, rows] of one axis where it has
        pos = positions[:, None] if (k if q is None else q).dim() == 3 else positions[None]
    else:
        pos = positions[None, None] if n == 1 else positions
    p_shape = pos.shape
    if len(p_shape) != 3 or p_shape[1] not in (1, batch) or p_shape[2] != rows:
        raise ValueError(f"{what}: positions {tuple(positions.shape)} do not fit {batch} x {rows} rows")
    if p_shape[0] < table.axes:
        raise ValueError(f"{what}: positions have {p_shape[0]} axes, the table needs {table.axes}")
    index = _device_index(torch, what, first, pos, table.inv_freq, first if y is None else y)
    st = pos.stride()
    _launch_rotary(torch, what, x, y, xo, yo, index, code, pos.data_ptr(), (st[0], st[1] if p_shape[1] == batch else 0, st[2]), table.inv_freq.data_ptr(),
                   table.axis.data_ptr(), 0, 0, _NO_STRIDES, table.scale, int(pos.dtype is torch.int64), int(table.pairing == "adjacent"), table.pairs)
    return shaped


def rotary_tables(q: Any, k: Any, cos: Any, sin: Any, *, pairing: str = "halves", in_place: bool = False) -> Tuple[Any, Any]:
    """`rotary` with the angles given as cosines and sines, float32 [batch, rows, pairs] (batch may be left out or 1; any strides), as a model
    computes them once for all its blocks."""
    torch = _torch()
    what = "rotary_tables"
    if pairing not in _PAIRINGS:
        raise ValueError(f"{what}: pairing {pairing!r} (one of {_PAIRINGS})")
    x, y, xo, yo, shaped, first = _rotary_operands(what, q, k, in_place)
    code = _dtype_code(torch, first.dtype, what, fp32=True)
    batch, rows, _, dim = first.shape
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f"{what}: cos and sin must be float32")
    if cos.shape != sin.shape or cos.stride() != sin.stride():
        raise ValueError(f"{what}: cos and sin differ in shape or strides")
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    if cos.dim() != 3 or cos.shape[0] not in (1, batch) or cos.shape[1] != rows or not 0 < 2 * cos.shape[2] <= dim <= 4096:
        raise ValueError(f"{what}: cos of {tuple(cos.shape)} does not fit {batch} x {rows} rows of heads of {dim} (at most 4096)")
    index = _device_index(torch, what, first, cos, sin, first if y is None else y)
    st = cos.stride()
    _launch_rotary(torch, what, x, y, xo, yo, index, code, 0, _NO_STRIDES, 0, 0, cos.data_ptr(), sin.data_ptr(),
                   (st[0] if cos.shape[0] == batch else 0, st[1], st[2]), 1.0, 0, int(pairing == "adjacent"), cos.shape[2])
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


def _steps(what: str, name: str, t: Any) -> Tuple[int, ...]:
    """Strides of batch, rows and heads; a dimension of one entry has none."""
    st = t.stride()
    steps = tuple(0 if n == 1 else x for n, x in zip(t.shape, st[:3]))
    if t.numel() and (st[3] != 1 or t.data_ptr() & 15 or (steps[0] | steps[1] | steps[2]) & 7):
        raise ValueError(f"{what}: {name} must be 16-byte aligned, strides multiples of 8, the elements of a head side by side")
    return steps


def attention(q: Any, k: Any, v: Any, *, key_ranges: Any = None, causal: bool = False, scale: Optional[float] = None, softcap: float = 0.0) -> Any:
    """Softmax attention of q [batch, rows, heads, dim] over k, v [batch, keys, kv_heads, dim] (or [rows, heads, dim] of packed documents), heads
    a multiple of kv_heads.  key_ranges int32 [batch or 1, rows, 2]: row i sees the keys [lo, hi), cut to what there is; an empty range gives
    zeros; None: every key, or with `causal` those up to the row itself (the last row stands at the last key).  scale defaults to dim ** -0.5; softcap
    c > 0 caps scores to c * tanh(score / c).  bfloat16 or float16; dim a multiple of 8 up to 256; any strides that are multiples of 8 with the elements
    of a head side by side, 16-byte aligned, rows of k and v at most 2^23 elements apart.
    -> new contiguous tensor of q's shape."""
    torch = _torch()
    what = "attention"
    shape = q.shape
    code = _dtype_code(torch, q.dtype, what, fp32=False)
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"{what}: q, k and v differ in type ({q.dtype}, {k.dtype}, {v.dtype})")
    if len(shape) != 4 or k.dim() != 4 or v.dim() != 4:
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
    if not 0 < scale < _FP32_MAX:
        raise ValueError(f"{what}: scale must be positive and finite")
    if not 0 <= softcap < _FP32_MAX:
        raise ValueError(f"{what}: softcap must not be negative (0: no cap)")
    at_q, at_k, at_v, st_q, st_k, st_v = q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(), k.stride(), v.stride()
    q0, q1, q2, q3 = st_q
    k0, k1, k2, k3 = st_k
    v0, v1, v2, v3 = st_v
    if (at_q | at_k | at_v) & 15 or (q0 | q1 | q2 | k0 | k1 | k2 | v0 | v1 | v2) & 7 or not q3 == k3 == v3 == 1:
        (q0, q1, q2), (k0, k1, k2), (v0, v1, v2) = (_steps(what, name, t) for name, t in (("q", q), ("k", k), ("v", v)))
    if key_ranges is not None:
        if causal:
            raise ValueError(f"{what}: causal goes without key_ranges (padded_ranges(..., prefix=0) makes causal ones)")
        r_shape = key_ranges.shape
        if key_ranges.dtype is not torch.int32 or len(r_shape) != 3 or r_shape[0] not in (1, batch) or r_shape[1] != rows or r_shape[2] != 2:
            raise ValueError(f"{what}: key_ranges must be int32 [{batch} or 1, {rows}, 2], not {key_ranges.dtype} {tuple(key_ranges.shape)}")
        index = _device_index(torch, what, q, k, v, key_ranges)
        if not key_ranges.is_contiguous() or key_ranges.data_ptr() & 7:
            key_ranges = key_ranges.clone(memory_format=torch.contiguous_format)
        ranges, ranges_batch = key_ranges.data_ptr(), 0 if r_shape[0] == 1 else 2 * rows
    else:
        index = _device_index(torch, what, q, k, v)
        ranges = ranges_batch = 0
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if batch and rows:
        need = _workspace_bytes(index, batch, rows, keys, heads, kv_heads, dim)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None  # torch's own reuse rules keep it this call's on this stream
        packed = _PACK_ATTN.pack(at_q, at_k, at_v, out.data_ptr(), ranges, q0, q1, q2, k0, k1, k2, v0, v1, v2, ranges_batch, work.data_ptr() if need else 0, need,
                                 code, batch, rows, keys, heads, kv_heads, dim, int(causal), scale, softcap)
        _lib.check(_lib.lib().mv_enc_attention(index, packed, _stream(torch, index)))
    return out if len(shape) == 4 else out.view(shape)


# --------------------------------------------------------------------------- the encoders' own blocks
_NAME = "mv_key_ranges"  # of the attention and mask functions registered with transformers
_DECODERS = ("GemmaAttention", "Qwen2VLAttention", "Qwen2_5_VLAttention")
_PACKED = ("VisionAttention", "Qwen2_5_VLVisionAttention")


class _Angles(tuple):
    """(cos, sin) as a rotary module returns them, and what they were made of: positions [axes, batch, rows] and the RotaryTable."""

    positions: Any = None
    table: Any = None


def enabled_by_env() -> bool:
    return os.environ.get("MV_ENCODER_FUSED_ATTENTION", "0") in ("1", "true", "yes")


def _kernel_takes(torch, query, key, value, scaling=None, softcap=None) -> bool:
    """Inference on a GPU in types, shapes and a layout ([batch, heads, rows, dim]) that `attention` has; anything else goes the framework's way."""
    return query.is_cuda and not torch.is_grad_enabled() and _fits(torch, query, key, value, scaling, softcap)


def _fits(torch, query, key, value, scaling=None, softcap=None) -> bool:
    dtype, device, dim = query.dtype, query.device, query.shape[-1]
    if dtype not in (torch.bfloat16, torch.float16) or dim % 8 or not 8 <= dim <= 256 or key.shape != value.shape or key.shape[0] != query.shape[0] or key.shape[3] != dim:
        return False
    if key.shape[1] < 1 or query.shape[1] < 1 or query.shape[1] % key.shape[1] or max(key.stride(2), value.stride(2)) > _MAX_ROW_STRIDE:
        return False
    scale, cap = dim**-0.5 if scaling is None else scaling, softcap or 0.0
    if not 0 < scale * 4 < _FP32_MAX or not 0 <= cap * 4 < _FP32_MAX or cap and not 1e-36 < scale / cap < 1e36:
        return False
    return all(t.dtype == dtype and t.device == device and t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(st % 8 for st in t.stride()[:-1]) for t in (query, key, value))


def _capped_attention(torch, module, query, key, value, mask, scaling, dropout, softcap, causal):
    """The formula of `attention` in plain operations, in 32 bits: capped scores where the kernel does not apply."""
    group, rows, keys = query.shape[1] // key.shape[1], query.shape[2], key.shape[2]
    k, v = (t.float().repeat_interleave(group, 1) for t in (key, value))
    s = torch.matmul(query.float(), k.transpose(2, 3).contiguous()) * (query.shape[3] ** -0.5 if scaling is None else scaling)
    s = softcap * torch.tanh(s / softcap)
    if causal:
        mask = torch.ones(rows, keys, dtype=torch.bool, device=query.device).tril()
    if mask is not None:
        s = s.masked_fill(~mask, -math.inf) if mask.dtype == torch.bool else s + mask
    p = torch.softmax(s, -1).masked_fill((s == -math.inf).all(-1, keepdim=True), 0.0)  # a row that sees nothing is zero
    p = torch.nn.functional.dropout(p, dropout, module.training)
    return torch.matmul(p, v).to(query.dtype).transpose(1, 2).contiguous()


def _is_causal(module, asked: Optional[bool]) -> bool:
    """Without a mask: what the forward asks for, else what the module says; one that says nothing is causal, as the framework's own function takes it."""
    return bool(getattr(module, "is_causal", True) if asked is None else asked)


def _interface_attention(module, query, key, value, attention_mask=None, scaling=None, dropout=0.0, softcap=None, is_causal=None, **kwargs):
    """transformers' attention function: query [batch, heads, rows, dim], key / value [batch, kv_heads, keys, dim] -> ([batch, rows, heads, dim], None)."""
    torch = _torch()
    ranges = attention_mask[:, 0] if attention_mask is not None and attention_mask.dtype == torch.int32 else None
    causal = attention_mask is None and query.shape[2] > 1 and _is_causal(module, is_causal)
    known = ranges is not None or attention_mask is None and not (causal and query.shape[2] != key.shape[2])
    extras = any(kwargs.get(name) is not None for name in ("s_aux", "position_bias"))  # sinks, added biases: not in the kernel
    if known and not dropout and not extras and _kernel_takes(torch, query, key, value, scaling, softcap):
        out = attention(query.transpose(1, 2), key.transpose(1, 2), value.transpose(1, 2), key_ranges=ranges, causal=causal, scale=scaling, softcap=softcap or 0.0)
        return out, None
    from transformers import AttentionInterface

    if ranges is not None:  # back to a boolean mask
        at = torch.arange(key.shape[2], device=query.device, dtype=torch.int32)
        attention_mask = ((at >= ranges[..., :1]) & (at < ranges[..., 1:]))[:, None]
    if softcap:  # the framework's function has none
        if extras:
            raise ValueError("attention: a softcap together with sinks or an added bias")
        return _capped_attention(torch, module, query, key, value, attention_mask, scaling, dropout, softcap, causal), None
    return AttentionInterface()["sdpa"](module, query, key, value, attention_mask, scaling=scaling, dropout=dropout, is_causal=is_causal, **kwargs)


def _interface_mask(*args, **kwargs):
    """transformers' mask function: once per forward, the mask as key ranges int32 [batch, 1, rows, 2] where every row's keys are one run (causal, padded,
    prefix and packed masks are), as the boolean mask otherwise (asking costs one wait for the GPU a forward).  None stays None: the attention function
    goes by the module's is_causal then, as the framework's own does."""
    from transformers import AttentionMaskInterface

    torch = _torch()
    mask = AttentionMaskInterface()["sdpa"](*args, **kwargs)
    if mask is None or mask.dtype != torch.bool or mask.dim() != 4 or mask.shape[1] != 1 or not mask.is_cuda or torch.cuda.is_current_stream_capturing():
        return mask
    ranges, exact = ranges_from_mask(mask[:, 0])
    return ranges[:, None] if bool(exact) else mask


def _rotary_forward(self, x, position_ids, *args, **kwargs):
    torch = _torch()
    angles = self._mv_attn_forward(x, position_ids, *args, **kwargs)
    if not x.is_cuda or torch.is_grad_enabled() or position_ids.dtype not in (torch.int32, torch.int64) or position_ids.dim() not in (2, 3):
        return angles
    freq, scale = self.inv_freq, float(getattr(self, "attention_scaling", 1.0))
    made_of = (freq, None if freq.is_inference() else freq._version, scale, x.device)  # a model that is cast or moved gets new frequencies
    kept = self._mv_rotary_table
    if kept is None or kept[0][0] is not freq or kept[0][1:] != made_of[1:]:
        sections = self._mv_rotary_sections
        axes = None if sections is None else [a for a, n in enumerate(sections) for _ in range(n)]
        kept = self._mv_rotary_table = made_of, RotaryTable(freq, axes, head_dim=2 * int(freq.shape[0]), scale=scale, device=x.device)
    table = kept[1]
    positions = position_ids[None] if position_ids.dim() == 2 else position_ids
    if positions.shape[0] < table.axes:
        return angles
    out = _Angles(angles)
    out.positions, out.table = positions, table
    return out


def _ours(torch, *projections) -> bool:
    """Whether what the projections return is this block's to overwrite: a plain linear layer's new tensor, which no hook has been handed."""
    return not torch.nn.modules.module._global_forward_hooks and all(type(p) is torch.nn.Linear and not p._forward_hooks for p in projections)


def _drops(module) -> bool:
    """Training mode (under no_grad) with dropout of the attention's weights: not in the kernel."""
    return bool(module.training and getattr(module, "attention_dropout", 0.0))


def _decoder_forward(self, *args, **kwargs):
    """q, k, v -> rotation (in place where they are the block's own) -> attention over key ranges -> output projection; what does not fit goes through the module's own forward."""
    torch = _torch()
    x, mask, angles = kwargs.get("hidden_states"), kwargs.get("attention_mask"), kwargs.get("position_embeddings")
    if (args or x is None or x.dim() != 3 or not x.is_cuda or torch.is_grad_enabled() or x.dtype not in (torch.bfloat16, torch.float16)
            or _drops(self) or (mask is not None and mask.dtype != torch.int32) or not isinstance(angles, _Angles) or angles.table.head_dim != self.head_dim or self.head_dim % 8 or self.head_dim > 256):
        return self._mv_attn_forward(*args, **kwargs)
    batch, rows = x.shape[:2]
    q, k, v = (proj(x).view(batch, rows, -1, self.head_dim) for proj in (self.q_proj, self.k_proj, self.v_proj))
    q, k = rotary(q, k, angles.positions, angles.table, in_place=_ours(torch, self.q_proj, self.k_proj))
    cache = kwargs.get("past_key_values")
    if cache is not None:
        heads_first = q.transpose(1, 2), *cache.update(k.transpose(1, 2), v.transpose(1, 2), self.layer_idx)
        if not _kernel_takes(torch, *heads_first, self.scaling):  # what a cache hands back may be of another type or layout
            out, _ = _interface_attention(self, *heads_first, mask, scaling=self.scaling, is_causal=kwargs.get("is_causal"))
            return self.o_proj(out.flatten(2)), None
        k, v = (t.transpose(1, 2) for t in heads_first[1:])
    if mask is not None:
        out = attention(q, k, v, key_ranges=mask[:, 0], scale=self.scaling)
    else:
        causal = rows > 1 and _is_causal(self, kwargs.get("is_causal"))
        if causal and k.shape[1] > rows:  # no mask over a longer cache: a prompt in front of its unfilled places
            k, v = k[:, :rows], v[:, :rows]
        out = attention(q, k, v, causal=causal, scale=self.scaling)
    return self.o_proj(out.flatten(2)), None


def _packed_forward(self, hidden_states, *args, **kwargs):
    """Packed patches: fused projection -> rotation by the tower's tables (as above) -> attention within each document or window -> output projection."""
    torch = _torch()
    x, offsets, angles = hidden_states, kwargs.get("cu_seqlens"), kwargs.get("position_embeddings")
    dim = self.head_dim
    if (args or x.dim() != 2 or not x.is_cuda or torch.is_grad_enabled() or x.dtype not in (torch.bfloat16, torch.float16) or _drops(self) or offsets is None or angles is None
            or offsets.dtype != torch.int32 or not offsets.is_contiguous() or offsets.device != x.device or angles[0].dtype != torch.float32
            or angles[0].shape != (x.shape[0], dim) or dim % 8 or dim > 256):
        return self._mv_attn_forward(hidden_states, *args, **kwargs)
    q, k, v = self.qkv(x).view(x.shape[0], 3, -1, dim).unbind(1)
    cos, sin = (t[:, : dim // 2] for t in angles)
    q, k = rotary_tables(q, k, cos, sin, in_place=_ours(torch, self.qkv))
    out = attention(q, k, v, key_ranges=document_ranges(offsets, x.shape[0]), scale=self.scaling)
    return self.proj(out.flatten(1))


def _implementations(model: Any) -> list:
    """(configuration, its attention function) of every part of the model."""
    seen: Dict[int, Any] = {}
    for mod in model.modules():
        config = getattr(mod, "config", None)
        if config is not None and hasattr(config, "_attn_implementation"):
            seen.setdefault(id(config), (config, config._attn_implementation))
    return list(seen.values())


def patch_attention(model: Any) -> Dict[str, int]:
    """Run the attention of a transformers encoder through this module, in place: the model's attention function becomes `attention` (with the mask
    of a forward as key ranges), its decoder blocks rotate by positions, its packed vision blocks attend all documents and windows in one launch (the
    framework takes them one by one).  Modules fall back to their own forward for anything the kernels do not take (not on a GPU, autograd on, another
    type, a mask with holes, a mask while a graph is captured, dropout of a model in training mode).  -> modules patched per kind.  `unpatch_attention` undoes it."""
    from transformers import AttentionInterface, AttentionMaskInterface

    counts = {"rotary": 0, "decoder": 0, "packed": 0}
    if hasattr(model, "_mv_attn_before"):
        return counts
    AttentionInterface.register(_NAME, _interface_attention)
    AttentionMaskInterface.register(_NAME, _interface_mask)
    model._mv_attn_before = _implementations(model)
    model.set_attn_implementation(_NAME)
    for mod in model.modules():
        cls, children = type(mod).__name__, {n for n, _ in mod.named_children()}
        if cls.endswith("RotaryEmbedding") and hasattr(mod, "inv_freq") and getattr(mod, "rope_type", None) == "default":
            config = getattr(mod, "config", None)
            params = getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {}
            sections = params.get("mrope_section")
            if sections is not None and sum(sections) != mod.inv_freq.shape[0]:
                continue
            mod._mv_rotary_sections, mod._mv_rotary_table = sections, None
            kind, forward = "rotary", _rotary_forward
        elif cls in _DECODERS and children == {"q_proj", "k_proj", "v_proj", "o_proj"}:
            kind, forward = "decoder", _decoder_forward
        elif cls in _PACKED and children == {"qkv", "proj"}:
            kind, forward = "packed", _packed_forward
        else:
            continue
        mod._mv_attn_forward = mod.forward
        mod.forward = types.MethodType(forward, mod)
        counts[kind] += 1
    return counts


def patch_on_request(model: Any, device: Any, asked: Optional[bool]) -> Dict[str, int]:
    """The `fused_attention=` option of the embedding models: True, or None with MV_ENCODER_FUSED_ATTENTION=1, patches a model on a GPU.  There are no kernels
    anywhere else: a request by name is answered by a warning there.  -> modules patched per kind"""
    if asked is not False and (asked or enabled_by_env()):
        if device.type == "cuda":
            return patch_attention(model)
        if asked:
            logger.warning("fused_attention: the model is on %s, its attention stays the framework's (the kernels need a GPU)", device)
    return {"rotary": 0, "decoder": 0, "packed": 0}


def unpatch_attention(model: Any) -> None:
    """Give every module its own forward back and the model the attention function it had."""
    if not hasattr(model, "_mv_attn_before"):
        return
    for config, name in model._mv_attn_before:  # one by one: set_attn_implementation leaves parts of a model that have been changed before
        config._attn_implementation = name
    del model._mv_attn_before
    for mod in model.modules():
        if hasattr(mod, "_mv_attn_forward"):
            mod.forward = mod._mv_attn_forward
            del mod._mv_attn_forward
        for name in ("_mv_rotary_table", "_mv_rotary_sections"):
            if hasattr(mod, name):
                delattr(mod, name)
