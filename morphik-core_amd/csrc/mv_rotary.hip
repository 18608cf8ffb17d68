// mv_rotary.hip -- rotary positions with several axes (time, height, width) for the queries and keys of the encoder blocks (reference
// formulation: model(**processor(x)), core/embedding/colpali_embedding_model.py:251-262; the rotation is inside transformers' blocks).
//
//   pair j of a head, token t:  angle = position[axis_j][t] * inv_freq_j
//   (x, y) -> scale * (x cos - y sin,  y cos + x sin);   x, y = elements (j, j + P) or (2 j, 2 j + 1) of the first 2 P; the rest is copied.
//
// One launch for q and k.  A block takes a few tokens: it computes their P cosines and sines once into LDS and sweeps all heads with them,
// so what remains is one read and one write of q and k.  Angles are 64-bit products reduced to revolutions before anything is rounded to
// 32 bits (a position of 10^5 at frequency 1 leaves 32 bits two decimal places of the angle); with 64-bit work for one pair in
// (heads + kv_heads) only, it is hidden behind the memory traffic.
//
// Bound by memory.  One MI355X, a copy of 1 GiB running at 5.1 TB/s: 8 x 1101 tokens x 18 heads of 128 in bf16 (81 MB) 15.7 us (5.2 TB/s, 4.5 from cold
// caches); 12512 x 32 heads of 80 inside a fused projection (132 MB) 25.5 us (5.2; 4.2 cold); 8002 x 9 heads of 256 in fp32 (148 MB) 27.9 us (5.3; 4.0
// cold).  A call of 20 tokens takes 4.5 us, most of it the launch.  Tried and not kept: the first vectors of every thread on their way before the
// angles are computed (18.3 -> 20.9 us cold: fewer waves fit), non-temporal stores (31 -> 38 us: the reader comes next).
#include <algorithm>

#include "mv_common.h"
#include "mv_index_priv.h"

namespace mv {
namespace {

struct RotaryArgs {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h;      // strides in elements
  int64_t qo_b, qo_l, qo_h, ko_b, ko_l, ko_h;
  const void* positions;                     // int32 / int64 [axes][batch][rows], or null: angles come as cosines and sines
  int64_t pos_a, pos_b, pos_l;
  const double* inv_freq;                    // [pairs]
  const int32_t* axis;                       // [pairs]
  const float *cos, *sin;                    // [batch][rows][pairs]
  int64_t tab_b, tab_l, tab_p;
  float scale;
  int32_t batch, rows, heads, kv_heads, dim, pairs, tokens;  // tokens: of a block
  int64_t total;                             // batch * rows
  int32_t pos64, copy_rest;                  // copy_rest: elements from 2 * pairs on are written too (not when in place)
};

template <int N>
struct Bytes;
template <>
struct Bytes<2> { using type = uint16_t; };
template <>
struct Bytes<4> { using type = uint32_t; };
template <>
struct Bytes<16> { using type = __attribute__((ext_vector_type(4))) unsigned int; };

// T: 0 fp32, 1 bf16, 2 fp16.  VE elements at a time: 16 bytes, or one where the sizes or alignments do not allow that.
template <int T>
struct Elem;
template <>
struct Elem<0> { using type = float; };
template <>
struct Elem<1> { using type = __bf16; };
template <>
struct Elem<2> { using type = _Float16; };

template <int T, int VE, bool ADJ>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  using E = typename Elem<T>::type;
  using Vec = typename Bytes<sizeof(E) * VE>::type;
  struct alignas(sizeof(E) * VE) Pack { E e[VE]; };
  extern __shared__ float2 lds_cs[];  // [tokens][pairs]
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n_tok = (int)(a.total - t0 < a.tokens ? a.total - t0 : a.tokens);
  for (int i = threadIdx.x; i < n_tok * a.pairs; i += 256) {
    const int64_t t = t0 + i / a.pairs, b = t / a.rows, l = t % a.rows;
    const int j = i % a.pairs;
    float2 cs;
    if (a.positions) {
      const int64_t at = (int64_t)a.axis[j] * a.pos_a + b * a.pos_b + l * a.pos_l;
      const double p = a.pos64 ? (double)reinterpret_cast<const int64_t*>(a.positions)[at] : (double)reinterpret_cast<const int32_t*>(a.positions)[at];
      const double rev = p * a.inv_freq[j] * 0.15915494309189535;  // 1 / (2 pi)
      const double half_turns = 2.0 * (rev - rint(rev));  // in [-1, 1]
      const float hi = (float)half_turns, lo = (float)(half_turns - (double)hi) * 3.1415927f;
      float sn, co;
      sincospif(hi, &sn, &co);  // at pi hi, and one step of the sum formulas for what 32 bits left over of the angle
      cs = make_float2(__builtin_fmaf(-lo, sn, co), __builtin_fmaf(lo, co, sn));
    } else {
      const int64_t at = b * a.tab_b + l * a.tab_l + j * a.tab_p;
      cs = make_float2(a.cos[at], a.sin[at]);
    }
    lds_cs[i] = make_float2(cs.x * a.scale, cs.y * a.scale);
  }
  __syncthreads();
  // work items of a token: for every head of q, then of k, the vectors that hold its pairs ("halves": a vector of x and the one of y that
  // belongs to it), then the vectors that are only copied
  const int rot_items = (ADJ ? 2 * a.pairs : a.pairs) / VE;
  const int items = rot_items + (a.copy_rest ? (a.dim - 2 * a.pairs) / VE : 0);
  const int per_token = items * (a.heads + a.kv_heads);
  for (int i = threadIdx.x; i < n_tok * per_token; i += 256) {
    const int tok = i / per_token, rest = i - tok * per_token;
    const int head = rest / items, it = rest - head * items;
    const int64_t t = t0 + tok, b = t / a.rows, l = t % a.rows;
    const bool is_k = head >= a.heads;
    const E* src = is_k ? reinterpret_cast<const E*>(a.k) + b * a.k_b + l * a.k_l + (head - a.heads) * a.k_h
                        : reinterpret_cast<const E*>(a.q) + b * a.q_b + l * a.q_l + head * a.q_h;
    E* dst = is_k ? reinterpret_cast<E*>(a.k_out) + b * a.ko_b + l * a.ko_l + (head - a.heads) * a.ko_h
                  : reinterpret_cast<E*>(a.q_out) + b * a.qo_b + l * a.qo_l + head * a.qo_h;
    if (it >= rot_items) {
      const int c = 2 * a.pairs + (it - rot_items) * VE;
      *reinterpret_cast<Vec*>(dst + c) = *reinterpret_cast<const Vec*>(src + c);
      continue;
    }
    const float2* cs = lds_cs + tok * a.pairs;
    if constexpr (ADJ) {
      if constexpr (VE == 1) {  // one element at a time still needs its neighbour: the even one's item does both
        if (it & 1) continue;
        const float x = (float)src[it], y = (float)src[it + 1];
        const float2 w = cs[it >> 1];
        dst[it] = (E)__builtin_fmaf(x, w.x, -y * w.y);
        dst[it + 1] = (E)__builtin_fmaf(y, w.x, x * w.y);
      } else {
        Pack v = __builtin_bit_cast(Pack, *reinterpret_cast<const Vec*>(src + it * VE));
#pragma unroll
        for (int e = 0; e < VE; e += 2) {
          const float x = (float)v.e[e], y = (float)v.e[e + 1];
          const float2 w = cs[(it * VE + e) >> 1];
          v.e[e] = (E)__builtin_fmaf(x, w.x, -y * w.y);
          v.e[e + 1] = (E)__builtin_fmaf(y, w.x, x * w.y);
        }
        *reinterpret_cast<Vec*>(dst + it * VE) = __builtin_bit_cast(Vec, v);
      }
    } else {
      Pack vx = __builtin_bit_cast(Pack, *reinterpret_cast<const Vec*>(src + it * VE));
      Pack vy = __builtin_bit_cast(Pack, *reinterpret_cast<const Vec*>(src + a.pairs + it * VE));
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float x = (float)vx.e[e], y = (float)vy.e[e];
        const float2 w = cs[it * VE + e];
        vx.e[e] = (E)__builtin_fmaf(x, w.x, -y * w.y);
        vy.e[e] = (E)__builtin_fmaf(y, w.x, x * w.y);
      }
      *reinterpret_cast<Vec*>(dst + it * VE) = __builtin_bit_cast(Vec, vx);
      *reinterpret_cast<Vec*>(dst + a.pairs + it * VE) = __builtin_bit_cast(Vec, vy);
    }
  }
}

template <int T>
void launch_rotary(const RotaryArgs& a, bool wide, bool adjacent, unsigned blocks, size_t lds, hipStream_t s) {
  constexpr int VE = 16 / sizeof(typename Elem<T>::type);
  if (wide && adjacent) hipLaunchKernelGGL((rotary_kernel<T, VE, true>), dim3(blocks), dim3(256), lds, s, a);
  else if (wide) hipLaunchKernelGGL((rotary_kernel<T, VE, false>), dim3(blocks), dim3(256), lds, s, a);
  else if (adjacent) hipLaunchKernelGGL((rotary_kernel<T, 1, true>), dim3(blocks), dim3(256), lds, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 1, false>), dim3(blocks), dim3(256), lds, s, a);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

int mv_enc_rotary(int device, const mv_rotary* p, void* stream) {
  if (!p || p->batch < 0 || p->rows < 0 || p->heads < 0 || p->kv_heads < 0 || p->dim < 1 || p->pairs < 0 || (int64_t)2 * p->pairs > p->dim) {
    set_error("mv_enc_rotary: bad sizes (at most dim / 2 pairs)");
    return MV_ERR_INVALID;
  }
  if (p->dtype != MV_F32 && p->dtype != MV_BF16 && p->dtype != MV_F16) {
    set_error("mv_enc_rotary: dtype must be MV_F32, MV_BF16 or MV_F16");
    return MV_ERR_INVALID;
  }
  if (p->dim > 4096) {
    set_error("mv_enc_rotary: head dimension %d (at most 4096)", p->dim);
    return MV_ERR_INVALID;
  }
  const int64_t total = (int64_t)p->batch * p->rows;
  if (total == 0 || (p->heads == 0 && p->kv_heads == 0)) return MV_OK;
  const bool tables = p->cos || p->sin;
  if ((p->heads && (!p->q || !p->q_out)) || (p->kv_heads && (!p->k || !p->k_out)) || (tables && (!p->cos || !p->sin || p->positions)) ||
      (!tables && p->pairs && (!p->positions || !p->inv_freq || !p->axis))) {
    set_error("mv_enc_rotary: missing operand (q / k with their outputs; positions with inv_freq and axis, or cos and sin)");
    return MV_ERR_INVALID;
  }
  RotaryArgs a = {};
  a.q = p->q, a.k = p->k, a.q_out = p->q_out, a.k_out = p->k_out;
  a.q_b = p->q_batch, a.q_l = p->q_row, a.q_h = p->q_head, a.k_b = p->k_batch, a.k_l = p->k_row, a.k_h = p->k_head;
  a.qo_b = p->q_out_batch, a.qo_l = p->q_out_row, a.qo_h = p->q_out_head, a.ko_b = p->k_out_batch, a.ko_l = p->k_out_row, a.ko_h = p->k_out_head;
  a.positions = tables ? nullptr : p->positions;
  a.pos64 = p->positions_are_64bit;
  a.pos_a = p->positions_axis, a.pos_b = p->positions_batch, a.pos_l = p->positions_row;
  a.inv_freq = p->inv_freq, a.axis = p->axis, a.cos = p->cos, a.sin = p->sin;
  a.tab_b = p->table_batch, a.tab_l = p->table_row, a.tab_p = p->table_pair;
  a.scale = p->scale;
  a.batch = p->batch, a.rows = p->rows, a.heads = p->heads, a.kv_heads = p->kv_heads, a.dim = p->dim, a.pairs = p->pairs, a.total = total;
  const bool in_place = (!p->heads || p->q == p->q_out) && (!p->kv_heads || p->k == p->k_out);
  a.copy_rest = !in_place && 2 * p->pairs < p->dim;

  // 16-byte vectors where every vector of pairs (and of the rest) starts at a multiple of 16 bytes; else element by element
  const int size = p->dtype == MV_F32 ? 4 : 2, ve = 16 / size;
  int64_t strides = 0;
  uintptr_t ptrs = 0;
  if (p->heads) strides |= a.q_b | a.q_l | a.q_h | a.qo_b | a.qo_l | a.qo_h, ptrs |= (uintptr_t)a.q | (uintptr_t)a.q_out;
  if (p->kv_heads) strides |= a.k_b | a.k_l | a.k_h | a.ko_b | a.ko_l | a.ko_h, ptrs |= (uintptr_t)a.k | (uintptr_t)a.k_out;
  if (ptrs & (size - 1)) {
    set_error("mv_enc_rotary: q and k must be aligned to their elements");
    return MV_ERR_INVALID;
  }
  const bool wide = !(ptrs & 15) && strides % ve == 0 && (p->adjacent ? 2 * p->pairs : p->pairs) % ve == 0 && (!a.copy_rest || p->dim % ve == 0);

  // tokens of a block: enough to give every thread a vector or two, as few as that, so that small calls still spread over the card (8 pages of 1101
  // tokens x 18 heads of 128, from memory: 18.3 us with 512 items a block, 22.2 with 256, 18.9 with 1024, 22.7 with 2048)
  const int64_t vecs = std::max<int64_t>(1, (int64_t)(p->heads + p->kv_heads) * p->dim / (wide ? 2 * ve : 2));
  int64_t tokens = std::max<int64_t>(1, 512 / vecs);
  tokens = std::min<int64_t>(tokens, std::max<int64_t>(1, 32768 / std::max<int64_t>(8, (int64_t)p->pairs * 8)));
  a.tokens = (int32_t)std::min<int64_t>(tokens, total);
  const int64_t blocks = (total + a.tokens - 1) / a.tokens;
  if (blocks > 0x7fffffff || (int64_t)a.tokens * (p->heads + p->kv_heads) * p->dim > 0x7fffffff) {
    set_error("mv_enc_rotary: too many tokens or heads for one launch");
    return MV_ERR_INVALID;
  }
  const size_t lds = (size_t)std::max(1, a.tokens * a.pairs) * sizeof(float2);
  DeviceGuard g(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->dtype == MV_F32) launch_rotary<0>(a, wide, p->adjacent, (unsigned)blocks, lds, s);
  else if (p->dtype == MV_BF16) launch_rotary<1>(a, wide, p->adjacent, (unsigned)blocks, lds, s);
  else launch_rotary<2>(a, wide, p->adjacent, (unsigned)blocks, lds, s);
  MV_HIP(hipGetLastError());
  return MV_OK;
}

}  // extern "C"
