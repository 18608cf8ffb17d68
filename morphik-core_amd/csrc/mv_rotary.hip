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
  int32_t pos64;
  int32_t rot_vecs, rot_ones, copy_vecs, copy_ones;  // work items of a head: vectors and single pairs that turn, vectors and elements that are copied
};

// T: 0 fp32, 1 bf16, 2 fp16
template <int T>
struct Elem;
template <>
struct Elem<0> { using type = float; };
template <>
struct Elem<1> { using type = __bf16; };
template <>
struct Elem<2> { using type = _Float16; };

// Items of 16 bytes whatever the alignment: heads of 72 have 36 pairs, so that the second halves start in the middle of 16 bytes, and odd numbers of pairs
// in the middle of a word.  Such loads and stores are single instructions too (element alignment is what they are compiled for).  Against items of one
// element wherever 16 bytes are not aligned, bf16: 12512 tokens x 32 heads of 72 57.8 -> 20.9 us, 8 x 1101 x 18 heads of 128 with 33 pairs 60.8 -> 18.5
// (adjacent 73.3 -> 19.1, in place 28.9 -> 16.8).
template <class E>
__device__ __forceinline__ void load(E (&v)[16 / sizeof(E)], const E* p) { __builtin_memcpy(v, p, 16); }
template <class E>
__device__ __forceinline__ void store(E* p, const E (&v)[16 / sizeof(E)]) { __builtin_memcpy(p, v, 16); }

// To the type of the result, from 32 bits in every kind of item: left to itself the compiler rounds some fp16 results straight from the product and sum, and
// then a pair turned in place could differ by the last bit from the same pair turned into a new tensor.
template <class E>
__device__ __forceinline__ E rounded(float x) {
  asm("" : "+v"(x));
  return (E)x;
}

template <int T, bool ADJ>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  using E = typename Elem<T>::type;
  constexpr int VE = 16 / sizeof(E);
  extern __shared__ float2 lds_cs[];  // [tokens][pairs]
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n_tok = (int)(a.total - t0 < a.tokens ? a.total - t0 : a.tokens);
  const int64_t b0 = t0 / a.rows;
  const uint32_t l0 = (uint32_t)(t0 % a.rows), rows = (uint32_t)a.rows;  // l0 + tokens stays below 2^32
  for (int i = threadIdx.x; i < n_tok * a.pairs; i += 256) {
    const uint32_t at_row = l0 + i / a.pairs;
    const int64_t b = b0 + at_row / rows, l = at_row % rows;
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
  // belongs to it; the last vector may reach back over the one before it), the pairs that fill no vector, and the same of what is only copied
  const int items = a.rot_vecs + a.rot_ones + a.copy_vecs + a.copy_ones;
  const int per_token = items * (a.heads + a.kv_heads);
  const int turned = ADJ ? 2 * a.pairs : a.pairs;  // elements that the vectors go over
  for (int i = threadIdx.x; i < n_tok * per_token; i += 256) {
    const int tok = i / per_token, rest = i - tok * per_token;
    const int head = rest / items;
    int it = rest - head * items;
    const uint32_t at_row = l0 + tok;
    const int64_t b = b0 + at_row / rows, l = at_row % rows;
    const bool is_k = head >= a.heads;
    const E* src = is_k ? reinterpret_cast<const E*>(a.k) + b * a.k_b + l * a.k_l + (head - a.heads) * a.k_h
                        : reinterpret_cast<const E*>(a.q) + b * a.q_b + l * a.q_l + head * a.q_h;
    E* dst = is_k ? reinterpret_cast<E*>(a.k_out) + b * a.ko_b + l * a.ko_l + (head - a.heads) * a.ko_h
                  : reinterpret_cast<E*>(a.q_out) + b * a.qo_b + l * a.qo_l + head * a.qo_h;
    const float2* cs = lds_cs + tok * a.pairs;
    if (it < a.rot_vecs) {
      const int c = min(it * VE, turned - VE);
      E x[VE], y[VE];
      load(x, src + c);
      if constexpr (ADJ) {
        const float2* cw = cs + (c >> 1);
#pragma unroll
        for (int e = 0; e < VE; e += 2) {
          const float2 w = cw[e / 2];
          y[e] = rounded<E>(__builtin_fmaf((float)x[e], w.x, -(float)x[e + 1] * w.y));
          y[e + 1] = rounded<E>(__builtin_fmaf((float)x[e + 1], w.x, (float)x[e] * w.y));
        }
        store(dst + c, y);
      } else {
        load(y, src + a.pairs + c);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float xe = (float)x[e], ye = (float)y[e];
          const float2 w = cs[c + e];
          x[e] = rounded<E>(__builtin_fmaf(xe, w.x, -ye * w.y));
          y[e] = rounded<E>(__builtin_fmaf(ye, w.x, xe * w.y));
        }
        store(dst + c, x);
        store(dst + a.pairs + c, y);
      }
      continue;
    }
    it -= a.rot_vecs;
    if (it < a.rot_ones) {
      const int j = (ADJ ? a.rot_vecs * (VE / 2) : a.rot_vecs * VE) + it, cx = ADJ ? 2 * j : j, cy = ADJ ? cx + 1 : j + a.pairs;
      const float x = (float)src[cx], y = (float)src[cy];
      const float2 w = cs[j];
      dst[cx] = rounded<E>(__builtin_fmaf(x, w.x, -y * w.y));
      dst[cy] = rounded<E>(__builtin_fmaf(y, w.x, x * w.y));
      continue;
    }
    it -= a.rot_ones;
    const int c = 2 * a.pairs, n = a.dim - c;
    if (it < a.copy_vecs) {
      const int at = c + min(it * VE, n - VE);
      E x[VE];
      load(x, src + at);
      store(dst + at, x);
    } else {
      const int at = c + it - a.copy_vecs;  // there are vectors or single elements, not both
      dst[at] = src[at];
    }
  }
}

template <int T>
void launch_rotary(const RotaryArgs& a, bool adjacent, unsigned blocks, size_t lds, hipStream_t s) {
  if (adjacent) hipLaunchKernelGGL((rotary_kernel<T, true>), dim3(blocks), dim3(256), lds, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, false>), dim3(blocks), dim3(256), lds, s, a);
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
  const bool q_in_place = p->heads && p->q == p->q_out, k_in_place = p->kv_heads && p->k == p->k_out;
  const bool copy = 2 * p->pairs < p->dim && ((p->heads && !q_in_place) || (p->kv_heads && !k_in_place));

  const int size = p->dtype == MV_F32 ? 4 : 2, ve = 16 / size;
  uintptr_t ptrs = 0;
  if (p->heads) ptrs |= (uintptr_t)a.q | (uintptr_t)a.q_out;
  if (p->kv_heads) ptrs |= (uintptr_t)a.k | (uintptr_t)a.k_out;
  if (ptrs & (size - 1)) {
    set_error("mv_enc_rotary: q and k must be aligned to their elements");
    return MV_ERR_INVALID;
  }
  // The last vector reaches back over the one before it, which writes the same values twice; in place, where it could read what has been turned
  // already, the pairs behind the last full vector go one by one.
  const int turned = p->adjacent ? 2 * p->pairs : p->pairs, rest = copy ? p->dim - 2 * p->pairs : 0;
  const bool reach_back = turned >= ve && !q_in_place && !k_in_place;
  a.rot_vecs = reach_back ? (turned + ve - 1) / ve : turned / ve;
  a.rot_ones = reach_back ? 0 : (turned - a.rot_vecs * ve) / (p->adjacent ? 2 : 1);
  a.copy_vecs = rest >= ve ? (rest + ve - 1) / ve : 0;
  a.copy_ones = rest >= ve ? 0 : rest;

  // tokens of a block: 1024 vectors, enough to give every thread a few, as few as that, so that small calls still spread over the card (8 pages of 1101
  // tokens x 18 heads of 128, from memory: 18.3 us with 1024 vectors a block, 22.2 with 512, 18.9 with 2048, 22.7 with 4096)
  const int64_t vectors = (p->adjacent ? 1 : 2) * a.rot_vecs + a.rot_ones + a.copy_vecs + a.copy_ones;
  int64_t tokens = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, (p->heads + (int64_t)p->kv_heads) * vectors));
  tokens = std::min<int64_t>(tokens, std::max<int64_t>(1, 32768 / std::max<int64_t>(8, (int64_t)p->pairs * 8)));
  a.tokens = (int32_t)std::min<int64_t>(tokens, total);
  const int64_t blocks = (total + a.tokens - 1) / a.tokens;
  if (blocks * 256 > 0xffffffff /* threads of a launch */ || (int64_t)a.tokens * (p->heads + p->kv_heads) * p->dim > 0x7fffffff) {
    set_error("mv_enc_rotary: too many tokens or heads for one launch");
    return MV_ERR_INVALID;
  }
  const size_t lds = (size_t)std::max(1, a.tokens * a.pairs) * sizeof(float2);
  DeviceGuard g(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->dtype == MV_F32) launch_rotary<0>(a, p->adjacent, (unsigned)blocks, lds, s);
  else if (p->dtype == MV_BF16) launch_rotary<1>(a, p->adjacent, (unsigned)blocks, lds, s);
  else launch_rotary<2>(a, p->adjacent, (unsigned)blocks, lds, s);
  MV_HIP(hipGetLastError());
  return MV_OK;
}

}  // extern "C"
