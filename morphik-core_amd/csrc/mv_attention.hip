// mv_attention.hip -- attention of the encoder blocks over key ranges (reference formulation: model(**processor(x)),
// core/embedding/colpali_embedding_model.py:251-262, 275-305; the attention is inside transformers' SigLIP / Gemma / Qwen2-VL blocks).
//
//   s_ij = scale * q_i . k_j,   with a cap c:  s_ij = c * tanh(s_ij / c)
//   o_i  = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)   over the keys lo_i <= j < hi_i;  an empty range gives zeros.
//
// A key range per row is every mask these encoders use: padding on either side, causal, a prefix that sees itself, documents or windows
// packed one behind the other.  Heads that share a K/V head are rows of ONE problem (row r = position r / group, head r % group): K and V
// are read once for all of them, and a single position still fills a matrix instruction.
#include <algorithm>
#include <cmath>

#include "mv_common.h"
#include "mv_index_priv.h"

namespace mv {
namespace {

using u32x2 = __attribute__((ext_vector_type(2))) unsigned int;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned int;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using lds_u32x4 = __attribute__((address_space(3))) u32x4;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kWaveRows = 32;                  // rows of a wave: the N of the 32x32x16 matrix instruction
constexpr int kBlockRows = kWaves * kWaveRows;
constexpr float kRescale = 8.f;                // running maxima move only when a score passes them by 2^8: the weights stay <= 256

constexpr int64_t kMaxRowStride = 1 << 23;    // elements: a tile's byte offsets stay below 2^31

struct AttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  const int32_t* ranges;  // [batch or 1][rows][2] or null: every row sees every key
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, o_b, o_l, o_h, range_b;  // strides in elements
  int32_t rows, keys, kv_heads, group, dim, tiles;  // tiles: blocks of kBlockRows over rows * group
  float qk;    // scale * log2(e); with a cap: scale / cap * 2 log2(e)
  float cap;   // cap * log2(e), 0 = none
};

template <bool BF16>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // round to nearest even
  const f32x2 v = {a, b};
  if constexpr (BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

template <bool BF16>
__device__ __forceinline__ float unpack(uint16_t h) {
  if constexpr (BF16) return __uint_as_float((uint32_t)h << 16);
  else return (float)__builtin_bit_cast(_Float16, h);
}

// log2 of the weight's numerator from the raw product q.k (see AttnArgs::qk)
template <bool CAP>
__device__ __forceinline__ float score(float s, float qk, float cap) {
  if constexpr (CAP) {  // cap * tanh(x) = cap - 2 cap / (1 + e^2x): 2e-7 of the cap off at worst, far below the weights' rounding
    const float e = __builtin_amdgcn_exp2f(s * qk);
    return __builtin_fmaf(-2.f * cap, __builtin_amdgcn_rcpf(1.f + e), cap);
  } else {
    return s * qk;
  }
}

// The rows of a wave once more, one key at a time with a select per key, for rows whose result is not finite: a matrix product with the
// weight 0 of a masked key would carry that key's NaN or infinity into the row.  Rare by nature (only where masked places hold such values, or
// where the row's own operands do), so it is simple rather than fast.
template <bool BF16, bool CAP>
__device__ void exact_row(const AttnArgs& a, const uint16_t* q, const uint16_t* k, const uint16_t* v, int lo, int hi, uint16_t* out) {
  const int lane = threadIdx.x & 63;
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) qv[c] = c * 64 + lane < a.dim ? unpack<BF16>(q[c * 64 + lane]) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; ++j) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + lane < a.dim) s = __builtin_fmaf(qv[c], unpack<BF16>(k[(int64_t)j * a.k_l + c * 64 + lane]), s);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
    const float t = score<CAP>(s, a.qk, a.cap);
    const float m2 = t > m ? t : m;
    const float alpha = m2 == m ? 1.f : __builtin_amdgcn_exp2f(m - m2);
    const float p = m2 == -INFINITY ? (t != t ? t : 0.f) : __builtin_amdgcn_exp2f(t - m2);
    m = m2;
    l = __builtin_fmaf(l, alpha, p);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + lane < a.dim) o[c] = __builtin_fmaf(o[c], alpha, p * unpack<BF16>(v[(int64_t)j * a.v_l + c * 64 + lane]));
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c * 64 + lane < a.dim) out[c * 64 + lane] = (uint16_t)pack2<BF16>(o[c] / l, 0.f);
}

// Where a 16-byte chunk of a staged row lies: chunk c of row r at r * CH + (c ^ swizzle(r)).  LDS serves 256 bytes a cycle: 16 lanes of a K read
// (one row each, the same column) and 32 lanes of a V read (four rows x four chunks each) have to meet all 16 chunk positions.
template <int CH>
__device__ __forceinline__ int swizzle_k(int r) {
  if constexpr (CH % 16 == 0) return r & 15;
  else if constexpr (CH % 8 == 0) return (r >> 1) & 7;
  else if constexpr (CH % 4 == 0) return (r >> 2) & 3;
  else return (r >> 3) & 1;
}
template <int CH>
__device__ __forceinline__ int swizzle_v(int r) {
  if constexpr (CH % 16 == 0) return (r & 3) << 2;
  else if constexpr (CH % 8 == 0) return ((r >> 1) & 1) << 2;
  else return 0;
}

// 64 lanes x 16 bytes from base + offset (per lane) to 1 KiB of LDS at `slot`, without passing through registers; lanes off in exec leave their 16 bytes
// alone.  The compiler does not count it: whoever reads the LDS waits with tile_barrier.
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, uint32_t slot) {
  uint32_t keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %1, %3\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(offset), "s"(slot), "s"(base)
      : "memory");
}
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// One block: 128 rows against the keys that any of them sees, in tiles of BK keys staged through LDS.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds 16 keys of ONE row per 32 x 32 product, so the softmax is arithmetic within
// the lane and one exchange with lane ^ 32.  The second product is transposed too, O^T = V^T P^T: its weight operand wants, per lane, eight
// keys of one row -- the very registers the first product left, when V is read in the same order of keys.  V^T comes out of LDS by the
// transposing read: 16 lanes that address four keys x 16 columns get one column each, four keys deep.
//
// Tiles are double-buffered: while one is computed the next is on its way from memory to LDS, and one barrier a tile both publishes the
// arrived one and frees the other.
template <bool BF16, int KC, int BK, bool CAP>
__global__ __launch_bounds__(kWaves * 64, 2) void attention_kernel(const AttnArgs a) {
  constexpr int DT = (KC + 1) / 2;             // 32-column tiles of the output; KC: 16-column steps of q.k
  constexpr int CH = 2 * KC;                   // 16-byte chunks of a row
  constexpr int VC = DT * 4;                   // and of a staged row of V (the last tile's unused columns hold anything: their results are dropped)
  constexpr int kThreads = kWaves * 64;
  constexpr int kLoadsK = (BK * CH + kThreads - 1) / kThreads, kLoadsV = (BK * VC + kThreads - 1) / kThreads;
  __shared__ __attribute__((aligned(1024))) u32x4 lds_k[2][BK * CH], lds_v[2][BK * VC];
  __shared__ int lds_range[kWaves][2];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;

  int id = blockIdx.x;
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const uint16_t* kb = a.k + b * a.k_b + hk * a.k_h;
  const uint16_t* vb = a.v + b * a.v_b + hk * a.v_h;

  // this lane's row
  const int64_t r = (int64_t)tile * kBlockRows + wave * kWaveRows + (lane & 31);
  const bool live = r < (int64_t)a.rows * a.group;
  const int pos = live ? (int)(r / a.group) : 0, head = hk * a.group + (live ? (int)(r % a.group) : 0);
  int lo = 0, hi = live ? a.keys : 0;
  if (live && a.ranges) {
    const int2 rg = *reinterpret_cast<const int2*>(a.ranges + b * a.range_b + (int64_t)pos * 2);
    lo = max(rg.x, 0);
    hi = min(rg.y, a.keys);
  }
  if (lo >= hi) lo = hi = 0;
  const bool empty = lo == hi;

  // keys that some row of the wave sees [w_lo, w_hi), that every row sees [in_lo, in_hi); the block's tiles cover all waves'
  int w_lo = empty ? 0x7fffffff : lo, w_hi = hi, in_lo = lo, in_hi = empty ? 0x7fffffff : hi;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    w_lo = min(w_lo, __shfl_xor(w_lo, s));
    w_hi = max(w_hi, __shfl_xor(w_hi, s));
    in_lo = max(in_lo, __shfl_xor(in_lo, s));
    in_hi = min(in_hi, __shfl_xor(in_hi, s));
  }
  w_lo = uniform(w_lo), w_hi = uniform(w_hi), in_lo = uniform(in_lo), in_hi = uniform(in_hi);
  if (lane == 0) {
    lds_range[wave][0] = w_lo;
    lds_range[wave][1] = w_hi;
  }
  __syncthreads();
  int k_lo = 0x7fffffff, k_hi = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    k_lo = min(k_lo, lds_range[w][0]);
    k_hi = max(k_hi, lds_range[w][1]);
  }
  k_lo = uniform(k_lo), k_hi = uniform(k_hi);

  // q: the columns 16 kk + 8 half ... + 7 of this lane's row
  const uint16_t* qr = a.q + b * a.q_b + (int64_t)pos * a.q_l + head * a.q_h;
  s16x8 qf[KC];
#pragma unroll
  for (int kk = 0; kk < KC; ++kk) {
    const int c = kk * 16 + half * 8;
    qf[kk] = live && c < a.dim ? *reinterpret_cast<const s16x8*>(qr + c) : s16x8{};
  }

  // staging: thread t moves the chunks at positions t, t + 256, ... of a tile.  Rows behind the last key are copies of it, columns behind the last
  // one copies of the first (a row that is finite stays so; the weights and the columns of q there are zero)
  const uint32_t k_step = (uint32_t)a.k_l * 2, v_step = (uint32_t)a.v_l * 2;
  auto place = [&](int i, int n, int sw, uint32_t step, int last) {
    const int row = i / n;
    int c = i % n ^ sw;
    c = c * 8 < a.dim ? c : 0;
    return (uint32_t)min(row, last) * step + (uint32_t)c * 16;
  };
  uint32_t k_off[kLoadsK], v_off[kLoadsV];
  auto offsets = [&](int last) {
#pragma unroll
    for (int n = 0; n < kLoadsK; ++n) k_off[n] = place(n * kThreads + threadIdx.x, CH, swizzle_k<CH>((n * kThreads + threadIdx.x) / CH), k_step, last);
#pragma unroll
    for (int n = 0; n < kLoadsV; ++n) v_off[n] = place(n * kThreads + threadIdx.x, VC, swizzle_v<VC>((n * kThreads + threadIdx.x) / VC), v_step, last);
  };
  offsets(BK);
  auto fetch = [&](int k0, int buf) {
    if (k0 + BK > k_hi) offsets(k_hi - 1 - k0);
    const uint16_t* kt = kb + (int64_t)k0 * a.k_l;
    const uint16_t* vt = vb + (int64_t)k0 * a.v_l;
    const uint32_t dk = uniform((uint32_t)(uintptr_t)(lds_u32x4*)&lds_k[buf][wave * 64]), dv = uniform((uint32_t)(uintptr_t)(lds_u32x4*)&lds_v[buf][wave * 64]);
#pragma unroll
    for (int n = 0; n < kLoadsK; ++n)
      if ((n + 1) * kThreads <= BK * CH || n * kThreads + wave * 64 < BK * CH) dma16(kt, k_off[n], dk + n * kThreads * 16);
#pragma unroll
    for (int n = 0; n < kLoadsV; ++n)
      if ((n + 1) * kThreads <= BK * VC || n * kThreads + wave * 64 < BK * VC) dma16(vt, v_off[n], dv + n * kThreads * 16);
  };

  f32x16 o[DT] = {};
  float m = -INFINITY, l = 0.f;
  if (k_lo < k_hi) fetch(k_lo, 0);

  int buf = 0;
  for (int k0 = k_lo; k0 < k_hi; k0 += BK, buf ^= 1) {
    tile_barrier();
    if (k0 + BK < k_hi) fetch(k0 + BK, buf ^ 1);
    if (k0 + BK <= w_lo || k0 >= w_hi) continue;  // nothing here for this wave

    const uint16_t* lk = reinterpret_cast<const uint16_t*>(lds_k[buf]);
    uint16_t* lv = reinterpret_cast<uint16_t*>(lds_v[buf]);
    f32x16 s[BK / 32] = {};
#pragma unroll
    for (int t = 0; t < BK / 32; ++t) {
      const int row = t * 32 + (lane & 31);
#pragma unroll
      for (int kk = 0; kk < KC; ++kk)
        s[t] = mfma<BF16>(*reinterpret_cast<const s16x8*>(lk + (row * CH + ((kk * 2 + half) ^ swizzle_k<CH>(row))) * 8), qf[kk], s[t]);
    }

    if constexpr (CAP) {
#pragma unroll
      for (int t = 0; t < BK / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = score<true>(s[t][e], a.qk, a.cap);
    }
    if (k0 < in_lo || k0 + BK > in_hi) {  // some row does not see some key of the tile
#pragma unroll
      for (int t = 0; t < BK / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = k0 + t * 32 + 8 * (e / 4) + 4 * half + e % 4;
          s[t][e] = key >= lo && key < hi ? s[t][e] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < BK / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float qk = CAP ? 1.f : a.qk;  // capped scores are logarithms already
    top *= qk;
    if (__any(top > m + kRescale)) {
      const float m2 = fmaxf(m, top);
      const float alpha = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
    // weights, rounded to the operands' type for the matrix instruction (half a step of it, below the output's own rounding)
    s16x8 p[BK / 16];
#pragma unroll
    for (int t = 0; t < BK / 32; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][c * 8 + 2 * e], qk, -base));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][c * 8 + 2 * e + 1], qk, -base));
          l += x + y;
          w[e] = pack2<BF16>(x, y);
        }
        p[t * 2 + c] = __builtin_bit_cast(s16x8, w);
      }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int c = 0; c < BK / 16; ++c) {
        // keys 16 c + 4 half + 0..3 and + 8..11 of column 32 d + (lane & 31)
        const int row = c * 16 + 4 * half + ((lane & 15) >> 2), chunk = d * 4 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        uint16_t* src = lv + (row * VC + (chunk ^ swizzle_v<VC>(row))) * 8 + 4 * (lane & 1);
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src);
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 8 * VC * 8));
        o[d] = mfma<BF16>(__builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7), p[c], o[d]);
      }
  }

  l += __shfl_xor(l, 32);
  const float inv = empty ? 0.f : 1.f / l;
  bool bad = false;
  uint16_t* orow = a.out + b * a.o_b + (int64_t)pos * a.o_l + head * a.o_h;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = d * 32 + e * 8 + half * 4;
      if (live && c < a.dim) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = o[d][e * 4 + i] * inv;
          x[i] = empty ? 0.f : y;
          bad |= !empty && !(fabsf(y) < INFINITY);
        }
        *reinterpret_cast<u32x2*>(orow + c) = u32x2{pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3])};
      }
    }
  uint64_t again = __ballot(bad);
  again = (again | again >> 32) & 0xffffffffu;
  while (again) {
    const int src = __builtin_ctzll(again);
    again &= again - 1;
    const int pos2 = __shfl(pos, src), head2 = __shfl(head, src), lo2 = __shfl(lo, src), hi2 = __shfl(hi, src);
    exact_row<BF16, CAP>(a, a.q + b * a.q_b + (int64_t)pos2 * a.q_l + head2 * a.q_h, kb, vb, lo2, hi2, a.out + b * a.o_b + (int64_t)pos2 * a.o_l + head2 * a.o_h);
  }
}

// Zero keys: every row is empty.
__global__ void zero_rows_kernel(uint32_t* out, int64_t words) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) out[i] = 0;
}

template <bool BF16, int KC, bool CAP>
void launch_attention(const AttnArgs& a, int64_t blocks, hipStream_t s) {
  constexpr int BK = KC > 8 ? 32 : 64;
  hipLaunchKernelGGL((attention_kernel<BF16, KC, BK, CAP>), dim3((unsigned)blocks), dim3(kWaves * 64), 0, s, a);
}

template <bool BF16, bool CAP>
void dispatch_dim(const AttnArgs& a, int64_t blocks, hipStream_t s) {
  const int kc = (a.dim + 15) / 16;
  if (kc <= 2) launch_attention<BF16, 2, CAP>(a, blocks, s);
  else if (kc <= 4) launch_attention<BF16, 4, CAP>(a, blocks, s);
  else if (kc == 5) launch_attention<BF16, 5, CAP>(a, blocks, s);
  else if (kc == 6) launch_attention<BF16, 6, CAP>(a, blocks, s);
  else if (kc <= 8) launch_attention<BF16, 8, CAP>(a, blocks, s);
  else if (kc <= 12) launch_attention<BF16, 12, CAP>(a, blocks, s);
  else launch_attention<BF16, 16, CAP>(a, blocks, s);
}

// ---------------------------------------------------------------- key ranges
// prefix < 0: a row sees all of its sequence; else the first `prefix` keys of it and those up to itself.
__device__ __forceinline__ int2 row_range(int64_t start, int64_t end, int64_t at, int64_t prefix) {
  if (at < start || at >= end) return make_int2(0, 0);
  int64_t hi = end;
  if (prefix >= 0) {
    hi = start + prefix < end ? start + prefix : end;
    hi = hi > at + 1 ? hi : at + 1;
  }
  return make_int2((int)(start < 0 ? 0 : start), (int)hi);
}

__global__ __launch_bounds__(256) void padded_ranges_kernel(const int32_t* starts, int64_t starts_stride, const int32_t* ends, int64_t ends_stride,
                                                            const int32_t* prefixes, int32_t prefix, int64_t total, int32_t rows, int64_t row_offset, int2* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t b = i / rows;
  out[i] = row_range(starts[b * starts_stride], ends[b * ends_stride], i % rows + row_offset, prefixes ? max(prefixes[b], 0) : prefix);
}

__global__ __launch_bounds__(256) void document_ranges_kernel(const int32_t* offsets, int32_t docs, const int32_t* prefixes, int32_t prefix, int32_t rows,
                                                              int2* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows) return;
  int lo = 0, hi = docs;  // the last document that starts at or before row i (documents of no rows lie in front of it)
  while (lo < hi) {
    const int mid = lo + ((hi - lo + 1) >> 1);
    if (offsets[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  out[i] = lo == docs ? make_int2(0, 0) : row_range(offsets[lo], offsets[lo + 1], i, prefixes ? max(prefixes[lo], 0) : prefix);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

int mv_enc_attention(int device, const mv_attn* p, void* stream) {
  if (!p || p->batch < 0 || p->rows < 0 || p->keys < 0 || p->keys > 0x7fffff00 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads) {
    set_error("mv_enc_attention: bad sizes (heads must be a positive multiple of kv_heads)");
    return MV_ERR_INVALID;
  }
  if (p->dtype != MV_BF16 && p->dtype != MV_F16) {
    set_error("mv_enc_attention: dtype must be MV_BF16 or MV_F16");
    return MV_ERR_INVALID;
  }
  if (p->dim < 8 || p->dim > 256 || p->dim % 8) {
    set_error("mv_enc_attention: head dimension %d (multiples of 8 up to 256)", p->dim);
    return MV_ERR_INVALID;
  }
  if (!(p->scale > 0.f) || !std::isfinite(p->scale) || !(p->softcap >= 0.f) || !std::isfinite(p->softcap)) {
    set_error("mv_enc_attention: scale must be positive and softcap not negative, both finite");
    return MV_ERR_INVALID;
  }
  if (p->batch == 0 || p->rows == 0) return MV_OK;
  uintptr_t all = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out);
  int64_t strides = p->q_batch | p->q_row | p->q_head;
  bool null = !p->q || !p->out;
  if (p->keys > 0) {
    all |= reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    strides |= p->k_batch | p->k_row | p->k_head | p->v_batch | p->v_row | p->v_head;
    null |= !p->k || !p->v;
  }
  if (null || (all & 15) || (strides & 7) || (reinterpret_cast<uintptr_t>(p->ranges) & 7) || (p->ranges_batch & 1)) {
    set_error("mv_enc_attention: pointers must be set and 16-byte aligned, strides multiples of 8 elements");
    return MV_ERR_INVALID;
  }
  if (p->k_row < 0 || p->k_row > kMaxRowStride || p->v_row < 0 || p->v_row > kMaxRowStride) {
    set_error("mv_enc_attention: rows of k or v more than %lld elements apart", (long long)kMaxRowStride);
    return MV_ERR_INVALID;
  }
  AttnArgs a = {};
  a.q = reinterpret_cast<const uint16_t*>(p->q);
  a.k = reinterpret_cast<const uint16_t*>(p->k);
  a.v = reinterpret_cast<const uint16_t*>(p->v);
  a.out = reinterpret_cast<uint16_t*>(p->out);
  a.ranges = reinterpret_cast<const int32_t*>(p->ranges);
  a.range_b = p->ranges_batch;
  a.q_b = p->q_batch, a.q_l = p->q_row, a.q_h = p->q_head;
  a.k_b = p->k_batch, a.k_l = p->k_row, a.k_h = p->k_head;
  a.v_b = p->v_batch, a.v_l = p->v_row, a.v_h = p->v_head;
  a.o_h = p->dim, a.o_l = (int64_t)p->heads * p->dim, a.o_b = a.o_l * p->rows;
  a.rows = p->rows, a.keys = p->keys, a.kv_heads = p->kv_heads, a.group = p->heads / p->kv_heads, a.dim = p->dim;
  if (p->softcap > 0.f) {
    a.qk = (float)((double)p->scale / p->softcap * 2.0 * 1.4426950408889634);
    a.cap = p->softcap * kLog2e;
  } else {
    a.qk = p->scale * kLog2e;
  }
  const int64_t tiles = ((int64_t)p->rows * a.group + kBlockRows - 1) / kBlockRows;
  const int64_t blocks = tiles * p->kv_heads * p->batch;
  if (tiles > 0x7fffffff || blocks > 0x7fffffff) {
    set_error("mv_enc_attention: too many rows for one launch");
    return MV_ERR_INVALID;
  }
  a.tiles = (int32_t)tiles;
  DeviceGuard g(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->keys == 0) {
    const int64_t words = (int64_t)p->batch * a.o_b / 2;
    hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)std::min<int64_t>((words + 255) / 256, 4096)), dim3(256), 0, s, reinterpret_cast<uint32_t*>(a.out), words);
  } else if (p->dtype == MV_BF16) {
    if (p->softcap > 0.f) dispatch_dim<true, true>(a, blocks, s);
    else dispatch_dim<true, false>(a, blocks, s);
  } else {
    if (p->softcap > 0.f) dispatch_dim<false, true>(a, blocks, s);
    else dispatch_dim<false, false>(a, blocks, s);
  }
  MV_HIP(hipGetLastError());
  return MV_OK;
}

int mv_enc_padded_ranges(int device, const int32_t* d_starts, int64_t starts_stride, const int32_t* d_ends, int64_t ends_stride, const int32_t* d_prefixes,
                         int32_t prefix, int32_t batch, int32_t rows, int64_t row_offset, int32_t* d_ranges, void* stream) {
  if (batch < 0 || rows < 0 || row_offset < 0 || ((int64_t)batch * rows > 0 && (!d_starts || !d_ends || !d_ranges || (reinterpret_cast<uintptr_t>(d_ranges) & 7)))) {
    set_error("mv_enc_padded_ranges: bad argument");
    return MV_ERR_INVALID;
  }
  const int64_t total = (int64_t)batch * rows;
  if (total == 0) return MV_OK;
  if ((total + 255) / 256 > 0x7fffffff) {
    set_error("mv_enc_padded_ranges: too many rows");
    return MV_ERR_INVALID;
  }
  DeviceGuard g(device);
  hipLaunchKernelGGL(padded_ranges_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), d_starts, starts_stride,
                     d_ends, ends_stride, d_prefixes, prefix, total, rows, row_offset, reinterpret_cast<int2*>(d_ranges));
  MV_HIP(hipGetLastError());
  return MV_OK;
}

int mv_enc_document_ranges(int device, const int32_t* d_offsets, int32_t docs, const int32_t* d_prefixes, int32_t prefix, int32_t rows, int32_t* d_ranges,
                           void* stream) {
  if (docs < 0 || rows < 0 || (rows > 0 && (!d_offsets || !d_ranges || (reinterpret_cast<uintptr_t>(d_ranges) & 7)))) {
    set_error("mv_enc_document_ranges: bad argument");
    return MV_ERR_INVALID;
  }
  if (rows == 0) return MV_OK;
  DeviceGuard g(device);
  hipLaunchKernelGGL(document_ranges_kernel, dim3((unsigned)(((int64_t)rows + 255) / 256)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), d_offsets, docs,
                     d_prefixes, prefix, rows, reinterpret_cast<int2*>(d_ranges));
  MV_HIP(hipGetLastError());
  return MV_OK;
}

}  // extern "C"
