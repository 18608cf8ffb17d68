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
#include <atomic>
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
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using lds_u32x4 = __attribute__((address_space(3))) u32x4;
using const_s16x8 = const __attribute__((address_space(4))) s16x8;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaveRows = 32;                  // rows of a wave: the N of the 32x32x16 matrix instruction
constexpr int kXcds = 8;
// By KC, the 16-column steps of a head.  Keys of a tile: two products deep where the registers allow it.  Waves of a SIMD at once: by registers.  Three
// would have 168 each of the 190 ... 200 that heads of 72 ... 96 take, and lose by it (8464 rows of heads of 80: 444 us with two, 475 with three).
// Waves of a block: eight share a tile's loads (2 x 4096 rows, heads of 128: 278 us with four, 270 with eight; 4 x 2048 of 256: 163 and 146), but for
// heads of 72 ... 96, whose tiles do not divide evenly among 512 threads and which vision towers use with short windows (heads of 80: 8464 rows 467 us
// with four, 543 with eight; windows of 64 rows 64 and 78).
constexpr int tile_keys(int kc) { return kc > 8 ? 32 : 64; }
constexpr int waves_per_simd(int kc) { return kc <= 4 ? 4 : 2; }
constexpr int block_waves(int kc) { return kc == 5 || kc == 6 ? 4 : 8; }
constexpr int blocks_per_cu(int kc, int waves) {  // by registers, by the 160 KB of LDS (tiles of K and V twice, 2 KB of ranges)
  const int by_waves = waves_per_simd(kc) * 4 / waves, by_lds = 160 * 1024 / (2 * tile_keys(kc) * (2 * kc + (kc + 1) / 2 * 4) * 16 + 2048);
  return by_waves < by_lds ? by_waves : by_lds;
}
constexpr int kFewWaves = 2;  // of a block of a short call: see few_waves()
// The widths that are built: a head takes the next wider one
constexpr int built_kc(int dim) { return dim <= 32 ? 2 : dim <= 64 ? 4 : dim <= 80 ? 5 : dim <= 96 ? 6 : dim <= 128 ? 8 : dim <= 192 ? 12 : 16; }
constexpr int kMatrix = 0x008, kDsRead = 0x100;  // classes of __builtin_amdgcn_sched_group_barrier
// Running maxima m move only when a score passes them by 2^rescale, and weights are 2^(score - m + lift): bf16 has the exponents of 32 bits, but in fp16 a
// weight below 2^-14 loses digits and one below 2^-25 is nothing, which thousands of weak keys beside a strong one miss (8463 keys 17.5 below it in e's
// logarithm: 2e-4 of their values, gone).  So fp16 weights fill the type up to 2^15, and what is lost lies below 2^-36 of the row's sum a key.
constexpr float rescale(bool bf16) { return bf16 ? 8.f : 4.f; }
constexpr float lift(bool bf16) { return bf16 ? 0.f : 11.f; }

// In place of a run's sum of weights: the row is not in pieces and done, the row sees nothing of the run
constexpr float kDone = -1.f, kUnseen = -2.f;

constexpr int64_t kMaxRowStride = 1 << 23;    // elements: a tile's byte offsets stay below 2^31
constexpr int64_t kMaxThreads = 0xffffffff;   // of a launch

struct AttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  const int32_t* ranges;  // [batch or 1][rows][2] or null: every row sees every key
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, o_b, o_l, o_h, range_b;  // strides in elements
  int32_t rows, keys, kv_heads, group, dim, tiles, block_rows, causal;  // tiles: blocks of block_rows over rows * group
  int32_t full, splits;  // blocks [0, full) take a tile each; the tiles behind them are cut into `splits` runs of keys, one block each
  float* partial;        // of those: [tile - full][split][rows of a tile] x (dim sums, maximum, sum of weights, 2 unused)
  float qk;    // scale * log2(e)
  float turn;  // with a cap: scale / cap * 2 log2(e), so that the score is cap * tanh(s turn ln(2) / 2)
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

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Capped scores, in log2: cap * tanh(x) of the raw product s = q.k, x = s scale / cap.
//  - From the exponential, cap (1 - 2 / (1 + e^2x)): within 2^-22 of the CAP, which is no measure of a score that is small beside it.  For caps up to
//    kNarrowCap that is 2^-15 of a weight at most (of the caps of 20 ... 50 that models use 2^-17), a sixteenth of the half step it is rounded by.
//  - As x times a polynomial in x^2 for |x| < 1/2 (least largest relative error: 2^-26), so within 2^-22 of the score itself: far below the cap it is the
//    uncapped score.  Wider caps take it, and the exponential where a wave holds a score that is further out.
// us without a cap, with a narrow one, with a wide one: 2 x 4096 rows of 16 heads of 128 253, 314, 344; of 64 147, 222, 236; 4 x 2048 rows of 8 heads of 256
// 130, 150, 172; 8464 rows of 16 heads of 80 456, 577, 668.  Tried for the wide ones: both forms and a select for every score (432 and 344 at 128 and 64
// columns), one of two loops by the tile's largest score (31 and 41 spilled registers at 64 and 256).
enum Cap { kNoCap, kNarrow, kWide };
constexpr float kNarrowCap = 100.f;
constexpr float kNear = 1.4426950408889634f;        // |s turn| of |x| = 1/2
constexpr float kHalfLn2Sq = 0.12011325347955035f;  // (ln(2) / 2)^2: x^2 = (s turn)^2 of these
__device__ __forceinline__ float cap_far(float s, float turn, float cap) {
  return cap * __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * turn)), 1.f);  // twice the cap may be more than 32 bits hold
}
__device__ __forceinline__ float cap_near(float s, float qk, float turn) {
  constexpr float k1 = -0.333331436f * kHalfLn2Sq, k2 = 0.13325879f * kHalfLn2Sq * kHalfLn2Sq, k3 = -0.0530455038f * kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq,
                  k4 = 0.0172415134f * kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq * kHalfLn2Sq;
  const float y = s * turn, z = y * y;
  return s * qk * __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(k4, z, k3), z, k2), z, k1), z, 1.f);
}

// log2 of the weight's numerator from the raw product q.k
template <int CAP>
__device__ __forceinline__ float score(const AttnArgs& a, float s) {
  if constexpr (CAP == kNoCap) return s * a.qk;
  else if constexpr (CAP == kNarrow) return __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * a.turn)), a.cap);
  else {
    const float near = cap_near(s, a.qk, a.turn);
    const bool is_far = !(fabsf(s) * a.turn < kNear);
    if (__builtin_expect(__any(is_far), 0) && is_far) return cap_far(s, a.turn, a.cap);
    return near;
  }
}

// Which rows of a wave (a bit each) may owe a result that is not finite to something they do not see.  In the matrix products a value that is not finite
// counts even under a zero: the values of a masked key of the tile under its weight, and in heads narrower than the kernel an infinite first chunk of K,
// which stands in for the columns that q holds zeros for.  All other rows are right as they are, also those that are not a number by a score of their own.
// One lane a key, over the tiles that this wave worked on; q, lo and hi are the lane's row and its range.
template <bool BF16, int KC, int CAP>
__device__ uint32_t spoiled_rows(const AttnArgs& a, const uint16_t* q, const uint16_t* k, const uint16_t* v, int k_lo, int k_hi, int w_lo, int w_hi, int in_lo,
                                 int in_hi, int lo, int hi) {
  constexpr int BK = tile_keys(KC);
  constexpr uint32_t kTop = BF16 ? 0x7f80 : 0x7c00;  // all bits of the exponent
  const int lane = threadIdx.x & 63;
  const bool narrow = a.dim < KC * 16;
  bool hit = false, lost = false;
  for (int k0 = k_lo; k0 < k_hi; k0 += BK) {
    const bool cut = k0 < in_lo || k0 + BK > in_hi;
    if (k0 + BK <= w_lo || k0 >= w_hi || !(cut || narrow)) continue;
    const bool mine = lane < BK && k0 + lane < k_hi;
    bool odd = false, inf = false;
    if (mine && cut) {
      const uint16_t* row = v + (int64_t)(k0 + lane) * a.v_l;
#pragma unroll 4
      for (int c = 0; c < a.dim; c += 8) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (w[e] & kTop) == kTop || (w[e] & kTop << 16) == kTop << 16;
      }
    }
    if (mine && narrow) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(k + (int64_t)(k0 + lane) * a.k_l);
#pragma unroll
      for (int e = 0; e < 4; ++e) inf |= (w[e] & 0x7fff) == kTop || (w[e] >> 16 & 0x7fff) == kTop;
    }
    const uint64_t odds = __ballot(odd), infs = __ballot(inf);
    const int from = min(max(lo - k0, 0), 64), to = min(max(hi - k0, 0), 64);
    const uint64_t sees = from < to ? ~0ull >> (64 - (to - from)) << from : 0;
    hit |= ((odds & ~sees) | (infs & sees)) != 0;
    if (k0 + BK > k_hi) hit |= odds >> (k_hi - 1 - k0) & 1;  // the rows behind the last key are copies of it, under weights of 0
    if (CAP != kNoCap) continue;  // a cap makes every infinite score finite
    for (uint64_t left = infs; left; left &= left - 1) {
      const int at = __builtin_ctzll(left);
      const bool asks = sees >> at & 1 && !lost;
      if (!__any(asks)) continue;
      const uint16_t* row = k + (int64_t)(k0 + at) * a.k_l;
      float s = 0.f;
      if (asks) {
#pragma unroll 2
        for (int c = 0; c < a.dim; c += 8) {
          const s16x8 qc = *reinterpret_cast<const s16x8*>(q + c), kc = *reinterpret_cast<const s16x8*>(row + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) s = __builtin_fmaf(unpack<BF16>((uint16_t)qc[e]), unpack<BF16>((uint16_t)kc[e]), s);
        }
        lost = s != -INFINITY;
      }
    }
  }
  const uint64_t hits = __ballot(hit && !lost);
  return (uint32_t)(hits | hits >> 32);
}

// Those rows once more, R of them at a time by a whole wave, with what a row does not see selected away: scores one key a lane, then the 64 keys'
// values, four columns a lane.
struct AgainRow {
  const uint16_t* q;
  uint16_t* out;
  float* partial;
  int lo, hi;
};
template <bool BF16, int CAP, int R>
__device__ void exact_rows(const AttnArgs& a, const AgainRow (&rows)[R], int count, const uint16_t* k, const uint16_t* v) {
  const int lane = threadIdx.x & 63, col = lane * 4;
  f32x4 o[R];
  float m[R], l[R];
  int from = 0x7fffffff, to = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    o[r] = f32x4{}, m[r] = -INFINITY, l[r] = 0.f;
    from = min(from, rows[r].lo), to = max(to, rows[r].hi);
  }
  for (int j0 = from; j0 < to; j0 += 64) {
    bool any = false;
#pragma unroll
    for (int r = 0; r < R; ++r) any |= rows[r].lo < j0 + 64 && rows[r].hi > j0;
    if (!any) continue;
    const int n = min(to - j0, 64), j = j0 + lane;
    const uint16_t* kr = k + (int64_t)(j0 + min(lane, n - 1)) * a.k_l;
    float s[R] = {};
#pragma unroll 2
    for (int c = 0; c < a.dim; c += 8) {
      const s16x8 kc = *reinterpret_cast<const s16x8*>(kr + c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const s16x8 qc = *(const_s16x8*)(uintptr_t)(rows[r].q + c);  // the same for all lanes: a scalar load
#pragma unroll
        for (int e = 0; e < 8; ++e) s[r] = __builtin_fmaf(unpack<BF16>((uint16_t)qc[e]), unpack<BF16>((uint16_t)kc[e]), s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool sees = j >= rows[r].lo && j < rows[r].hi;
      const float t = score<CAP>(a, s[r]);
      float m2 = sees ? fmaxf(m[r], t) : m[r];
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) m2 = fmaxf(m2, __shfl_xor(m2, x));
      const float alpha = m2 == m[r] ? 1.f : __builtin_amdgcn_exp2f(m[r] - m2);
      const float p = m2 == -INFINITY ? (t != t ? t : 0.f) : __builtin_amdgcn_exp2f(t - m2);
      m[r] = m2;
      l[r] = __builtin_fmaf(l[r], alpha, sees ? p : 0.f);
      o[r] *= alpha;
      s[r] = sees ? p : -1.f;  // not seen
    }
    const uint16_t* vr = v + (int64_t)j0 * a.v_l + (col < a.dim ? col : 0);
#pragma unroll 4
    for (int i = 0; i < n; ++i, vr += a.v_l) {
      const s16x4 vc = *reinterpret_cast<const s16x4*>(vr);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s[r]), i));
        if (w < 0.f) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] = __builtin_fmaf(w, unpack<BF16>((uint16_t)vc[e]), o[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= count) break;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l[r] += __shfl_xor(l[r], x);
    if (col < a.dim) {
      if (rows[r].partial) *reinterpret_cast<f32x4*>(rows[r].partial + col) = o[r];
      else *reinterpret_cast<u32x2*>(rows[r].out + col) = u32x2{pack2<BF16>(o[r][0] / l[r], o[r][1] / l[r]), pack2<BF16>(o[r][2] / l[r], o[r][3] / l[r])};
    }
    if (rows[r].partial && lane == 0) *reinterpret_cast<float2*>(rows[r].partial + a.dim) = make_float2(m[r], l[r]);
  }
}

using const_args = const __attribute__((address_space(4))) AttnArgs;

// The end of a wave with rows (a bit each in `again`) whose result is not finite.  2048 rows of 8 heads of 128 in 46 us: 46 when every row sees an infinite
// value, 106 when a causal mask hides it from the rows in front of it, 205 in pages beside it.  Not inlined, and with the kernel's arguments read anew:
// inlined, its scalar registers crowd the loop's (4 x 2048 rows of heads of 256 136 -> 145 us).
template <bool BF16, int KC, int CAP>
__attribute__((noinline)) __device__ void mend_rows(const_args* args, uint32_t again_, int b_, int hk_, int pos, int head, int lo, int hi, int k_lo_, int k_hi_,
                                                    int w_lo_, int w_hi_, int in_lo_, int in_hi_, float* partial_, bool cut_) {
  const uint64_t at = (uint64_t)args;
  const AttnArgs& a = *(const AttnArgs*)(const_args*)((uint64_t)(uint32_t)uniform((int)(at >> 32)) << 32 | (uint32_t)uniform((int)at));
  const int b = uniform(b_), hk = uniform(hk_);
  const uint16_t *k = a.k + b * a.k_b + hk * a.k_h, *v = a.v + b * a.v_b + hk * a.v_h;
  float* partial = uniform(cut_) ? partial_ : nullptr;
  uint32_t again = uniform(again_);
  again &= spoiled_rows<BF16, KC, CAP>(a, a.q + b * a.q_b + (int64_t)pos * a.q_l + head * a.q_h, k, v, uniform(k_lo_), uniform(k_hi_), uniform(w_lo_), uniform(w_hi_),
                                       uniform(in_lo_), uniform(in_hi_), lo, hi);
  while (again) {
    constexpr int kAgain = 8;
    AgainRow rows[kAgain];
    int count = 0;
#pragma unroll
    for (int i = 0; i < kAgain; ++i) {
      const int src = again ? __builtin_ctz(again) : 0;
      const int64_t pos2 = uniform(__shfl(pos, src)), head2 = uniform(__shfl(head, src));
      rows[i] = {a.q + b * a.q_b + pos2 * a.q_l + head2 * a.q_h, a.out + b * a.o_b + pos2 * a.o_l + head2 * a.o_h, partial ? partial + src * (a.dim + 4) : nullptr,
                 again ? uniform(__shfl(lo, src)) : 0x7fffffff, again ? uniform(__shfl(hi, src)) : 0};
      count += again != 0;
      again &= again - 1;
    }
    exact_rows<BF16, CAP, kAgain>(a, rows, count, k, v);
  }
}

// Where a 16-byte chunk of a staged row lies: chunk c of row r at r * CH + (c ^ swizzle(r)).  LDS serves 256 bytes a cycle: 16 lanes of a K read
// (one row each, the same column) and 32 lanes of a V read (four rows x four chunks each) have to meet all 16 chunk positions.  Measured: no
// conflict at any width.
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
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %2"
      :
      : "v"(offset), "s"(slot), "s"(base)
      : "memory", "m0");
}
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float first_lane(float x) { return __int_as_float(uniform(__float_as_int(x))); }

// One block: 32 rows a wave against the keys that any of them sees, in tiles of BK keys staged through LDS.
//
// Scores are computed transposed, S^T = K Q^T: a lane then holds 16 keys of ONE row per 32 x 32 product, so the softmax is arithmetic within
// the lane and one exchange with lane ^ 32.  The second product is transposed too, O^T = V^T P^T: its weight operand wants, per lane, eight
// keys of one row -- the very registers the first product left, when V is read in the same order of keys.  V^T comes out of LDS by the
// transposing read: 16 lanes that address four keys x 16 columns get one column each, four keys deep.
//
// Tiles are double-buffered: while one is computed the next is on its way from memory to LDS, and one barrier a tile both publishes the
// arrived one and frees the other (three or four places instead of two: no gain at any width).
//
// What bounds it: a SIMD's two waves share the matrix unit and the vector unit (busy 0.51 and 0.45 of the time at 128 columns, 0.46 and 0.58 at 80, 0.45 and
// 0.29 at 256, 0.40 and 0.63 at 64, where four waves share them) -- reads of LDS, the exchange of maxima and the barrier leave gaps that they do not fill.
// One MI355X, whose library reaches 1.30 PFLOP/s in a large bf16 product: 2 x 4096 rows of 16 heads of 128 250 us (1.10 PFLOP/s), of 64 146 ... 155 us (0.92),
// 4 x 2048 rows of 8 heads of 256 over one K/V head 130 us (1.06), 8464 rows of 16 heads of 80 437 us (0.84; the 16-column and 32-column steps round 80 up
// to 80 and 96).  Tried and not kept: two
// groups of waves half a tile apart (289 us at 128), the weights of 32 keys beside the products of the next 32 (292), 64 rows a wave
// (289, and 209 at 256), wave priorities (no change).
template <bool BF16, int KC, int CAP, int kWaves>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(waves_per_simd(KC), waves_per_simd(KC)))) void attention_kernel(
    const AttnArgs a) {
  constexpr int kBlockRows = kWaves * kWaveRows;
  constexpr int BK = tile_keys(KC);
  constexpr int DT = (KC + 1) / 2;             // 32-column tiles of the output; KC: 16-column steps of q.k
  constexpr int CH = 2 * KC;                   // 16-byte chunks of a row
  constexpr int VC = DT * 4;                   // and of a staged row of V (the last tile's unused columns hold anything: their results are dropped)
  constexpr int kThreads = kWaves * 64;
  constexpr int kLoadsK = (BK * CH + kThreads - 1) / kThreads, kLoadsV = (BK * VC + kThreads - 1) / kThreads;
  __shared__ u32x4 lds_k[2][BK * CH], lds_v[2][BK * VC];
  __shared__ int lds_range[kWaves][2];
  __shared__ int2 lds_rows[kBlockRows];  // the rows' key ranges: two registers less in the loop, where heads of 256 have none to spare (144 -> 136 us)
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;

  // Blocks of one K/V head next to each other on one XCD (its L2 then holds that head's keys once): consecutive block numbers go round the XCDs, so
  // number x + 8 i becomes the i-th of XCD x's run.  The cut tiles, of equal length among themselves, are dealt out the same way behind the others.
  const int run = blockIdx.x < a.full ? a.full : gridDim.x - a.full;
  const int at = blockIdx.x < a.full ? blockIdx.x : blockIdx.x - a.full;
  const int x = at & (kXcds - 1), each = run / kXcds, more = run % kXcds;
  int id = x * each + min(x, more) + at / kXcds, split = 0;
  float* partial = nullptr;
  if (blockIdx.x >= a.full) {
    split = id % a.splits;
    id /= a.splits;
    if (a.splits > 1) partial = a.partial + ((int64_t)id * a.splits + split) * min((int64_t)kBlockRows, (int64_t)a.rows * a.group) * (a.dim + 4);
    id += a.full;
  }
  const int tile = a.tiles - 1 - id % a.tiles;  // the last rows first: under a causal mask they have the most to do
  id /= a.tiles;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const uint16_t* kb = a.k + b * a.k_b + hk * a.k_h;
  const uint16_t* vb = a.v + b * a.v_b + hk * a.v_h;

  // this lane's row
  const uint32_t all = (uint32_t)a.rows * (uint32_t)a.group;  // below 2^31
  // keys that some row of the wave sees [w_lo, w_hi), that every row sees [in_lo, in_hi); the block's tiles cover all waves'
  int w_lo = 0x7fffffff, w_hi = 0, in_lo = 0, in_hi = 0x7fffffff;
  const uint32_t r = (uint32_t)tile * kBlockRows + wave * kWaveRows + (lane & 31);
  const bool live = r < all;
  int pos = live ? (int)(r / (uint32_t)a.group) : 0, head = hk * a.group + (live ? (int)(r % (uint32_t)a.group) : 0);
  // q: the columns 16 kk + 8 half ... + 7 of this lane's row
  const uint16_t* qr = a.q + b * a.q_b + (int64_t)pos * a.q_l + head * a.q_h;
  s16x8 qf[KC];
#pragma unroll
  for (int kk = 0; kk < KC; ++kk) {
    const int c = kk * 16 + half * 8;
    qf[kk] = live && c < a.dim ? *reinterpret_cast<const s16x8*>(qr + c) : s16x8{};
  }
  int lo = 0, hi = live ? a.keys : 0;
  if (live && a.ranges) {
    const int2 rg = *reinterpret_cast<const int2*>(a.ranges + b * a.range_b + (int64_t)pos * 2);
    lo = max(rg.x, 0);
    hi = min(rg.y, a.keys);
  } else if (live && a.causal) {
    hi = (int)min((int64_t)pos + 1 + a.keys - a.rows, (int64_t)a.keys);
  }
  if (lo >= hi) {
    lo = hi = 0;
  } else {
    w_lo = in_lo = lo;
    w_hi = in_hi = hi;
  }
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
  if (half == 0) lds_rows[wave * kWaveRows + lane] = make_int2(lo, hi);
  __syncthreads();
  int k_lo = 0x7fffffff, k_hi = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    k_lo = min(k_lo, lds_range[w][0]);
    k_hi = max(k_hi, lds_range[w][1]);
  }
  k_lo = uniform(k_lo), k_hi = uniform(k_hi);
  if (k_lo >= k_hi) k_lo = k_hi = 0;  // no row of the block sees anything: positions stay far from the end of 32 bits
  if (partial) {
    const int tiles = (k_hi - k_lo + BK - 1) / BK;
    const int pieces = max(min(a.splits, tiles / 2), 1);  // short ranges stay in one piece
    if (pieces == 1) {
      if (split) return;
      if (live && half == 0) *reinterpret_cast<float2*>(partial + (wave * kWaveRows + lane) * (a.dim + 4) + a.dim) = make_float2(-INFINITY, kDone);
      partial = nullptr;
    } else {
      const int share = (tiles + pieces - 1) / pieces * BK;  // whole tiles
      k_lo = (int)min((int64_t)k_lo + (int64_t)split * share, (int64_t)k_hi);
      k_hi = (int)min((int64_t)k_lo + share, (int64_t)k_hi);
    }
  }

  // q has arrived before the tiles' loads start: the compiler would wait for it inside the loop, and with it for the tile just sent for (8464 rows of heads
  // of 80: 479 -> 447 us)
#pragma unroll
  for (int kk = 0; kk < KC; ++kk) asm volatile("" : "+v"(qf[kk]));

  // Staging: thread t moves the chunks at positions t, t + kThreads, ... of a tile.  Rows behind the last key are copies of it, columns behind the last
  // one copies of the first (a row that is finite stays so; the weights and the columns of q there are zero).  Where kThreads positions are whole rows and
  // whole periods of the swizzle, the chunks of a thread differ by whole rows: one register of offsets, but for the last tile.
  constexpr bool kEven = kThreads % CH == 0 && kThreads / CH % 16 == 0 && VC == CH;
  constexpr int kOffsets = kEven ? 1 : (kLoadsK > kLoadsV ? kLoadsK : kLoadsV);
  const uint32_t k_step = (uint32_t)a.k_l * 2, v_step = (uint32_t)a.v_l * 2;
  auto place_k = [&](int n, int last) {
    const int i = n * kThreads + threadIdx.x, row = i / CH, c = i % CH ^ swizzle_k<CH>(row);
    return (uint32_t)min(row, last) * k_step + (c * 8 < a.dim ? c * 16 : 0);
  };
  auto place_v = [&](int n, int last) {
    const int i = n * kThreads + threadIdx.x, row = i / VC, c = i % VC ^ swizzle_v<VC>(row);
    return (uint32_t)min(row, last) * v_step + (c * 8 < a.dim ? c * 16 : 0);
  };
  uint32_t k_off[kOffsets], v_off[kOffsets];
#pragma unroll
  for (int n = 0; n < kOffsets; ++n) k_off[n] = place_k(n, BK), v_off[n] = place_v(n, BK);
  const uint16_t *kt = kb + (int64_t)k_lo * a.k_l, *vt = vb + (int64_t)k_lo * a.v_l;  // of the tile sent for next
  const uint32_t dk = uniform((uint32_t)(uintptr_t)(lds_u32x4*)&lds_k[0][wave * 64]), dv = uniform((uint32_t)(uintptr_t)(lds_u32x4*)&lds_v[0][wave * 64]);
  auto fetch = [&](int k0, int buf) {
    const uint32_t sk = dk + buf * (BK * CH * 16), sv = dv + buf * (BK * VC * 16);
    const int last = k_hi - 1 - k0;
    if (last >= BK - 1) {
#pragma unroll
      for (int n = 0; n < kLoadsK; ++n)
        if ((n + 1) * kThreads <= BK * CH || n * kThreads + wave * 64 < BK * CH)
          dma16(kEven ? kt + n * (kThreads / CH) * a.k_l : kt, k_off[kEven ? 0 : n], sk + n * kThreads * 16);
#pragma unroll
      for (int n = 0; n < kLoadsV; ++n)
        if ((n + 1) * kThreads <= BK * VC || n * kThreads + wave * 64 < BK * VC)
          dma16(kEven ? vt + n * (kThreads / VC) * a.v_l : vt, v_off[kEven ? 0 : n], sv + n * kThreads * 16);
    } else {
#pragma unroll
      for (int n = 0; n < kLoadsK; ++n)
        if ((n + 1) * kThreads <= BK * CH || n * kThreads + wave * 64 < BK * CH) dma16(kt, place_k(n, last), sk + n * kThreads * 16);
#pragma unroll
      for (int n = 0; n < kLoadsV; ++n)
        if ((n + 1) * kThreads <= BK * VC || n * kThreads + wave * 64 < BK * VC) dma16(vt, place_v(n, last), sv + n * kThreads * 16);
    }
    kt += a.k_l * BK;
    vt += a.v_l * BK;
  };

  f32x16 o[DT] = {};
  float m = -INFINITY, l = 0.f;
  const float qk = CAP == kNoCap ? a.qk : 1.f;  // capped scores are logarithms already
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
      for (int kk = 0; kk < KC; ++kk) {
        const s16x8 kf = *reinterpret_cast<const s16x8*>(lk + (row * CH + ((kk * 2 + half) ^ swizzle_k<CH>(row))) * 8);
        s[t] = mfma<BF16>(kf, qf[kk], s[t]);
      }
    }
    // reads run ahead of their products, as far as there are registers (left to itself the compiler waits for each; heads of 128: 261 -> 252 us)
    __builtin_amdgcn_sched_group_barrier(kDsRead, KC > 12 ? 3 : 6, 1);
#pragma unroll
    for (int n = 0; n < KC * BK / 32; ++n) {
      __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 1);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 1);
    }

    const bool cut = k0 < in_lo || k0 + BK > in_hi;  // some row does not see some key of the tile
    s16x8 p[BK / 16];
    if constexpr (CAP != kNoCap) {
#pragma unroll
      for (int t = 0; t < BK / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = score<CAP>(a, s[t][e]);
    }
    if (cut) {
      const int2 row = lds_rows[wave * kWaveRows + (lane & 31)];
#pragma unroll
      for (int t = 0; t < BK / 32; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = k0 + t * 32 + 8 * (e / 4) + 4 * half + e % 4;
          s[t][e] = key >= row.x && key < row.y ? s[t][e] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < BK / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
    top = fmaxf(top, __shfl_xor(top, 32)) * qk;
    if (__any(top > m + rescale(BF16))) {
      const float m2 = fmaxf(m, top);
      const float alpha = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m - lift(BF16);
    // weights, rounded to the operands' type for the matrix instruction (half a step of it, like the result's own rounding)
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
        const s16x8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
        o[d] = mfma<BF16>(vf, p[c], o[d]);
      }
    __builtin_amdgcn_sched_group_barrier(kDsRead, KC > 12 ? 4 : 8, 0);
#pragma unroll
    for (int n = 0; n < DT * BK / 16; ++n) {
      __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
    }
  }

  l += __shfl_xor(l, 32);
  uint32_t again_r = (uint32_t)tile * kBlockRows + threadIdx.x / 64 * kWaveRows + (threadIdx.x & 31);
  asm("" : "+v"(again_r));  // the row once more: two registers less across the loop
  const bool live_e = again_r < all;
  pos = live_e ? (int)(again_r / (uint32_t)a.group) : 0, head = hk * a.group + (live_e ? (int)(again_r % (uint32_t)a.group) : 0);
  const int2 row = lds_rows[wave * kWaveRows + (lane & 31)];
  const int lo_s = max(row.x, k_lo), hi_s = min(row.y, k_hi);  // what this block saw of the row's range
  const bool nothing = lo_s >= hi_s;
  const float inv = partial ? 1.f : 1.f / l;
  float odd = 0.f;  // NaN from the first value on that is not finite
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[d][e] *= inv;
      if (d * 32 + e / 4 * 8 < a.dim) odd = __builtin_fmaf(o[d][e], 0.f, odd);
    }
  const bool bad = live_e && !nothing && odd != odd;
  uint16_t* orow = a.out + b * a.o_b + (int64_t)pos * a.o_l + head * a.o_h;
  float* prow = partial + (wave * kWaveRows + (lane & 31)) * (a.dim + 4);
  // columns 32 d + 8 e + 4 half + 0..3 of this lane's row
  if (!partial) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d * 32 + e * 8 < a.dim && live_e) {
          const u32x2 w = {pack2<BF16>(o[d][e * 4], o[d][e * 4 + 1]), pack2<BF16>(o[d][e * 4 + 2], o[d][e * 4 + 3])};
          *reinterpret_cast<u32x2*>(orow + d * 32 + e * 8 + half * 4) = nothing ? u32x2{0, 0} : w;
        }
  } else if (live_e) {
    if (half == 0) *reinterpret_cast<float2*>(prow + a.dim) = nothing ? make_float2(-INFINITY, kUnseen) : make_float2(m - lift(BF16), l);
    if (!nothing) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d * 32 + e * 8 < a.dim)
            *reinterpret_cast<f32x4*>(prow + d * 32 + e * 8 + half * 4) = f32x4{o[d][e * 4], o[d][e * 4 + 1], o[d][e * 4 + 2], o[d][e * 4 + 3]};
    }
  }
  const uint64_t bads = __ballot(bad);
  if (bads)
    mend_rows<BF16, KC, CAP>((const_args*)__builtin_amdgcn_kernarg_segment_ptr(), (uint32_t)(bads | bads >> 32), b, hk, pos, head, lo_s, hi_s, k_lo, k_hi, w_lo, w_hi,
                             in_lo, in_hi, partial + wave * kWaveRows * (a.dim + 4), partial != nullptr);
}

// Joins the runs of keys of the cut tiles: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, join_runs of a wave at a time with the maximum moving as
// in the loop above.  W waves share a row (every W-th run each), added up in their order.  Bound by latency: what a run left lies in another XCD's L2 or
// behind it, so all loads of a round are sent for before anything is waited for (3 x 1 row of 16 heads over 16001 keys: 4.5 us; one round trip after the other 6.8).
constexpr int join_runs(int w) { return w == 1 ? 8 : 16; }
template <bool BF16, int W>
__global__ __launch_bounds__(256) void join_kernel(const AttnArgs a) {
  constexpr int kRows = 4 / W, kRuns = join_runs(W);  // rows of a block, runs of a wave in a round
  __shared__ f32x4 lds_o[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t all = (int64_t)a.rows * a.group;
  const int stored = (int)min((int64_t)a.block_rows, all), blocks = (stored + kRows - 1) / kRows;
  const int in_tile = (int)(blockIdx.x % blocks) * kRows + wave / W, cut = blockIdx.x / blocks;
  int id = a.full + cut;
  const int tile = a.tiles - 1 - id % a.tiles;
  id /= a.tiles;
  const int hk = id % a.kv_heads, b = id / a.kv_heads;
  const int64_t r = (int64_t)tile * a.block_rows + in_tile;
  const bool live = in_tile < stored && r < all;  // of the whole group of W waves
  const int64_t step = (int64_t)stored * (a.dim + 4);
  const float* src = a.partial + (int64_t)cut * a.splits * step + (int64_t)(live ? in_tile : 0) * (a.dim + 4);
  float m = -INFINITY, l = 0.f;
  bool seen = false, done = false;
  f32x4 o = {};
  const int own = uniform(wave % W), splits = live ? a.splits : 0;
  for (int s0 = 0; s0 < splits; s0 += kRuns * W) {
    float2 ml = make_float2(-INFINITY, kUnseen);  // of run s0 + lane
    if (lane < kRuns * W && s0 + lane < splits) ml = *reinterpret_cast<const float2*>(src + (s0 + lane) * step + a.dim);
    if constexpr (W == 1) {  // not in pieces after all: the row is done, and where there are many rows their sums are not worth sending for
      if (s0 == 0 && first_lane(ml.y) == kDone) return;
    }
    f32x4 part[kRuns];
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      part[i] = f32x4{};
      if (s0 + i * W + own < splits && lane * 4 < a.dim) part[i] = *reinterpret_cast<const f32x4*>(src + (s0 + i * W + own) * step + lane * 4);
    }
    if (s0 == 0) done = first_lane(ml.y) == kDone;
    float top = ml.x;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float m2 = fmaxf(m, top), alpha = m2 == m ? 1.f : __builtin_amdgcn_exp2f(m - m2);
    // below 0 where the row sees nothing of the run (its sums were never written)
    const float w = ml.y == kUnseen ? -1.f : m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m2);
    m = m2;
    l *= alpha;
    if (!(w < 0.f)) {
      seen = true;
      l = __builtin_fmaf(ml.y, w, l);
    }
    o *= alpha;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      if (s0 + i * W + own >= splits) break;
      const float wi = __shfl(w, i * W + own);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(wi < 0.f ? 0.f : part[i][e], wi, o[e]);
    }
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
  if constexpr (W > 1) {
    lds_o[wave][lane] = o;
    __syncthreads();
    if (wave % W) return;
#pragma unroll
    for (int i = 1; i < W; ++i) o += lds_o[wave + i][lane];
  }
  const float inv = __any(seen) ? 1.f / l : 0.f;  // a row whose scores are all -infinity is seen: not a number, as in one piece
  if (live && !done && lane * 4 < a.dim) {
    const int64_t pos = r / a.group, head = hk * a.group + r % a.group;
    *reinterpret_cast<u32x2*>(a.out + b * a.o_b + pos * a.o_l + head * a.o_h + lane * 4) =
        u32x2{pack2<BF16>(o[0] * inv, o[1] * inv), pack2<BF16>(o[2] * inv, o[3] * inv)};
  }
}

template <bool BF16>
void launch_join(const AttnArgs& a, int64_t cut, int64_t stored, hipStream_t s) {
  if (a.splits >= 16 && cut * stored <= 2048) hipLaunchKernelGGL((join_kernel<BF16, 4>), dim3((unsigned)(cut * stored)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((join_kernel<BF16, 1>), dim3((unsigned)(cut * ((stored + 3) / 4))), dim3(256), 0, s, a);
}

// Zero keys: every row is empty.
__global__ void zero_rows_kernel(uint32_t* out, int64_t words) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) out[i] = 0;
}

// How the tiles of a call are dealt out.  A card takes blocks_per_cu a CU at once; the tiles of the last, partly filled round are cut into
// runs of keys, as many as fill it, where what that saves (a tile takes about kTileUs per tile of keys in a filled CU) is more than writing,
// reading and joining the runs' 32-bit sums costs (kJoinUs for the launch, kJoinBytesPerUs).
struct Plan {
  int64_t waves, block_rows, blocks, full, cut, splits, bytes;
};
// Where eight-wave blocks would leave most of the card idle, blocks of two waves spread the rows over four times the CUs: where all of them fit at once and
// the keys are few enough not to be cut along instead (us, bf16: 20 rows x 8 heads of 256 12.0 -> 7.9, 32 x 39 rows x 12 of 128 9.9 -> 7.2, 4 x 256 x 8 of
// 256 26.2 -> 18.0, 4 x 500 39.3 -> 29.7, 2 x 500 x 12 of 128 20.0 -> 14.2; 1030 x 8 of 256, 33 tiles of keys, 43.1 -> 52.3, 1101 x 12 of 128, 18 tiles,
// 35.9 -> 39.5, heads of 192, 25 tiles, 33.2 -> 30.4).  Rows that fill one block either way gain little (16 x 60 x 16 of 64 6.1 -> 5.6) and are better cut (40 x 1 row of 16 heads over 500 keys
// 12.5 -> 14.9); heads of 72 ... 96, in four waves otherwise, lose (600 x 16 of 80 21.7 -> 23.5).
bool few_waves(int64_t all, int64_t keys, int64_t problems, int kc, int64_t cus) {
  constexpr int kRows = kFewWaves * kWaveRows;
  return block_waves(kc) == 8 && keys <= (all > kRows ? 16 : 2) * tile_keys(kc) && (all + kRows - 1) / kRows * problems <= 2 * cus;
}
constexpr double kTileUs = 2.3, kJoinUs = 4.0, kJoinBytesPerUs = 4e6;

Plan plan(int64_t batch, int64_t rows, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim, int64_t cus) {
  const int kc = built_kc((int)dim);
  const int64_t all = rows * (heads / kv_heads);
  Plan p = {};
  p.waves = few_waves(all, keys, kv_heads * batch, kc, cus) ? kFewWaves : block_waves(kc);
  p.block_rows = p.waves * kWaveRows;
  const int64_t slots = cus * blocks_per_cu(kc, (int)p.waves);
  p.blocks = (all + p.block_rows - 1) / p.block_rows * kv_heads * batch;
  p.full = p.blocks / slots * slots;
  p.cut = p.blocks - p.full;
  p.splits = 1;
  if (p.cut == 0) return p;
  const int64_t key_tiles = (keys + tile_keys(kc) - 1) / tile_keys(kc);
  const int64_t piece = std::min<int64_t>(p.block_rows, all) * (dim + 4) * 4;
  // t(n) = key_tiles / n * kTileUs + kJoinUs + n * moved: least at n = sqrt(key_tiles * kTileUs / moved), then evened out to whole tiles
  const double moved = 2.0 * p.cut * piece / kJoinBytesPerUs;
  int64_t n = (int64_t)std::sqrt(key_tiles * kTileUs / moved);
  n = std::min<int64_t>(n, std::min<int64_t>(slots / p.cut, key_tiles));
  if (n < 2) return p;
  const int64_t share = (key_tiles + n - 1) / n;
  n = (key_tiles + share - 1) / share;
  if (share * kTileUs + kJoinUs + n * moved < key_tiles * kTileUs) p.splits = n;
  if (p.splits > 1) p.bytes = p.cut * p.splits * piece;
  return p;
}

int cu_count(int device) {
  static std::atomic<int> known[64];
  if (device < 0 || device >= 64) return 256;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) n = 256;
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <bool BF16, int KC, int CAP>
void launch_attention(const AttnArgs& a, int64_t blocks, hipStream_t s) {
  constexpr int kMany = block_waves(KC);
  if constexpr (kMany == 8) {
    if (a.block_rows == kFewWaves * kWaveRows) {
      hipLaunchKernelGGL((attention_kernel<BF16, KC, CAP, kFewWaves>), dim3((unsigned)blocks), dim3(kFewWaves * 64), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((attention_kernel<BF16, KC, CAP, kMany>), dim3((unsigned)blocks), dim3(kMany * 64), 0, s, a);
}

template <bool BF16, int CAP>
void dispatch_dim(const AttnArgs& a, int64_t blocks, hipStream_t s) {
  switch (built_kc(a.dim)) {
    case 2: return launch_attention<BF16, 2, CAP>(a, blocks, s);
    case 4: return launch_attention<BF16, 4, CAP>(a, blocks, s);
    case 5: return launch_attention<BF16, 5, CAP>(a, blocks, s);
    case 6: return launch_attention<BF16, 6, CAP>(a, blocks, s);
    case 8: return launch_attention<BF16, 8, CAP>(a, blocks, s);
    case 12: return launch_attention<BF16, 12, CAP>(a, blocks, s);
    default: return launch_attention<BF16, 16, CAP>(a, blocks, s);
  }
}

template <bool BF16>
void dispatch_cap(const AttnArgs& a, float softcap, int64_t blocks, hipStream_t s) {
  if (softcap == 0.f) dispatch_dim<BF16, kNoCap>(a, blocks, s);
  else if (softcap <= kNarrowCap) dispatch_dim<BF16, kNarrow>(a, blocks, s);
  else dispatch_dim<BF16, kWide>(a, blocks, s);
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
  if (!p || p->batch < 0 || p->rows < 0 || p->keys < 0 || p->keys > 0x7ffff000 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads) {
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
  const int64_t k_row = p->keys > 1 ? p->k_row : 0, v_row = p->keys > 1 ? p->v_row : 0;  // one key has no step
  if (k_row < 0 || k_row > kMaxRowStride || v_row < 0 || v_row > kMaxRowStride) {
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
  a.k_b = p->k_batch, a.k_l = k_row, a.k_h = p->k_head;
  a.v_b = p->v_batch, a.v_l = v_row, a.v_h = p->v_head;
  a.o_h = p->dim, a.o_l = (int64_t)p->heads * p->dim, a.o_b = a.o_l * p->rows;
  a.rows = p->rows, a.keys = p->keys, a.kv_heads = p->kv_heads, a.group = p->heads / p->kv_heads, a.dim = p->dim, a.causal = p->causal && !p->ranges;
  a.qk = p->scale * kLog2e;
  if (p->softcap > 0.f) {
    a.turn = (float)((double)p->scale / p->softcap * 2.0 * 1.4426950408889634);
    a.cap = p->softcap * kLog2e;
  }
  if (!(a.qk > 0.f) || !std::isfinite(a.qk) || !std::isfinite(a.cap) || (p->softcap > 0.f && (!(a.turn > 0.f) || !std::isfinite(a.turn)))) {
    set_error("mv_enc_attention: scale or scale / softcap leaves 32 bits");
    return MV_ERR_INVALID;
  }
  const int64_t tall = (int64_t)p->rows * a.group;  // rows of one K/V head
  const Plan pl = plan(p->batch, p->rows, p->keys, p->heads, p->kv_heads, p->dim, cu_count(device));
  const int64_t blocks = pl.full + pl.cut * pl.splits;
  if (tall > 0x7ffff000 || pl.blocks > 0x7fffffff || blocks * pl.waves * 64 > kMaxThreads) {
    set_error("mv_enc_attention: too many rows for one launch");
    return MV_ERR_INVALID;
  }
  if (pl.bytes > 0 && (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 15) || p->workspace_bytes < pl.bytes)) {
    set_error("mv_enc_attention: needs a 16-byte aligned workspace of %lld bytes (mv_enc_attention_workspace_bytes)", (long long)pl.bytes);
    return MV_ERR_INVALID;
  }
  a.block_rows = (int32_t)pl.block_rows;
  a.tiles = (int32_t)((tall + a.block_rows - 1) / a.block_rows);
  a.full = (int32_t)pl.full, a.splits = (int32_t)pl.splits;
  a.partial = reinterpret_cast<float*>(p->workspace);
  DeviceGuard g(device);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (p->keys == 0) {
    const int64_t words = (int64_t)p->batch * a.o_b / 2;
    hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)std::min<int64_t>((words + 255) / 256, 4096)), dim3(256), 0, s, reinterpret_cast<uint32_t*>(a.out), words);
  } else if (p->dtype == MV_BF16) {
    dispatch_cap<true>(a, p->softcap, blocks, s);
  } else {
    dispatch_cap<false>(a, p->softcap, blocks, s);
  }
  MV_HIP(hipGetLastError());
  if (p->keys > 0 && pl.splits > 1) {
    if (p->dtype == MV_BF16) launch_join<true>(a, pl.cut, std::min<int64_t>(tall, a.block_rows), s);
    else launch_join<false>(a, pl.cut, std::min<int64_t>(tall, a.block_rows), s);
    MV_HIP(hipGetLastError());
  }
  return MV_OK;
}

int64_t mv_enc_attention_workspace_bytes(int device, int32_t batch, int32_t rows, int32_t keys, int32_t heads, int32_t kv_heads, int32_t dim) {
  if (batch < 0 || rows < 0 || keys < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 8 || dim > 256 || dim % 8) {
    set_error("mv_enc_attention_workspace_bytes: bad sizes");
    return MV_ERR_INVALID;
  }
  return plan(batch, rows, keys, heads, kv_heads, dim, cu_count(device)).bytes;
}

int mv_enc_padded_ranges(int device, const int32_t* d_starts, int64_t starts_stride, const int32_t* d_ends, int64_t ends_stride, const int32_t* d_prefixes,
                         int32_t prefix, int32_t batch, int32_t rows, int64_t row_offset, int32_t* d_ranges, void* stream) {
  if (batch < 0 || rows < 0 || row_offset < 0 || ((int64_t)batch * rows > 0 && (!d_starts || !d_ends || !d_ranges || (reinterpret_cast<uintptr_t>(d_ranges) & 7)))) {
    set_error("mv_enc_padded_ranges: bad argument");
    return MV_ERR_INVALID;
  }
  const int64_t total = (int64_t)batch * rows;
  if (total == 0) return MV_OK;
  if ((total + 255) / 256 * 256 > kMaxThreads) {
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
