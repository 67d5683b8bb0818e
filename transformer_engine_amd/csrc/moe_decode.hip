// A mixture-of-experts layer for a few tokens (include/transformer_engine/amd_ext.h).
//
//   p = softmax(logits[t]);  ids = the top_k largest (ties: lowest index);  weights = p[ids], or p[ids] / sum p[ids]
//   h[t, j] = silu(W1[e, :F] x[t]) * (W1[e, F:] x[t]),   out[t] = sum_j weights[t, j] W2[e] h[t, j],   e = ids[t, j]
//
// Token slots of a tile that no token fills read the expert's last one again and their results are dropped.
// A decode batch is bound by the weights of the experts it hits (3 F H values each, read once): a workgroup owns some rows of one
// expert's matrix, finds that expert's tokens itself by scanning the routing table (T * top_k <= 4096 entries, out of cache) and
// leaves at once if there are none, so the host never learns the routing and nothing has to be sorted first.  The weights are
// the A operand (16 rows x 32 k), the tokens the B operand; the four waves split k and join in LDS.
// Products are exact in the matrix instruction and accumulated in fp32; FP8 weights are widened in registers (exact) and their
// scale multiplies the finished sums; h stays a pair of bf16 terms.  Every token's top_k results are added in order j by the
// last kernel: no atomics.
// Measured (H = 4096, F = 14336, FC1 and FC2 in us): bf16, one token, 2 experts hit 85 and 43 (5.5 TB/s); FP8, 64 tokens, 8 experts hit 228 and 122
// (4.1 and 3.9 TB/s: converting the weights takes part of the time that loading them leaves).  Five tokens through 64 FP8 experts of H = 2048,
// F = 1408: 39 and 27.  Router and combine are latencies, 5 us each.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "act_math.h"
#include "common.h"
#include "device_utils.h"
#include "mfma16.h"
#include "transformer_engine/amd_ext.h"

namespace te {
namespace {

constexpr int kMaxTokens = 256;
constexpr int kMaxPairs = 4096;
constexpr int kMaxExperts = 1024;  // of the router: 16 logits per lane
constexpr int kWaves = 4;

struct fp8_t {
  uint8_t bits;
};

// ------------------------------------------------------------------------------------------------ router
// value order in the high word (NaN below everything), lower index first in the low word; never 0
__device__ __forceinline__ uint64_t order_key(float v, int e) {
  const uint32_t b = __float_as_uint(v);
  const uint32_t order = v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~e);
}

// up to 64 experts, one wave per token, one logit per lane: a lane's rank is the number of larger keys
__global__ __launch_bounds__(256) void topk64_kernel(const void *logits, int dtype, int *ids, float *weights, int64_t tokens,
                                                     int experts, int top_k, bool renormalize) {
  const int lane = threadIdx.x & 63;
  const int64_t t = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (t >= tokens) return;
  const bool mine = lane < experts;
  const float v = mine ? load1(logits, t * experts + lane, dtype) + 0.f : -__builtin_inff();  // -0 becomes +0: they tie
  const uint64_t key = mine ? order_key(v, lane) : 0;
  const uint32_t hi = static_cast<uint32_t>(key >> 32), lo = static_cast<uint32_t>(key);
  int rank = 0;
#pragma unroll 8
  for (int e = 0; e < experts; ++e) {
    const uint64_t other = (static_cast<uint64_t>(__builtin_amdgcn_readlane(hi, e)) << 32) |
                           static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, e));
    rank += other > key;
  }
  const bool chosen = mine && rank < top_k;
  const float top = wave_max(v);
  const float x = mine ? expf(v - top) : 0.f;
  float total = renormalize && !chosen ? 0.f : x;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if (chosen) {
    ids[t * top_k + rank] = lane;
    weights[t * top_k + rank] = x / total;
  }
}

// one wave per token, N logits per lane
template <int N>
__global__ __launch_bounds__(256) void topk_kernel(const void *logits, int dtype, int *ids, float *weights, int64_t tokens,
                                                   int experts, int top_k, bool renormalize) {
  const int lane = threadIdx.x & 63;
  const int64_t t = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (t >= tokens) return;
  float v[N];
  uint64_t key[N];  // 0 = none
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * 64 + lane;
    key[i] = 0;
    v[i] = -__builtin_inff();
    if (e < experts) {
      v[i] = load1(logits, t * experts + e, dtype) + 0.f;  // -0 becomes +0: they tie
      key[i] = order_key(v[i], e);
      top = fmaxf(top, v[i]);
    }
  }
  top = wave_max(top);
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) total += i * 64 + lane < experts ? expf(v[i] - top) : 0.f;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  float chosen = 0.f, mine = 0.f;
  for (int j = 0; j < top_k; ++j) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) best = key[i] > best ? key[i] : best;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), off, 64);
      best = other > best ? other : best;
    }
    const int e = static_cast<int>(~static_cast<uint32_t>(best));
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (key[i] == best) {
        x = v[i];
        key[i] = 0;
      }
    x = expf(__shfl(x, e & 63, 64) - top);
    chosen += x;
    if (lane == j) {
      mine = x;
      ids[t * top_k + j] = e;
    }
  }
  if (lane < top_k) weights[t * top_k + lane] = mine / (renormalize ? chosen : total);
}

// ------------------------------------------------------------------------------------------------ expert products
// Thirty-two bytes of a weight row per lane: the four lane groups of a wave cover one 128-byte line of each of 16 rows.
// `operands` widens them to matrix operands of eight k each (in E's format, exact).
template <typename E>
__device__ __forceinline__ u32x2 widen4(uint32_t w);  // four FP8 (E4M3) -> four E
template <>
__device__ __forceinline__ u32x2 widen4<bf16_t>(uint32_t w) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
}
template <>
__device__ __forceinline__ u32x2 widen4<f16_t>(uint32_t w) {
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
}

template <typename W>
struct Line;
template <>
struct Line<uint16_t> {
  static constexpr int kOps = 2;      // operands per lane
  static constexpr int kBlock = 64;   // k per wave
  u32x4 v[2];
  __device__ __forceinline__ void load(const uint16_t *p) {
    v[0] = load8(p);
    v[1] = load8(p + 8);
  }
  __device__ __forceinline__ void load_any(const uint16_t *p, int n, const uint16_t *end) {
    v[0] = load8_any(p, n, end);
    v[1] = load8_any(p + 8, n - 8, end);
  }
  template <typename E>
  __device__ __forceinline__ u32x4 operand(int i) const {
    return v[i];
  }
};
template <>
struct Line<fp8_t> {
  static constexpr int kOps = 4;
  static constexpr int kBlock = 128;
  typedef uint32_t any __attribute__((ext_vector_type(4), aligned(1)));
  u32x4 v[2];
  __device__ __forceinline__ void load(const fp8_t *p) {
    v[0] = *reinterpret_cast<const any *>(p);
    v[1] = *reinterpret_cast<const any *>(p + 16);
  }
  __device__ __forceinline__ void load_any(const fp8_t *p, int n, const fp8_t *) {
    v[0] = v[1] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
#pragma unroll 1
      for (int i = 0; i < min(n - 4 * w, 4); ++i) v[w >> 2][w & 3] |= static_cast<uint32_t>(p[4 * w + i].bits) << (8 * i);
    }
  }
  template <typename E>
  __device__ __forceinline__ u32x4 operand(int i) const {
    const u32x2 a = widen4<E>(v[i >> 1][2 * (i & 1)]), b = widen4<E>(v[i >> 1][2 * (i & 1) + 1]);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
};

// the routing table's entries of expert `e`, in rising order, into `list`; returns how many.  256 threads
__device__ __forceinline__ int find_pairs(const int *ids, int pairs, int e, uint16_t *list, int *scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n = 0;
  for (int p0 = 0; p0 < pairs; p0 += 256) {
    const int p = p0 + threadIdx.x;
    const bool hit = p < pairs && ids[p] == e;
    const uint64_t m = __ballot(hit);
    if (lane == 0) scratch[wave] = __popcll(m);
    __syncthreads();
    int at = n;
    for (int w = 0; w < wave; ++w) at += scratch[w];
    if (hit) list[at + __popcll(m & ((1ull << lane) - 1))] = static_cast<uint16_t>(p);
    n += scratch[0] + scratch[1] + scratch[2] + scratch[3];
    __syncthreads();
  }
  return n;
}

// The blocks of k of one of KW waves (every KW-th), U at a time, every load of them on its way before the first product waits.  What is
// left over goes singly, the row's ragged end last.  Stage<U, GUARD>: load(block) and multiply(acc).
template <int U, int KW, template <int, bool> class Stage, typename Args, typename Acc>
__device__ __forceinline__ void for_blocks(const Args &args, int k, int block, int first, Acc &acc) {
  const int full = k / block;
  int b = first;
  for (; b + KW * (U - 1) < full; b += KW * U) {
    Stage<U, false> s;
    s.load(args, b);
    __builtin_amdgcn_sched_barrier(0);
    s.multiply(args, acc);
  }
  if constexpr (U > 1) {
    for (; b < full; b += KW) {
      Stage<1, false> s;
      s.load(args, b);
      s.multiply(args, acc);
    }
  }
  if (b == full && k % block != 0) {
    Stage<1, true> s;
    s.load(args, b);
    s.multiply(args, acc);
  }
}

struct Fc1Args {
  const void *x, *w;       // [tokens][hidden], [experts][2 ffn][hidden]
  const float *scale_inv;  // [experts], null: 1
  const int *ids;          // [tokens][top_k]
  uint16_t *h_hi, *h_lo;   // [pairs][ffn]
  int pairs, top_k, experts, hidden, ffn;
};

template <typename W, typename E, int MT, int FT, int KW, bool SMALL>
struct Fc1 {
  const W *gate[FT];        // this lane's rows of the gate half
  int64_t up;               // from there to the other half's
  const uint16_t *row[MT];  // this lane's tokens
  const W *w_end;           // ends of the arrays (SMALL)
  const uint16_t *x_end;
  int hidden, lane;

  template <int U, bool GUARD>
  struct Stage {
    typedef Line<W> L;
    static constexpr int N = L::kOps;
    L g[U][FT], u[U][FT];
    u32x4 x[U][MT][N];
    // SMALL: rows of fewer than 8 N elements.  GUARD: the row's ragged end.  A lane past it takes the last 8 N elements (see mfma16.h);
    // x alone is cleared of what other lanes hold.
    __device__ __forceinline__ void load(const Fc1 &p, int block) {
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int at = (block + s * KW) * L::kBlock + (p.lane >> 4) * (8 * N), k = GUARD ? min(at, p.hidden - 8 * N) : at;
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          if constexpr (SMALL) {
            g[s][f].load_any(p.gate[f] + at, p.hidden - at, p.w_end);
            u[s][f].load_any(p.gate[f] + p.up + at, p.hidden - at, p.w_end);
          } else {
            g[s][f].load(p.gate[f] + k);
            u[s][f].load(p.gate[f] + p.up + k);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int o = 0; o < N; ++o) {
            if constexpr (SMALL) x[s][m][o] = load8_any(p.row[m] + at + 8 * o, p.hidden - at - 8 * o, p.x_end);
            else x[s][m][o] = load8(p.row[m] + k + 8 * o);
            if constexpr (GUARD && !SMALL) x[s][m][o] = without_head(x[s][m][o], at - k - 8 * o);
          }
      }
    }
    __device__ __forceinline__ void multiply(const Fc1 &p, f32x4 (&acc)[FT * MT * 2]) const {
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int o = 0; o < N; ++o)
#pragma unroll
          for (int f = 0; f < FT; ++f) {
            const u32x4 go = g[s][f].template operand<E>(o), uo = u[s][f].template operand<E>(o);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              f32x4 *a = acc + 2 * (f * MT + m);
              a[0] = mfma16<E>(go, x[s][m][o], a[0]);
              a[1] = mfma16<E>(uo, x[s][m][o], a[1]);
            }
          }
    }
  };
};

// Sum over the KW waves that share a row group's k; D's registers as they are: token = lane % 16, rows 4 (lane / 16) + i.
template <int KW, int N>
__device__ __forceinline__ void join_waves(f32x4 (&acc)[N], f32x4 (*red)[64], int wave, int lane) {
  if constexpr (KW > 1) {
    __syncthreads();  // the last join's sums are read
#pragma unroll
    for (int i = 0; i < N; ++i) red[wave * N + i][lane] = acc[i];
    __syncthreads();
    // each wave adds up its share of the group's registers
    const int first = wave / KW * KW;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i % KW == wave % KW) {
        f32x4 s = red[first * N + i][lane];
#pragma unroll
        for (int w = 1; w < KW; ++w) s += red[(first + w) * N + i][lane];
        acc[i] = s;
      }
  }
}

// grid: (4 / KW) 16 FT rows of the gate half (and the same of the other) x experts
template <typename W, typename E, int MT, int FT, int U, int KW, bool SMALL>
__global__ __launch_bounds__(256) void fc1_kernel(Fc1Args p) {
  __shared__ uint16_t list[kMaxPairs];
  __shared__ int scratch[kWaves];
  __shared__ f32x4 red[KW > 1 ? kWaves * 2 * FT * MT : 1][64];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int e = blockIdx.y, f0 = (blockIdx.x * (kWaves / KW) + wave / KW) * (16 * FT);
  const int n = __builtin_amdgcn_readfirstlane(find_pairs(p.ids, p.pairs, e, list, scratch));
  if (n == 0) return;
  const W *w = static_cast<const W *>(p.w) + static_cast<int64_t>(e) * 2 * p.ffn * p.hidden;
  typedef Fc1<W, E, MT, FT, KW, SMALL> Side;
  Side side;
  side.up = static_cast<int64_t>(p.ffn) * p.hidden;
  side.hidden = p.hidden;
  side.lane = lane;
  side.w_end = static_cast<const W *>(p.w) + static_cast<int64_t>(p.experts) * 2 * p.ffn * p.hidden;
  side.x_end = static_cast<const uint16_t *>(p.x) + static_cast<int64_t>(p.pairs / p.top_k) * p.hidden;
#pragma unroll
  for (int f = 0; f < FT; ++f) side.gate[f] = w + static_cast<int64_t>(min(f0 + f * 16 + (lane & 15), p.ffn - 1)) * p.hidden;
  const float scale = p.scale_inv != nullptr ? p.scale_inv[e] : 1.f;
  for (int n0 = 0; n0 < n; n0 += 16 * MT) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int pair = list[min(n0 + m * 16 + (lane & 15), n - 1)];
      side.row[m] = static_cast<const uint16_t *>(p.x) + static_cast<int64_t>(pair / p.top_k) * p.hidden;
    }
    f32x4 acc[FT * MT * 2] = {};  // [f][m][gate, up]
    for_blocks<U, KW, Side::template Stage>(side, p.hidden, Line<W>::kBlock, wave % KW, acc);
    // gate and up of one tile stay with one wave
    f32x4 g[FT * MT], u[FT * MT];
#pragma unroll
    for (int i = 0; i < FT * MT; ++i) {
      g[i] = acc[2 * i];
      u[i] = acc[2 * i + 1];
    }
    join_waves<KW>(g, red, wave, lane);
    join_waves<KW>(u, red, wave, lane);
#pragma unroll
    for (int i = 0; i < FT * MT; ++i) {
      const int f = i / MT, m = i % MT;
      const int at = n0 + m * 16 + (lane & 15), col = f0 + f * 16 + (lane >> 4) * 4;
      if (i % KW != wave % KW || at >= n) continue;
      const int64_t o = static_cast<int64_t>(list[at]) * p.ffn + col;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float a = g[i][r] * scale, b = u[i][r] * scale;
        __bf16 hi, lo;
        split1(a * sigmoid_f(a) * b, hi, lo);
        if (col + r < p.ffn) {
          p.h_hi[o + r] = bits16(hi);
          p.h_lo[o + r] = bits16(lo);
        }
      }
    }
  }
}

struct Fc2Args {
  const uint16_t *h_hi, *h_lo;  // [pairs][ffn]
  const void *w;                // [experts][hidden][ffn]
  const float *scale_inv;       // [experts], null: 1
  const int *ids;               // [tokens][top_k]
  const float *weights;         // [tokens][top_k]
  float *y;                     // [pairs][hidden]
  int pairs, experts, hidden, ffn;
};

// the format in which stored weights meet h's bf16 terms: FP8 is widened (exact), 16-bit types stay
template <typename W, typename E>
struct Fc2Type {
  typedef E type;
};
template <typename E>
struct Fc2Type<fp8_t, E> {
  typedef bf16_t type;
};

template <typename W, typename E, int MT, int FT, int KW, bool SMALL>
struct Fc2 {
  const W *w[FT];                // this lane's rows
  const uint16_t *hi[MT];        // this lane's tokens
  int64_t lo;                    // from hi to their second terms
  const W *w_end;                // ends of the arrays (SMALL)
  const uint16_t *h_end;
  int ffn, lane;

  template <int U, bool GUARD>
  struct Stage {
    typedef Line<W> L;
    typedef typename Fc2Type<W, E>::type T;
    static constexpr int N = L::kOps;
    L r[U][FT];
    u32x4 h[U][MT][N][2];
    __device__ __forceinline__ void load(const Fc2 &p, int block) {
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int at = (block + s * KW) * L::kBlock + (p.lane >> 4) * (8 * N), k = GUARD ? min(at, p.ffn - 8 * N) : at;
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          if constexpr (SMALL) r[s][f].load_any(p.w[f] + at, p.ffn - at, p.w_end);
          else r[s][f].load(p.w[f] + k);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int o = 0; o < N; ++o)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint16_t *from = p.hi[m] + t * p.lo;
              if constexpr (SMALL) h[s][m][o][t] = load8_any(from + at + 8 * o, p.ffn - at - 8 * o, p.h_end);
              else h[s][m][o][t] = load8(from + k + 8 * o);
              if constexpr (GUARD && !SMALL) h[s][m][o][t] = without_head(h[s][m][o][t], at - k - 8 * o);
            }
      }
    }
    __device__ __forceinline__ void multiply(const Fc2 &p, f32x4 (&acc)[FT * MT]) const {
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int o = 0; o < N; ++o)
#pragma unroll
          for (int f = 0; f < FT; ++f) {
            const Terms<T> terms(r[s][f].template operand<T>(o));
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[f * MT + m] = mfma16_split<T>(terms, h[s][m][o][0], h[s][m][o][1], acc[f * MT + m]);
          }
    }
  };
};

// grid: (4 / KW) 16 FT rows of the output x experts
template <typename W, typename E, int MT, int FT, int U, int KW, bool SMALL>
__global__ __launch_bounds__(256) void fc2_kernel(Fc2Args p) {
  __shared__ uint16_t list[kMaxPairs];
  __shared__ int scratch[kWaves];
  __shared__ f32x4 red[KW > 1 ? kWaves * FT * MT : 1][64];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int e = blockIdx.y, c0 = (blockIdx.x * (kWaves / KW) + wave / KW) * (16 * FT);
  const int n = __builtin_amdgcn_readfirstlane(find_pairs(p.ids, p.pairs, e, list, scratch));
  if (n == 0) return;
  typedef Fc2<W, E, MT, FT, KW, SMALL> Side;
  Side side;
  side.lo = p.h_lo - p.h_hi;
  side.ffn = p.ffn;
  side.lane = lane;
  side.w_end = static_cast<const W *>(p.w) + static_cast<int64_t>(p.experts) * p.hidden * p.ffn;
  side.h_end = p.h_hi + 2 * side.lo;
#pragma unroll
  for (int f = 0; f < FT; ++f)
    side.w[f] = static_cast<const W *>(p.w) + (static_cast<int64_t>(e) * p.hidden + min(c0 + f * 16 + (lane & 15), p.hidden - 1)) * p.ffn;
  const float scale = p.scale_inv != nullptr ? p.scale_inv[e] : 1.f;
  for (int n0 = 0; n0 < n; n0 += 16 * MT) {
#pragma unroll
    for (int m = 0; m < MT; ++m) side.hi[m] = p.h_hi + static_cast<int64_t>(list[min(n0 + m * 16 + (lane & 15), n - 1)]) * p.ffn;
    f32x4 acc[FT * MT] = {};
    for_blocks<U, KW, Side::template Stage>(side, p.ffn, Line<W>::kBlock, wave % KW, acc);
    join_waves<KW>(acc, red, wave, lane);
#pragma unroll
    for (int i = 0; i < FT * MT; ++i) {
      const int f = i / MT, m = i % MT;
      const int at = n0 + m * 16 + (lane & 15), col = c0 + f * 16 + (lane >> 4) * 4;
      if (i % KW != wave % KW || at >= n) continue;
      const float factor = scale * p.weights[list[at]];
      float *y = p.y + static_cast<int64_t>(list[at]) * p.hidden + col;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < p.hidden) y[r] = acc[i][r] * factor;
    }
  }
}

// grid: columns x tokens
template <typename E>
__global__ __launch_bounds__(256) void combine_kernel(const float *y, const int *ids, E *out, int top_k, int hidden, int experts) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int64_t t = blockIdx.y;
  if (c >= hidden) return;
  float s = 0.f;
  for (int j0 = 0; j0 < top_k; j0 += 8) {  // eight at a time on their way
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = min(j0 + i, top_k - 1), id = ids[t * top_k + j];
      const bool there = j0 + i < top_k && id >= 0 && id < experts;
      v[i] = there ? y[(t * top_k + j) * hidden + c] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
  narrow(s, out[t * hidden + c]);
}

// ------------------------------------------------------------------------------------------------ host
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Layer {
  int tokens, top_k, experts, hidden, ffn;
};
size_t hidden_bytes(const Layer &l) { return round_up(static_cast<size_t>(l.tokens) * l.top_k * l.ffn * 2, 256); }
size_t workspace_bytes(const Layer &l) {
  return 2 * hidden_bytes(l) + round_up(static_cast<size_t>(l.tokens) * l.top_k * l.hidden * 4, 256);
}

Layer layer_of(size_t tokens, size_t top_k, size_t experts, size_t hidden, size_t ffn) {
  NVTE_CHECK(tokens <= kMaxTokens, "this layer takes up to ", kMaxTokens, " tokens, got ", tokens,
             ": use the grouped GEMM for larger batches");
  NVTE_CHECK(top_k >= 1 && top_k <= 64 && tokens * top_k <= kMaxPairs, "top_k must be 1 to 64 and tokens * top_k up to ", kMaxPairs,
             ", got top_k=", top_k, " for ", tokens, " tokens");
  NVTE_CHECK(experts >= 1 && experts <= 65535, "number of experts must be 1 to 65535, got ", experts);
  NVTE_CHECK(hidden >= 1 && hidden <= (1u << 20) && ffn >= 1 && ffn <= (1u << 20), "hidden and ffn sizes must be 1 to 2^20, got ",
             hidden, " and ", ffn);
  return {static_cast<int>(tokens), static_cast<int>(top_k), static_cast<int>(experts), static_cast<int>(hidden), static_cast<int>(ffn)};
}

template <typename W, typename E, int MT, int FT1, int U1, int KW1, int FT2, int U2, int KW2>
void launch(const Layer &l, const Fc1Args &a, const Fc2Args &b, E *out, hipStream_t stream) {
  constexpr int kShort = 8 * Line<W>::kOps;
  const dim3 grid1(ceil_div(l.ffn, kWaves / KW1 * 16 * FT1), l.experts), grid2(ceil_div(l.hidden, kWaves / KW2 * 16 * FT2), l.experts);
  const dim3 small1(ceil_div(l.ffn, 16), l.experts), small2(ceil_div(l.hidden, 16), l.experts);
  if (l.hidden >= kShort) hipLaunchKernelGGL((fc1_kernel<W, E, MT, FT1, U1, KW1, false>), grid1, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((fc1_kernel<W, E, 1, 1, 1, 4, true>), small1, dim3(256), 0, stream, a);
  NVTE_CHECK_HIP(hipGetLastError());
  if (l.ffn >= kShort) hipLaunchKernelGGL((fc2_kernel<W, E, MT, FT2, U2, KW2, false>), grid2, dim3(256), 0, stream, b);
  else hipLaunchKernelGGL((fc2_kernel<W, E, 1, 1, 1, 4, true>), small2, dim3(256), 0, stream, b);
  NVTE_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL((combine_kernel<E>), dim3(ceil_div(l.hidden, 256), l.tokens), dim3(256), 0, stream, b.y, b.ids, out, l.top_k,
                     l.hidden, l.experts);
  NVTE_CHECK_HIP(hipGetLastError());
}

template <typename W, typename E>
void run(const Layer &l, const Fc1Args &a, const Fc2Args &b, void *out, hipStream_t stream) {
  E *o = static_cast<E *>(out);
  // Twice the mean number of tokens per expert.  Up to 16 of them take one operand of tokens and few rows per workgroup; more tokens want
  // more of both, since the tokens are read again for every row group and the weights again for every token group.  The layer in us,
  // E = 8, H = 4096, F = 2048, bf16 (FP8), the three forms in their order here:
  //   rule 16: 32 tokens, top 2  87 (58) / 103 (60) / 111 (77)      rule 64: 64 tokens, top 4  191 (137) / 164 (95) / 122 (93)
  //   rule 32: 64 tokens, top 2  119 (83) / 105 (63) / 115 (83)     rule 64: 64 tokens, top 8  306 (222) / 203 (122) / 141 (116)
  const int per_expert = std::min(l.tokens, 2 * l.tokens * l.top_k / l.experts);
  if (per_expert <= 16) launch<W, E, 1, 1, sizeof(W), 4, 2, sizeof(W), 4>(l, a, b, o, stream);
  else if (per_expert <= 32) launch<W, E, 2, 2, 1, 4, 8, 1, 4>(l, a, b, o, stream);
  else launch<W, E, 4, 2, 1, 2, 4, 1, 4>(l, a, b, o, stream);
}

}  // namespace
}  // namespace te

using namespace te;

extern "C" {

void nvte_amd_moe_topk(const void *logits, int *topk_ids, float *topk_weights, size_t tokens, size_t num_experts, size_t top_k,
                       int renormalize, int dtype, hipStream_t stream) {
  api_guard("nvte_amd_moe_topk", [&] {
    NVTE_CHECK(is_high_precision(static_cast<DType>(dtype)), "logits have dtype=", dtype_name(static_cast<DType>(dtype)),
               ", but expected float32, float16 or bfloat16");
    NVTE_CHECK(num_experts >= 1 && num_experts <= kMaxExperts, "number of experts must be 1 to ", kMaxExperts, ", got ", num_experts);
    NVTE_CHECK(top_k >= 1 && top_k <= 64 && top_k <= num_experts, "top_k must be 1 to 64 and at most the number of experts (",
               num_experts, "), got ", top_k);
    NVTE_CHECK(tokens <= (1u << 26) - 4, "too many tokens: ", tokens);  // 64 threads each, fewer than 2^32 in a launch
    if (tokens == 0) return;
    NVTE_CHECK(logits && topk_ids && topk_weights, "a required pointer is NULL");
    auto launch_topk = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(ceil_div(tokens, 4)), dim3(256), 0, stream, logits, dtype, topk_ids, topk_weights,
                         static_cast<int64_t>(tokens), static_cast<int>(num_experts), static_cast<int>(top_k), renormalize != 0);
    };
    if (num_experts <= 64) launch_topk(topk64_kernel);
    else if (num_experts <= 256) launch_topk(topk_kernel<4>);
    else launch_topk(topk_kernel<kMaxExperts / 64>);
    NVTE_CHECK_HIP(hipGetLastError());
  });
}

size_t nvte_amd_moe_forward_workspace_size(size_t tokens, size_t top_k, size_t num_experts, size_t hidden, size_t ffn) {
  return api_guard("nvte_amd_moe_forward_workspace_size",
                   [&]() -> size_t { return workspace_bytes(layer_of(tokens, top_k, num_experts, hidden, ffn)); });
}

void nvte_amd_moe_forward(const void *x, const void *w_fc1, const void *w_fc2, const float *fc1_scale_inv,
                          const float *fc2_scale_inv, const int *topk_ids, const float *topk_weights, void *out, size_t tokens,
                          size_t top_k, size_t num_experts, size_t hidden, size_t ffn, int dtype, int weight_dtype,
                          void *workspace, size_t workspace_size, hipStream_t stream) {
  api_guard("nvte_amd_moe_forward", [&] {
    const Layer l = layer_of(tokens, top_k, num_experts, hidden, ffn);
    const DType t = static_cast<DType>(dtype), wt = static_cast<DType>(weight_dtype);
    NVTE_CHECK(t == kNVTEBFloat16 || t == kNVTEFloat16, "activations must be bfloat16 or float16, got ", dtype_name(t));
    NVTE_CHECK(wt == t || wt == kNVTEFloat8E4M3, "weights come in the activations' dtype or in FP8 E4M3, got ", dtype_name(wt));
    NVTE_CHECK(wt == kNVTEFloat8E4M3 || (fc1_scale_inv == nullptr && fc2_scale_inv == nullptr), "only FP8 weights have scales");
    if (l.tokens == 0) return;
    NVTE_CHECK(x && w_fc1 && w_fc2 && topk_ids && topk_weights && out, "a required pointer is NULL");
    NVTE_CHECK(wt != kNVTEFloat8E4M3 || (fc1_scale_inv && fc2_scale_inv), "FP8 weights need their scale_inv");
    const size_t need = workspace_bytes(l);
    NVTE_CHECK(workspace != nullptr && workspace_size >= need, "workspace of ", workspace_size, " bytes, but ", need, " are needed");
    NVTE_CHECK(aligned16(workspace), "the workspace must be 16-byte aligned");
    char *ws = static_cast<char *>(workspace);
    uint16_t *hi = reinterpret_cast<uint16_t *>(ws), *lo = reinterpret_cast<uint16_t *>(ws + hidden_bytes(l));
    float *y = reinterpret_cast<float *>(ws + 2 * hidden_bytes(l));
    const Fc1Args a{x, w_fc1, fc1_scale_inv, topk_ids, hi, lo, l.tokens * l.top_k, l.top_k, l.experts, l.hidden, l.ffn};
    const Fc2Args b{hi, lo, w_fc2, fc2_scale_inv, topk_ids, topk_weights, y, l.tokens * l.top_k, l.experts, l.hidden, l.ffn};
    if (wt == kNVTEFloat8E4M3) {
      t == kNVTEBFloat16 ? run<fp8_t, bf16_t>(l, a, b, out, stream) : run<fp8_t, f16_t>(l, a, b, out, stream);
    } else {
      t == kNVTEBFloat16 ? run<uint16_t, bf16_t>(l, a, b, out, stream) : run<uint16_t, f16_t>(l, a, b, out, stream);
    }
  });
}

}  // extern "C"
