// A mixture-of-experts layer for a few tokens (include/transformer_engine/amd_ext.h).
//
//   p = softmax(logits[t]);  ids = the top_k largest (ties: lowest index);  weights = p[ids], or p[ids] / sum p[ids]
//   h[t, j] = silu(W1[e, :F] x[t]) * (W1[e, F:] x[t]),   out[t] = sum_j weights[t, j] W2[e] h[t, j],   e = ids[t, j]
//
// A decode batch is bound by the weights of the experts it hits (3 F H values each, read once): a workgroup owns 16 rows of one
// expert's matrix, finds that expert's tokens itself by scanning the routing table (T * top_k <= 4096 entries, out of cache) and
// leaves at once if there are none, so the host never learns the routing and nothing has to be sorted first.  The weights are
// the A operand (16 rows x 32 k), the tokens the B operand; the four waves split k and join in LDS.
// Products are exact in the matrix instruction and accumulated in fp32; FP8 weights are widened in registers (exact) and their
// scale multiplies the finished sums; h stays a pair of bf16 terms.  Every token's top_k results are added in order j by the
// last kernel: no atomics.
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
// one wave per token, N logits per lane
template <int N>
__global__ __launch_bounds__(256) void topk_kernel(const void *logits, int dtype, int *ids, float *weights, int64_t tokens,
                                                   int experts, int top_k, bool renormalize) {
  const int lane = threadIdx.x & 63;
  const int64_t t = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (t >= tokens) return;
  float v[N];
  uint64_t key[N];  // value order in the high word (NaN below everything), lower index first in the low word; 0 = none
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * 64 + lane;
    key[i] = 0;
    v[i] = -__builtin_inff();
    if (e < experts) {
      v[i] = load1(logits, t * experts + e, dtype) + 0.f;  // -0 becomes +0: they tie
      const uint32_t b = __float_as_uint(v[i]);
      const uint32_t order = v[i] != v[i] ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
      key[i] = (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~e);
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
// sixteen weights of one row at k .. k + 15, as two operands of eight in E's format
template <typename E>
__device__ __forceinline__ u32x2 widen4(uint32_t w);  // four FP8 (E4M3) -> four E, exact
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
struct Raw16;
template <>
struct Raw16<uint16_t> {
  u32x4 v[2];
  template <bool VEC>
  static __device__ __forceinline__ Raw16 load(const uint16_t *row, int64_t k, int64_t n) {
    return {{row8<VEC>(row, k, n), row8<VEC>(row, k + 8, n)}};
  }
  template <typename E>
  __device__ __forceinline__ void operands(u32x4 (&o)[2]) const {
    o[0] = v[0];
    o[1] = v[1];
  }
};
template <>
struct Raw16<fp8_t> {
  u32x4 v;
  template <bool VEC>
  static __device__ __forceinline__ Raw16 load(const fp8_t *row, int64_t k, int64_t n) {
    Raw16 r{{0u, 0u, 0u, 0u}};
    if constexpr (VEC) {
      if (k < n) r.v = *reinterpret_cast<const u32x4 *>(row + k);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < n) r.v[i >> 2] |= static_cast<uint32_t>(row[k + i].bits) << (8 * (i & 3));
    }
    return r;
  }
  template <typename E>
  __device__ __forceinline__ void operands(u32x4 (&o)[2]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 a = widen4<E>(v[2 * h]), b = widen4<E>(v[2 * h + 1]);
      o[h] = u32x4{a[0], a[1], b[0], b[1]};
    }
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

struct Fc1Args {
  const void *x, *w;       // [tokens][hidden], [experts][2 ffn][hidden]
  const float *scale_inv;  // [experts], null: 1
  const int *ids;          // [tokens][top_k]
  uint16_t *h_hi, *h_lo;   // [pairs][ffn]
  int pairs, top_k, hidden, ffn;
};

template <typename W, typename E, int MT, bool VEC>
__device__ __forceinline__ void fc1_sum(const Fc1Args &p, const W *gate, const W *up, const uint16_t *const (&row)[MT], int tiles,
                                        int wave, int lane, f32x4 (&acc)[2][MT]) {
  for (int k0 = wave * 64; k0 < p.hidden; k0 += kWaves * 64) {
    const int k = k0 + 16 * (lane >> 4);
    const Raw16<W> g = Raw16<W>::template load<VEC>(gate, k, p.hidden), u = Raw16<W>::template load<VEC>(up, k, p.hidden);
    u32x4 x[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < tiles) {
        x[m][0] = row8<VEC>(row[m], k, p.hidden);
        x[m][1] = row8<VEC>(row[m], k + 8, p.hidden);
      }
    u32x4 go[2], uo[2];
    g.template operands<E>(go);
    u.template operands<E>(uo);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < tiles) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          acc[0][m] = mfma16<E>(go[h], x[m][h], acc[0][m]);
          acc[1][m] = mfma16<E>(uo[h], x[m][h], acc[1][m]);
        }
      }
  }
}

// grid: 16 rows of the gate half (and the same of the other) x experts
template <typename W, typename E, int MT>
__global__ __launch_bounds__(256) void fc1_kernel(Fc1Args p, bool vec) {
  __shared__ uint16_t list[kMaxPairs];
  __shared__ int scratch[kWaves];
  __shared__ float red[kWaves][2 * MT * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.y, f0 = blockIdx.x * 16;
  const int n = find_pairs(p.ids, p.pairs, e, list, scratch);
  const int f_row = min(f0 + (lane & 15), p.ffn - 1);
  const W *w = static_cast<const W *>(p.w) + static_cast<int64_t>(e) * 2 * p.ffn * p.hidden;
  const W *gate = w + static_cast<int64_t>(f_row) * p.hidden, *up = gate + static_cast<int64_t>(p.ffn) * p.hidden;
  const float scale = p.scale_inv != nullptr ? p.scale_inv[e] : 1.f;
  for (int n0 = 0; n0 < n; n0 += 16 * MT) {
    const uint16_t *row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int pair = list[min(n0 + m * 16 + (lane & 15), n - 1)];
      row[m] = static_cast<const uint16_t *>(p.x) + static_cast<int64_t>(pair / p.top_k) * p.hidden;
    }
    const int tiles = min(MT, (n - n0 + 15) / 16);
    f32x4 acc[2][MT] = {};
    if (vec) fc1_sum<W, E, MT, true>(p, gate, up, row, tiles, wave, lane, acc);
    else fc1_sum<W, E, MT, false>(p, gate, up, row, tiles, wave, lane, acc);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][((s * MT + m) * 4 + i) * 64 + lane] = acc[s][m][i];
    __syncthreads();
    for (int q = threadIdx.x; q < tiles * 256; q += 256) {
      const int f = q & 15, tok = (q >> 4) & 15, m = q >> 8;
      const int slot = (m * 4 + (f & 3)) * 64 + (f >> 2) * 16 + tok;
      float g = 0.f, u = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        g += red[v][slot];
        u += red[v][MT * 256 + slot];
      }
      g *= scale;
      u *= scale;
      const int at = n0 + m * 16 + tok;
      if (at < n && f0 + f < p.ffn) {
        __bf16 hi, lo;
        split1(g * sigmoid_f(g) * u, hi, lo);
        const int64_t o = static_cast<int64_t>(list[at]) * p.ffn + f0 + f;
        p.h_hi[o] = bits16(hi);
        p.h_lo[o] = bits16(lo);
      }
    }
    __syncthreads();
  }
}

struct Fc2Args {
  const uint16_t *h_hi, *h_lo;  // [pairs][ffn]
  const void *w;                // [experts][hidden][ffn]
  const float *scale_inv;       // [experts], null: 1
  const int *ids;               // [tokens][top_k]
  const float *weights;         // [tokens][top_k]
  float *y;                     // [pairs][hidden]
  int pairs, hidden, ffn;
};

// eight stored weights as bf16 terms: FP8 is widened first (exact), 16-bit types as they are
template <typename W, typename E>
struct Fc2Terms {
  typedef E type;
};
template <typename E>
struct Fc2Terms<fp8_t, E> {
  typedef bf16_t type;
};

template <typename W, typename E, int MT, bool VEC>
__device__ __forceinline__ void fc2_sum(const Fc2Args &p, const W *w, const int64_t (&row)[MT], int tiles, int wave, int lane,
                                        f32x4 (&acc)[MT]) {
  typedef typename Fc2Terms<W, E>::type T;
  for (int k0 = wave * 64; k0 < p.ffn; k0 += kWaves * 64) {
    const int k = k0 + 16 * (lane >> 4);
    const Raw16<W> r = Raw16<W>::template load<VEC>(w, k, p.ffn);
    u32x4 hi[MT][2], lo[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < tiles) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          hi[m][h] = row8<VEC>(p.h_hi + row[m], k + 8 * h, p.ffn);
          lo[m][h] = row8<VEC>(p.h_lo + row[m], k + 8 * h, p.ffn);
        }
      }
    u32x4 o[2];
    r.template operands<T>(o);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Terms<T> terms(o[h]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (m < tiles) acc[m] = mfma16_split<T>(terms, hi[m][h], lo[m][h], acc[m]);
    }
  }
}

// grid: 16 rows of the output x experts
template <typename W, typename E, int MT>
__global__ __launch_bounds__(256) void fc2_kernel(Fc2Args p, bool vec) {
  __shared__ uint16_t list[kMaxPairs];
  __shared__ int scratch[kWaves];
  __shared__ float red[kWaves][MT * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.y, c0 = blockIdx.x * 16;
  const int n = find_pairs(p.ids, p.pairs, e, list, scratch);
  const int c_row = min(c0 + (lane & 15), p.hidden - 1);
  const W *w = static_cast<const W *>(p.w) + (static_cast<int64_t>(e) * p.hidden + c_row) * p.ffn;
  const float scale = p.scale_inv != nullptr ? p.scale_inv[e] : 1.f;
  for (int n0 = 0; n0 < n; n0 += 16 * MT) {
    int64_t row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) row[m] = static_cast<int64_t>(list[min(n0 + m * 16 + (lane & 15), n - 1)]) * p.ffn;
    const int tiles = min(MT, (n - n0 + 15) / 16);
    f32x4 acc[MT] = {};
    if (vec) fc2_sum<W, E, MT, true>(p, w, row, tiles, wave, lane, acc);
    else fc2_sum<W, E, MT, false>(p, w, row, tiles, wave, lane, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[wave][(m * 4 + i) * 64 + lane] = acc[m][i];
    __syncthreads();
    for (int q = threadIdx.x; q < tiles * 256; q += 256) {
      const int c = q & 15, tok = (q >> 4) & 15, m = q >> 8;
      const int slot = (m * 4 + (c & 3)) * 64 + (c >> 2) * 16 + tok;
      float y = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) y += red[v][slot];
      const int at = n0 + m * 16 + tok;
      if (at < n && c0 + c < p.hidden) p.y[static_cast<int64_t>(list[at]) * p.hidden + c0 + c] = y * scale * p.weights[list[at]];
    }
    __syncthreads();
  }
}

// grid: columns x tokens
template <typename E>
__global__ __launch_bounds__(256) void combine_kernel(const float *y, const int *ids, E *out, int top_k, int hidden, int experts) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int64_t t = blockIdx.y;
  if (c >= hidden) return;
  float s = 0.f;
  for (int j = 0; j < top_k; ++j) {
    const int id = ids[t * top_k + j];
    if (id >= 0 && id < experts) s += y[(t * top_k + j) * hidden + c];
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

template <typename W, typename E, int MT>
void launch(const Layer &l, const Fc1Args &a, const Fc2Args &b, E *out, hipStream_t stream) {
  const int step = sizeof(W) == 1 ? 16 : 8;
  const bool v1 = l.hidden % step == 0 && aligned16(a.x) && aligned16(a.w);
  const bool v2 = l.ffn % step == 0 && aligned16(b.w);
  hipLaunchKernelGGL((fc1_kernel<W, E, MT>), dim3(ceil_div(l.ffn, 16), l.experts), dim3(256), 0, stream, a, v1);
  NVTE_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL((fc2_kernel<W, E, MT>), dim3(ceil_div(l.hidden, 16), l.experts), dim3(256), 0, stream, b, v2);
  NVTE_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL((combine_kernel<E>), dim3(ceil_div(l.hidden, 256), l.tokens), dim3(256), 0, stream, b.y, b.ids, out, l.top_k,
                     l.hidden, l.experts);
  NVTE_CHECK_HIP(hipGetLastError());
}

template <typename W, typename E>
void run(const Layer &l, const Fc1Args &a, const Fc2Args &b, void *out, hipStream_t stream) {
  E *o = static_cast<E *>(out);
  if (l.tokens <= 16) launch<W, E, 1>(l, a, b, o, stream);
  else if (l.tokens <= 32) launch<W, E, 2>(l, a, b, o, stream);
  else launch<W, E, 4>(l, a, b, o, stream);
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
    NVTE_CHECK(tokens < (1ull << 31), "too many tokens: ", tokens);
    if (tokens == 0) return;
    NVTE_CHECK(logits && topk_ids && topk_weights, "a required pointer is NULL");
    auto launch_topk = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(ceil_div(tokens, 4)), dim3(256), 0, stream, logits, dtype, topk_ids, topk_weights,
                         static_cast<int64_t>(tokens), static_cast<int>(num_experts), static_cast<int>(top_k), renormalize != 0);
    };
    if (num_experts <= 64) launch_topk(topk_kernel<1>);
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
    const Fc1Args a{x, w_fc1, fc1_scale_inv, topk_ids, hi, lo, l.tokens * l.top_k, l.top_k, l.hidden, l.ffn};
    const Fc2Args b{hi, lo, w_fc2, fc2_scale_inv, topk_ids, topk_weights, y, l.tokens * l.top_k, l.hidden, l.ffn};
    if (wt == kNVTEFloat8E4M3) {
      t == kNVTEBFloat16 ? run<fp8_t, bf16_t>(l, a, b, out, stream) : run<fp8_t, f16_t>(l, a, b, out, stream);
    } else {
      t == kNVTEBFloat16 ? run<uint16_t, bf16_t>(l, a, b, out, stream) : run<uint16_t, f16_t>(l, a, b, out, stream);
    }
  });
}

}  // extern "C"
