// Low-rank adapters of many requests beside a shared projection (include/transformer_engine/amd_ext.h).
//
//   v[t] = A_a x[t]                      y[t]  = base[t]      + s_a B_a v[t]          a = ids[t], none if out of range
//   u[t] = B_a^T dy[t]                   dx[t] = base_grad[t] + s_a A_a^T u[t]
//   dA_a = sum_t s_a u[t] (x) x[t]       dB_a  = sum_t dy[t] (x) s_a v[t]             sums over the tokens of adapter a
//
// Four kernels: `shrink` (activations to rank vectors), `expand` (rank vectors to activations), `wgrad` (outer products summed
// over an adapter's tokens) and its `join`; `plan` lists the tokens of every adapter for the last two.  All of them are bound by
// the activations they stream (2 T (K + O) bytes and more against 2 T r (K + O) operations, r <= 128); the pools stay in L2.
// A tile of tokens walks the distinct adapters among its own tokens, so any order of ids is right; values of other
// adapters' rows are never added, only selected, so a NaN or Inf stays in its own rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "common.h"
#include "device_utils.h"
#include "mfma16.h"
#include "transformer_engine/amd_ext.h"

namespace te {
namespace {

constexpr int kMaxRank = 128;
constexpr int kMaxAdapters = 4096;  // of a backward pass: the plan kernel's histogram in LDS

__device__ __forceinline__ int valid_id(const int *ids, int64_t t, int64_t tokens, int num) {
  if (t >= tokens) return -1;
  const int id = ids[t];
  return id >= 0 && id < num ? id : -1;
}

// ====================================================================================
// shrink: out[slice][t][j] = sum over the slice's k of in[t][k] * w(j, k)
// w(j, k) = pool[a][j][k], or pool[a][k][j] (KMAJOR)
// ====================================================================================
struct ShrinkArgs {
  const uint16_t *in, *pool;
  const int *ids;
  float *out;
  int64_t tokens;
  int features, rank, num, slice;
};

template <typename E, int RT, int MT, int NW, bool VEC, bool KMAJOR>
__device__ __forceinline__ void shrink_sum(const ShrinkArgs &p, const uint16_t *const (&row)[MT], const uint16_t *w, int wave,
                                           int lane, int begin, int end, f32x4 (&acc)[MT][RT]) {
  const int kg = (lane >> 4) * 8;
  // NW * 64 elements of k per turn; a wave's two steps of 32 are one 128-byte line of every row
  for (int k0 = begin + wave * 64; k0 < end; k0 += NW * 64) {
    u32x4 a[2][MT], b[2][RT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * h + kg;
      // what lies behind the slice belongs to the next one; `end` is a multiple of 64 or the row's end
#pragma unroll
      for (int m = 0; m < MT; ++m) a[h][m] = row8<VEC>(row[m], k, end);
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const int col = min(j * 16 + (lane & 15), p.rank - 1);  // columns from `rank` on are computed and not kept
        if constexpr (KMAJOR) {
          u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k + i < end) v[i >> 1] |= static_cast<uint32_t>(w[static_cast<int64_t>(k + i) * p.rank + col]) << (16 * (i & 1));
          b[h][j] = v;
        } else {
          b[h][j] = row8<VEC>(w + static_cast<int64_t>(col) * p.features, k, end);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[m][j] = mfma16<E>(a[h][m], b[h][j], acc[m][j]);
  }
}

// grid: token tiles x slices x phases (the tile's n-th distinct adapter is phase n % gridDim.z's)
template <typename E, int RT, int MT, int NW, bool KMAJOR>
__global__ __launch_bounds__(NW * 64) void shrink_kernel(ShrinkArgs p, bool vec) {
  __shared__ float red[NW][MT * RT * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (16 * MT);
  const int id = lane < 16 * MT ? valid_id(p.ids, t0 + lane, p.tokens, p.num) : -1;
  const uint16_t *row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) row[m] = p.in + min(t0 + m * 16 + (lane & 15), p.tokens - 1) * p.features;
  const int begin = blockIdx.y * p.slice, end = min(begin + p.slice, p.features);

  unsigned phase = 0;
  for (uint64_t left = __ballot(id >= 0); left != 0;) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mine = __ballot(id == cur);
    left &= ~mine;
    if (phase++ % gridDim.z != blockIdx.z) continue;
    f32x4 acc[MT][RT] = {};
    const uint16_t *w = p.pool + static_cast<int64_t>(cur) * p.rank * p.features;
    if (vec) shrink_sum<E, RT, MT, NW, true, KMAJOR>(p, row, w, wave, lane, begin, end, acc);
    else shrink_sum<E, RT, MT, NW, false, KMAJOR>(p, row, w, wave, lane, begin, end, acc);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < RT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][((m * RT + j) * 4 + i) * 64 + lane] = acc[m][j][i];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * RT * 256; e += NW * 64) {
      const int l = e & 63, i = (e >> 6) & 3, j = (e >> 8) % RT, m = (e >> 8) / RT;
      const int tok = m * 16 + (l >> 4) * 4 + i, col = j * 16 + (l & 15);
      float s = 0.f;
#pragma unroll
      for (int n = 0; n < NW; ++n) s += red[n][e];
      if (((mine >> tok) & 1) && col < p.rank) p.out[(blockIdx.y * p.tokens + t0 + tok) * p.rank + col] = s;
    }
    __syncthreads();
  }
}

// ====================================================================================
// expand: out[t][c] = base[t][c] + s_a sum_j (sum over slices of low[slice][t][j]) * w(c, j)
// w(c, j) = pool[a][c][j], or pool[a][j][c] (RMAJOR)
// ====================================================================================
struct ExpandArgs {
  const float *low;
  const uint16_t *pool, *base;  // base may be null (zero) or out itself
  const float *scaling;         // null: 1
  const int *ids;
  uint16_t *out;
  int64_t tokens;
  int slices, features, rank, num, cols;  // cols: columns per workgroup, a multiple of 512
};

// the eight operands of columns c0 + 8 m + f (m = lane % 16): one per f, eight ranks j0 + 8 (lane / 16) of each
template <bool VEC, bool RMAJOR>
__device__ __forceinline__ void pool_block(const uint16_t *w, int lane, int c0, int j0, int features, int rank, u32x4 (&f)[8]) {
  const int c = c0 + 8 * (lane & 15), j = j0 + 8 * (lane >> 4);
  if constexpr (RMAJOR) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = j + i < rank ? row8<VEC>(w + static_cast<int64_t>(j + i) * features, c, features) : u32x4{0u, 0u, 0u, 0u};
    transpose8x8(f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = c + i < features ? row8<VEC>(w + static_cast<int64_t>(c + i) * rank, j, rank) : u32x4{0u, 0u, 0u, 0u};
  }
}

template <typename E>
__device__ __forceinline__ void store_row8(const ExpandArgs &p, int64_t t, int c, bool vec, const float (&add)[8]) {
  const int64_t at = t * p.features + c;
  if (vec) {
    if (c >= p.features) return;
    float b[8] = {};
    if (p.base != nullptr) Raw8<E>::load_cached(reinterpret_cast<const E *>(p.base) + at).widen8(b);
    E o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) narrow(b[k] + add[k], o[k]);
    *reinterpret_cast<u32x4 *>(p.out + at) = *reinterpret_cast<const u32x4 *>(o);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c + k >= p.features) return;
      const float b = p.base != nullptr ? widen(reinterpret_cast<const E *>(p.base)[at + k]) : 0.f;
      narrow(b + add[k], reinterpret_cast<E *>(p.out)[at + k]);
    }
  }
}

template <typename E, int KT, int MT, bool VEC, bool RMAJOR>
__device__ __forceinline__ void expand_columns(const ExpandArgs &p, bool vec_rows, int64_t t0, int id, uint64_t tokens_used,
                                               const u32x4 (&hi)[MT][KT], const u32x4 (&lo)[MT][KT], int wave, int lane) {
  const int begin = blockIdx.y * p.cols, end = min(begin + p.cols, p.features);
  int my_id[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) my_id[m] = __shfl(id, m * 16 + (lane & 15), 64);
  for (int c0 = begin + wave * 128; c0 < end; c0 += 512) {
    f32x4 res[MT][8] = {};
    for (uint64_t left = tokens_used; left != 0;) {
      const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      left &= ~__ballot(id == cur);
      const uint16_t *w = p.pool + static_cast<int64_t>(cur) * p.rank * p.features;
      f32x4 acc[MT][8] = {};
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        u32x4 f[8];
        pool_block<VEC, RMAJOR>(w, lane, c0, k * 32, p.features, p.rank, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const Terms<E> terms(f[i]);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][i] = mfma16_split<E>(terms, hi[m][k], lo[m][k], acc[m][i]);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) res[m][i] = my_id[m] == cur ? acc[m][i] : res[m][i];
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int64_t t = t0 + m * 16 + (lane & 15);
      if (t >= p.tokens) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float add[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) add[k] = res[m][k][i];
        store_row8<E>(p, t, c0 + 8 * (4 * (lane >> 4) + i), vec_rows, add);
      }
    }
  }
}

// grid: token tiles x column ranges
template <typename E, int KT, int MT, bool RMAJOR>
__global__ __launch_bounds__(256) void expand_kernel(ExpandArgs p, bool vec_pool, bool vec_rows) {
  constexpr int kRow = KT * 32 + 8;  // 16-byte aligned rows, neighbouring rows in different banks
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[16 * MT][kRow], s_lo[16 * MT][kRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (16 * MT);
  const int id = lane < 16 * MT ? valid_id(p.ids, t0 + lane, p.tokens, p.num) : -1;
  const uint64_t used = __ballot(id >= 0);
  if (used == 0 && p.base == p.out) return;
  for (int e = threadIdx.x; e < 16 * MT * KT * 32; e += 256) {
    const int tok = e / (KT * 32), j = e % (KT * 32);
    float v = 0.f;
    if (((used >> tok) & 1) && j < p.rank) {
      for (int s = 0; s < p.slices; ++s) v += p.low[(s * p.tokens + t0 + tok) * p.rank + j];
      if (p.scaling != nullptr) v *= p.scaling[p.ids[t0 + tok]];
    }
    __bf16 h, l;
    split1(v, h, l);
    s_hi[tok][j] = bits16(h);
    s_lo[tok][j] = bits16(l);
  }
  __syncthreads();
  u32x4 hi[MT][KT], lo[MT][KT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      hi[m][k] = *reinterpret_cast<const u32x4 *>(&s_hi[m * 16 + (lane & 15)][k * 32 + (lane >> 4) * 8]);
      lo[m][k] = *reinterpret_cast<const u32x4 *>(&s_lo[m * 16 + (lane & 15)][k * 32 + (lane >> 4) * 8]);
    }
  if (vec_pool) expand_columns<E, KT, MT, true, RMAJOR>(p, vec_rows, t0, id, used, hi, lo, wave, lane);
  else expand_columns<E, KT, MT, false, RMAJOR>(p, vec_rows, t0, id, used, hi, lo, wave, lane);
}

// ====================================================================================
// plan: the tokens of every adapter in rising order, and how many work items of `per_item` tokens it has
// one workgroup per adapter; every one counts all ids for itself (T * 4 bytes out of L2), so nothing is exchanged
// ====================================================================================
struct Plan {
  int *order;       // [tokens]
  int *token_base;  // [num + 1] first entry of every adapter in `order`
  int *item_base;   // [num + 1] first work item of every adapter
};

__device__ __forceinline__ int block_sum_int(int v, int *scratch) {  // 256 threads, valid in every thread
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  const int s = scratch[0] + scratch[1] + scratch[2] + scratch[3];
  __syncthreads();
  return s;
}

__global__ __launch_bounds__(256) void plan_kernel(const int *ids, int64_t tokens, int num, int per_item, Plan out) {
  __shared__ int hist[kMaxAdapters];
  __shared__ int scratch[4];
  const int a = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < num; i += 256) hist[i] = 0;
  __syncthreads();
  for (int64_t t = threadIdx.x; t < tokens; t += 256) {
    const int id = valid_id(ids, t, tokens, num);
    if (id >= 0) atomicAdd(&hist[id], 1);
  }
  __syncthreads();
  int before = 0, items = 0;
  for (int i = threadIdx.x; i < a; i += 256) {
    before += hist[i];
    items += (hist[i] + per_item - 1) / per_item;
  }
  before = block_sum_int(before, scratch);
  items = block_sum_int(items, scratch);
  const int mine = hist[a];
  if (threadIdx.x == 0) {
    out.token_base[a] = before;
    out.item_base[a] = items;
    if (a == num - 1) {
      out.token_base[num] = before + mine;
      out.item_base[num] = items + (mine + per_item - 1) / per_item;
    }
  }
  int at = before;
  const int stop = before + mine;
  for (int64_t t0 = 0; t0 < tokens && at < stop; t0 += 256) {
    const int64_t t = t0 + threadIdx.x;
    const bool hit = valid_id(ids, t, tokens, num) == a;
    const uint64_t m = __ballot(hit);
    if (lane == 0) scratch[wave] = __popcll(m);
    __syncthreads();
    int off = at;
    for (int w = 0; w < wave; ++w) off += scratch[w];
    if (hit) out.order[off + __popcll(m & ((1ull << lane) - 1))] = static_cast<int>(t);
    at += scratch[0] + scratch[1] + scratch[2] + scratch[3];
    __syncthreads();
  }
}

// ====================================================================================
// wgrad: one work item's dA [r][K] = sum_t w[t] (x) x[t] and dB [O][r] = sum_t dy[t] (x) w[t]
// ====================================================================================
struct WgradSide {
  const uint16_t *z;  // activations [tokens][features]
  const float *low;   // rank vectors [slices][tokens][rank]
  void *grad;         // [num][rank][features] or [num][features][rank]
  float *part;        // per item, the same layout in fp32
  int slices, features, groups;  // groups: workgroups along the features, 512 columns each
  bool vec;
};
struct WgradArgs {
  WgradSide a, b;
  const float *scaling;
  Plan plan;
  int64_t tokens;
  int rank, num, per_item, grad_type;
};

constexpr int kStep = 64;  // tokens whose rank vectors are staged at a time

template <typename E, int RT, bool VEC, bool IS_B>
__device__ __forceinline__ void wgrad_side(const WgradArgs &p, const WgradSide &side, int group, uint16_t (*s_hi)[RT][512],
                           uint16_t (*s_lo)[RT][512]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int item = blockIdx.y;
  if (item >= p.plan.item_base[p.num]) return;
  int a = 0;
  for (int hi = p.num; hi - a > 1;) {  // the adapter whose items hold this one (adapters without tokens have none)
    const int mid = (a + hi) >> 1;
    if (p.plan.item_base[mid] <= item) a = mid; else hi = mid;
  }
  const int first = p.plan.token_base[a] + (item - p.plan.item_base[a]) * p.per_item;
  const int last = min(first + p.per_item, p.plan.token_base[a + 1]);
  const bool whole = p.plan.item_base[a + 1] - p.plan.item_base[a] == 1;
  const float scale = p.scaling != nullptr ? p.scaling[a] : 1.f;
  const int c0 = group * 512 + wave * 128, c = c0 + 8 * (lane & 15);
  const int j0 = blockIdx.z * 64, ranks = min(p.rank - j0, 64);
  f32x4 acc[RT][8] = {};
  for (int s0 = first; s0 < last; s0 += kStep) {
    u32x4 z[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = s0 + h * 32 + (lane >> 4) * 8 + i;
        z[h][i] = at < last ? row8<VEC>(side.z + static_cast<int64_t>(p.plan.order[at]) * side.features, c, side.features)
                            : u32x4{0u, 0u, 0u, 0u};
      }
    __syncthreads();  // the last step's operands are read
    for (int e = threadIdx.x; e < kStep * RT * 16; e += 256) {
      const int tok = e / (RT * 16), j = e % (RT * 16), at = s0 + tok;
      float v = 0.f;
      if (at < last && j < ranks) {
        const int64_t t = p.plan.order[at];
        for (int s = 0; s < side.slices; ++s) v += side.low[(s * p.tokens + t) * p.rank + j0 + j];
        v *= scale;
      }
      __bf16 h, l;
      split1(v, h, l);
      const int slot = (j & 15) * 8 + ((tok >> 3) & 3) * 128 + (tok & 7);  // operand order: lane, then eight tokens
      s_hi[tok >> 5][j >> 4][slot] = bits16(h);
      s_lo[tok >> 5][j >> 4][slot] = bits16(l);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      transpose8x8(z[h]);
      u32x4 wh[RT], wl[RT];
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        wh[j] = *reinterpret_cast<const u32x4 *>(&s_hi[h][j][lane * 8]);
        wl[j] = *reinterpret_cast<const u32x4 *>(&s_lo[h][j][lane * 8]);
      }
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const Terms<E> terms(z[h][f]);
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j][f] = mfma16_split<E, !IS_B>(terms, wh[j], wl[j], acc[j][f]);
      }
    }
  }
  const int64_t size = static_cast<int64_t>(p.rank) * side.features;
  const int64_t base = (whole ? a : item) * size;
  void *out = whole ? side.grad : side.part;
  const int type = whole ? p.grad_type : kNVTEFloat32;
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        if constexpr (IS_B) {  // rows are features, columns ranks
          const int row = c0 + 8 * (4 * (lane >> 4) + i) + f, col = j * 16 + (lane & 15);
          if (row < side.features && col < ranks) store1(out, base + static_cast<int64_t>(row) * p.rank + j0 + col, type, acc[j][f][i]);
        } else {
          const int row = j * 16 + (lane >> 4) * 4 + i, col = c + f;
          if (row < ranks && col < side.features)
            store1(out, base + static_cast<int64_t>(j0 + row) * side.features + col, type, acc[j][f][i]);
        }
      }
}

// grid: column groups of dA, then of dB  x  work items (an upper bound; the rest leave at once)  x  64 ranks
template <typename E, int RT>
__global__ __launch_bounds__(256) void wgrad_kernel(WgradArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[kStep / 32][RT][512], s_lo[kStep / 32][RT][512];
  const int group = blockIdx.x;
  if (group < p.a.groups) {
    if (p.a.vec) wgrad_side<E, RT, true, false>(p, p.a, group, s_hi, s_lo);
    else wgrad_side<E, RT, false, false>(p, p.a, group, s_hi, s_lo);
  } else {
    if (p.b.vec) wgrad_side<E, RT, true, true>(p, p.b, group - p.a.groups, s_hi, s_lo);
    else wgrad_side<E, RT, false, true>(p, p.b, group - p.a.groups, s_hi, s_lo);
  }
}

// join: the sum of an adapter's work items in their order; zero for an adapter without tokens.  grid: elements x adapters
__global__ __launch_bounds__(256) void join_kernel(WgradArgs p) {
  const int a = blockIdx.y;
  const int first = p.plan.item_base[a], items = p.plan.item_base[a + 1] - first;
  if (items == 1) return;
  const int64_t size_a = static_cast<int64_t>(p.rank) * p.a.features, size_b = static_cast<int64_t>(p.rank) * p.b.features;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < size_a + size_b; e += gridDim.x * 256ll) {
    const bool is_a = e < size_a;
    const float *part = is_a ? p.a.part : p.b.part;
    const int64_t at = is_a ? e : e - size_a, size = is_a ? size_a : size_b;
    float s = 0.f;
    for (int i = 0; i < items; ++i) s += part[(first + i) * size + at];
    store1(is_a ? p.a.grad : p.b.grad, a * size + at, p.grad_type, s);
  }
}

// ====================================================================================
// host
// ====================================================================================
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Shape {
  int64_t tokens;
  int in, out, rank, num;
  DType type;
};

Shape shape_of(size_t tokens, size_t in, size_t out, size_t rank, size_t num, int dtype) {
  const DType t = static_cast<DType>(dtype);
  NVTE_CHECK(t == kNVTEBFloat16 || t == kNVTEFloat16, "adapters take bfloat16 or float16, got ", dtype_name(t));
  NVTE_CHECK(rank >= 1 && rank <= kMaxRank, "rank must be 1 to ", kMaxRank, ", got ", rank);
  NVTE_CHECK(in >= 1 && in <= (1u << 24) && out >= 1 && out <= (1u << 24), "features must be 1 to 2^24, got ", in, " and ", out);
  NVTE_CHECK(num >= 1 && num <= INT_MAX, "at least one adapter is needed, got ", num);
  NVTE_CHECK(tokens < (1ull << 31) - 64, "too many tokens: ", tokens);
  return {static_cast<int64_t>(tokens), static_cast<int>(in), static_cast<int>(out), static_cast<int>(rank), static_cast<int>(num), t};
}

// Few tokens leave most CUs without a tile, so the features are cut into slices (a multiple of 64, at least 256) until about
// 512 workgroups run; whoever reads the rank vectors adds the slices.
int slice_of(int64_t tokens, int features) {
  const int64_t tiles = std::max<int64_t>(1, (tokens + 15) / 16);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(512 / tiles, ceil_div(features, 256)));
  return static_cast<int>(round_up(ceil_div(features, static_cast<size_t>(want)), 64));
}
int num_slices(int64_t tokens, int features) { return static_cast<int>(ceil_div(features, slice_of(tokens, features))); }

template <typename E, bool KMAJOR, int RT, int MT, int NW>
void launch_shrink(const ShrinkArgs &p, int slices, bool vec, hipStream_t stream) {
  const int64_t tiles = (p.tokens + 16 * MT - 1) / (16 * MT);
  // a decode tile's adapters go to workgroups of their own while there are too few tiles
  const int64_t most = std::min<int64_t>(std::min<int64_t>(p.num, p.tokens), 16);
  const int64_t phases = std::max<int64_t>(1, std::min<int64_t>(most, 2048 / (tiles * slices)));
  hipLaunchKernelGGL((shrink_kernel<E, RT, MT, NW, KMAJOR>), dim3(tiles, slices, phases), dim3(NW * 64), 0, stream, p, vec);
  NVTE_CHECK_HIP(hipGetLastError());
}

template <typename E, bool KMAJOR>
void shrink(const void *in, const void *pool, const int *ids, float *out, int64_t tokens, int features, int rank, int num,
            hipStream_t stream) {
  const ShrinkArgs p{static_cast<const uint16_t *>(in), static_cast<const uint16_t *>(pool), ids, out, tokens, features, rank, num,
                     slice_of(tokens, features)};
  const int slices = num_slices(tokens, features);
  const bool vec = features % 8 == 0 && aligned16(in) && (KMAJOR || aligned16(pool));
  const bool many = tokens >= 4096;
  if (rank <= 16) {
    many ? launch_shrink<E, KMAJOR, 1, 2, 8>(p, slices, vec, stream) : launch_shrink<E, KMAJOR, 1, 1, 4>(p, slices, vec, stream);
  } else if (rank <= 32) {
    many ? launch_shrink<E, KMAJOR, 2, 2, 8>(p, slices, vec, stream) : launch_shrink<E, KMAJOR, 2, 1, 4>(p, slices, vec, stream);
  } else if (rank <= 64) {
    launch_shrink<E, KMAJOR, 4, 1, 4>(p, slices, vec, stream);
  } else {
    launch_shrink<E, KMAJOR, 8, 1, 4>(p, slices, vec, stream);
  }
}

template <typename E, bool RMAJOR, int KT, int MT>
void launch_expand(ExpandArgs p, bool vec_pool, bool vec_rows, hipStream_t stream) {
  const int64_t tiles = (p.tokens + 16 * MT - 1) / (16 * MT);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(ceil_div(p.features, 512), 2048 / tiles));
  p.cols = static_cast<int>(round_up(ceil_div(p.features, static_cast<size_t>(want)), 512));
  hipLaunchKernelGGL((expand_kernel<E, KT, MT, RMAJOR>), dim3(tiles, ceil_div(p.features, p.cols)), dim3(256), 0, stream, p,
                     vec_pool, vec_rows);
  NVTE_CHECK_HIP(hipGetLastError());
}

template <typename E, bool RMAJOR>
void expand(const ExpandArgs &p, hipStream_t stream) {
  const bool vec_pool = (RMAJOR ? p.features : p.rank) % 8 == 0 && aligned16(p.pool);
  const bool vec_rows = p.features % 8 == 0 && aligned16(p.out) && aligned16(p.base);
  const bool many = p.tokens >= 1024;
  if (p.rank <= 32) {
    many ? launch_expand<E, RMAJOR, 1, 2>(p, vec_pool, vec_rows, stream) : launch_expand<E, RMAJOR, 1, 1>(p, vec_pool, vec_rows, stream);
  } else if (p.rank <= 64) {
    many ? launch_expand<E, RMAJOR, 2, 2>(p, vec_pool, vec_rows, stream) : launch_expand<E, RMAJOR, 2, 1>(p, vec_pool, vec_rows, stream);
  } else {
    launch_expand<E, RMAJOR, 4, 1>(p, vec_pool, vec_rows, stream);
  }
}

template <typename E>
void launch_wgrad(const WgradArgs &p, unsigned items, hipStream_t stream) {
  const dim3 grid(p.a.groups + p.b.groups, items, ceil_div(p.rank, 64));
  if (p.rank <= 16) hipLaunchKernelGGL((wgrad_kernel<E, 1>), grid, dim3(256), 0, stream, p);
  else if (p.rank <= 32) hipLaunchKernelGGL((wgrad_kernel<E, 2>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((wgrad_kernel<E, 4>), grid, dim3(256), 0, stream, p);
  NVTE_CHECK_HIP(hipGetLastError());
}

// how many tokens a work item sums: enough items for about four waves per CU, no fewer than 64 tokens each
int tokens_per_item(const Shape &s) {
  const int64_t columns = ceil_div(s.in, 512) + ceil_div(s.out, 512);
  const int64_t items = std::max<int64_t>(1, 512 / columns);
  return static_cast<int>(round_up(std::max<size_t>(64, ceil_div(s.tokens, items)), 64));
}
int64_t most_items(const Shape &s) { return s.tokens / tokens_per_item(s) + std::min<int64_t>(s.num, s.tokens); }

struct BackwardWorkspace {
  size_t low, order, token_base, item_base, part_a, part_b, bytes;
};
BackwardWorkspace backward_workspace(const Shape &s) {
  BackwardWorkspace w{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  w.low = take(static_cast<size_t>(num_slices(s.tokens, s.out)) * s.tokens * s.rank * sizeof(float));
  w.order = take(s.tokens * sizeof(int));
  w.token_base = take((s.num + 1) * sizeof(int));
  w.item_base = take((s.num + 1) * sizeof(int));
  w.part_a = take(static_cast<size_t>(most_items(s)) * s.rank * s.in * sizeof(float));
  w.part_b = take(static_cast<size_t>(most_items(s)) * s.rank * s.out * sizeof(float));
  w.bytes = at;
  return w;
}

template <typename E>
void backward(const Shape &s, const void *x, const void *dy, const void *a, const void *b, const int *ids, const float *scaling,
              const float *low, const void *base_grad, void *dx, void *da, void *db, int grad_type, char *ws, hipStream_t stream) {
  const BackwardWorkspace w = backward_workspace(s);
  float *up = reinterpret_cast<float *>(ws + w.low);
  if (s.tokens > 0) {
    shrink<E, true>(dy, b, ids, up, s.tokens, s.out, s.rank, s.num, stream);
    if (dx != nullptr)
      expand<E, true>({up, static_cast<const uint16_t *>(a), static_cast<const uint16_t *>(base_grad), scaling, ids,
                       static_cast<uint16_t *>(dx), s.tokens, num_slices(s.tokens, s.out), s.in, s.rank, s.num, 0}, stream);
  }
  if (da == nullptr) return;
  WgradArgs p{};
  p.a = {static_cast<const uint16_t *>(x), up, da, reinterpret_cast<float *>(ws + w.part_a), num_slices(s.tokens, s.out), s.in,
         static_cast<int>(ceil_div(s.in, 512)), s.in % 8 == 0 && aligned16(x)};
  p.b = {static_cast<const uint16_t *>(dy), low, db, reinterpret_cast<float *>(ws + w.part_b), num_slices(s.tokens, s.in), s.out,
         static_cast<int>(ceil_div(s.out, 512)), s.out % 8 == 0 && aligned16(dy)};
  p.scaling = scaling;
  p.plan = {reinterpret_cast<int *>(ws + w.order), reinterpret_cast<int *>(ws + w.token_base), reinterpret_cast<int *>(ws + w.item_base)};
  p.tokens = s.tokens;
  p.rank = s.rank;
  p.num = s.num;
  p.per_item = tokens_per_item(s);
  p.grad_type = grad_type;
  hipLaunchKernelGGL(plan_kernel, dim3(s.num), dim3(256), 0, stream, ids, s.tokens, s.num, p.per_item, p.plan);
  NVTE_CHECK_HIP(hipGetLastError());
  const int64_t items = most_items(s);
  NVTE_CHECK(items <= 65535, "too many work items: ", items);
  if (items > 0) launch_wgrad<E>(p, static_cast<unsigned>(items), stream);
  const int64_t elements = static_cast<int64_t>(s.rank) * (static_cast<int64_t>(s.in) + s.out);
  const int64_t blocks = std::min<int64_t>(ceil_div(elements, 256), std::max<int64_t>(1, 4096 / s.num));
  hipLaunchKernelGGL(join_kernel, dim3(blocks, s.num), dim3(256), 0, stream, p);
  NVTE_CHECK_HIP(hipGetLastError());
}

}  // namespace
}  // namespace te

using namespace te;

extern "C" {

size_t nvte_amd_lora_num_slices(size_t tokens, size_t features) {
  return api_guard("nvte_amd_lora_num_slices", [&]() -> size_t {
    NVTE_CHECK(features >= 1 && features <= (1u << 24) && tokens < (1ull << 31) - 64, "bad sizes ", tokens, " and ", features);
    return num_slices(static_cast<int64_t>(tokens), static_cast<int>(features));
  });
}

void nvte_amd_lora_forward(const void *x, const void *a, const void *b, const int *adapter_ids, const float *scaling,
                           const void *base, void *out, float *low, size_t tokens, size_t in_features, size_t out_features,
                           size_t rank, size_t num_adapters, int dtype, hipStream_t stream) {
  api_guard("nvte_amd_lora_forward", [&] {
    const Shape s = shape_of(tokens, in_features, out_features, rank, num_adapters, dtype);
    if (s.tokens == 0) return;
    NVTE_CHECK(x && a && b && adapter_ids && out && low, "a required pointer is NULL");
    const ExpandArgs p{low, static_cast<const uint16_t *>(b), static_cast<const uint16_t *>(base), scaling, adapter_ids,
                       static_cast<uint16_t *>(out), s.tokens, num_slices(s.tokens, s.in), s.out, s.rank, s.num, 0};
    if (s.type == kNVTEBFloat16) {
      shrink<bf16_t, false>(x, a, adapter_ids, low, s.tokens, s.in, s.rank, s.num, stream);
      expand<bf16_t, false>(p, stream);
    } else {
      shrink<f16_t, false>(x, a, adapter_ids, low, s.tokens, s.in, s.rank, s.num, stream);
      expand<f16_t, false>(p, stream);
    }
  });
}

size_t nvte_amd_lora_backward_workspace_size(size_t tokens, size_t in_features, size_t out_features, size_t rank,
                                             size_t num_adapters) {
  return api_guard("nvte_amd_lora_backward_workspace_size", [&]() -> size_t {
    return backward_workspace(shape_of(tokens, in_features, out_features, rank, num_adapters, kNVTEBFloat16)).bytes;
  });
}

void nvte_amd_lora_backward(const void *x, const void *dy, const void *a, const void *b, const int *adapter_ids,
                            const float *scaling, const float *low, const void *base_grad, void *dx, void *da, void *db,
                            size_t tokens, size_t in_features, size_t out_features, size_t rank, size_t num_adapters, int dtype,
                            int grad_dtype, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  api_guard("nvte_amd_lora_backward", [&] {
    const Shape s = shape_of(tokens, in_features, out_features, rank, num_adapters, dtype);
    NVTE_CHECK(grad_dtype == dtype || grad_dtype == kNVTEFloat32, "adapter gradients come in the adapters' dtype or in float32, got ",
               dtype_name(static_cast<DType>(grad_dtype)));
    NVTE_CHECK((da == nullptr) == (db == nullptr), "da and db come together");
    NVTE_CHECK(da == nullptr || s.num <= kMaxAdapters, "a backward pass takes up to ", kMaxAdapters, " adapters, got ", s.num);
    NVTE_CHECK(s.tokens == 0 || (x && dy && a && b && adapter_ids && low), "a required pointer is NULL");
    const size_t need = backward_workspace(s).bytes;
    NVTE_CHECK(workspace != nullptr && workspace_bytes >= need, "workspace of ", workspace_bytes, " bytes, but ", need, " are needed");
    NVTE_CHECK(aligned16(workspace), "the workspace must be 16-byte aligned");
    char *ws = static_cast<char *>(workspace);
    if (s.type == kNVTEBFloat16)
      backward<bf16_t>(s, x, dy, a, b, adapter_ids, scaling, low, base_grad, dx, da, db, grad_dtype, ws, stream);
    else
      backward<f16_t>(s, x, dy, a, b, adapter_ids, scaling, low, base_grad, dx, da, db, grad_dtype, ws, stream);
  });
}

}  // extern "C"
