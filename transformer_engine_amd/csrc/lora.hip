// Low-rank adapters of many requests beside a shared projection (include/transformer_engine/amd_ext.h).
//
//   v[t] = A_a x[t]                      y[t]  = base[t]      + s_a B_a v[t]          a = ids[t], none if out of range
//   u[t] = B_a^T dy[t]                   dx[t] = base_grad[t] + s_a A_a^T u[t]
//   dA_a = sum_t s_a u[t] (x) x[t]       dB_a  = sum_t dy[t] (x) s_a v[t]             sums over the tokens of adapter a
//
// Forward: `shrink` (activations to rank vectors), then `expand` (rank vectors to activations).  Backward: `prepare` (the tokens
// of every adapter; B transposed, so that `shrink` reads it like A), `shrink`, `expand` together with `pack` (rank vectors as matrix
// operands, in the tokens' order), `wgrad` (outer products summed over an adapter's tokens), `join`.
// All of them are bound by the activations they stream (2 T (K + O) bytes and more against 2 T r (K + O) operations, r <= 128);
// the pools stay in L2.  A tile of tokens walks the distinct adapters among its own tokens, so any order of ids is right;
// values of other adapters' rows are never added, only selected, so a NaN or Inf stays in its own rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.h"
#include "device_utils.h"
#include "mfma16.h"
#include "transformer_engine/amd_ext.h"

namespace te {
namespace {

constexpr int kMaxRank = 128;
constexpr size_t kMaxTokens = 1u << 27;  // keeps every grid below 2^32 threads
constexpr int kMaxAdapters = 4096;  // of a backward pass: the plan kernel's histogram in LDS

__device__ __forceinline__ int valid_id(const int *ids, int64_t t, int64_t tokens, int num) {
  if (t >= tokens) return -1;
  const int id = ids[t];
  return id >= 0 && id < num ? id : -1;
}

constexpr int kBlock = 32;

// The tokens of every adapter in rising order, then those without one; each list padded to whole blocks with its last token, marked
// by the sign bit (see `prepare`).  Whatever a workgroup asks of it is one load away: these kernels are short, and a search through the
// adapters' first blocks was a chain of loads at the head of each.
struct Plan {
  int *order;      // [most_blocks * 32]; null: tokens are taken as they come
  int *owner;      // [most_blocks] each block's adapter, num: none
  int *ends;       // [2] blocks with an adapter, all blocks
  int *item_base;  // [num + 1] first work item of every adapter, and the end
  int2 *items;     // [most_items] each work item's first and last + 1 block; null: not wanted, nor item_base
};

// a lane's token of a tile of 16 MT, and its adapter: -1 none, -2 no token
struct TileToken {
  int64_t t;
  int id;
};
__device__ __forceinline__ TileToken tile_token(const Plan &plan, const int *ids, int64_t tile, int size, int lane, int64_t tokens,
                                                int num) {
  if (plan.order == nullptr) {
    const int64_t t = tile * size + lane;
    return {min(t, tokens - 1), lane < size && t < tokens ? valid_id(ids, t, tokens, num) : -2};
  }
  const int block = static_cast<int>(tile * size / kBlock);
  // past the end they are whatever memory held
  const int end = plan.ends[1], v = plan.order[tile * size + min(lane, size - 1)], a = plan.owner[block];
  if (block >= end) return {0, -2};
  return {v & INT_MAX, lane < size && v >= 0 ? (a < num ? a : -1) : -2};
}

// ====================================================================================
// shrink: out[slice][t][j] = sum over the slice's k of in[t][k] * pool[a][j][k]
// Reads every activation once (2 T K bytes); tokens are the rows of the product, ranks its columns, both operands come from memory in
// the matrix layout (eight consecutive k per lane), so LDS only joins the waves' sums.  8192 x 4096, rank 32: 21 us (3.2 TB/s);
// 8192 x 14336 right after the pass that wrote it: 74 us, of which the writing back of that pass's lines is part; 96 x 4096 with 48
// adapters of rank 16 (12.6 MB of pool, each adapter read by about two tiles): 6.0 us.
// ====================================================================================
struct ShrinkArgs {
  const uint16_t *in, *pool;
  const int *ids;
  Plan plan;
  float *out;
  int64_t tokens;
  int features, rank, num, slice;
};

template <int MT, int RT, bool GUARD, bool SMALL>
struct ShrinkBlock {  // 64 k of every row: one 128-byte line, 32 bytes of it per lane, two operands
  u32x4 a[MT][2], b[RT][2];
  // GUARD: the slice's ragged end, which is the row's (slices are multiples of 64)
  __device__ __forceinline__ void load(const ShrinkArgs &p, const uint16_t *const (&row)[MT], const uint16_t *const (&w)[RT], int k,
                                       int end) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = k + 8 * h, from = GUARD ? min(at, end - 8) : at;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (SMALL) a[m][h] = load8_any(row[m] + at, end - at, p.in + p.tokens * p.features);
        else if constexpr (GUARD) a[m][h] = without_head(load8(row[m] + from), at - from);
        else a[m][h] = load8(row[m] + from);
      }
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        if constexpr (SMALL) b[j][h] = load8_any(w[j] + at, end - at, p.pool + static_cast<int64_t>(p.num) * p.rank * p.features);
        else if constexpr (GUARD) b[j][h] = without_head(load8(w[j] + from), at - from);
        else b[j][h] = load8(w[j] + from);
      }
    }
  }
  template <typename E>
  __device__ __forceinline__ void multiply(f32x4 (&acc)[MT][RT]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[m][j] = mfma16<E>(a[m][h], b[j][h], acc[m][j]);
  }
};

// SMALL: rows of fewer than eight elements.
// grid: token tiles x slices x phases (the tile's n-th distinct adapter is phase n % gridDim.z's); the NW waves share the slice
template <typename E, int RT, int MT, int NW, int U, bool SMALL>
__global__ __launch_bounds__(NW * 64) void shrink_kernel(ShrinkArgs p) {
  __shared__ f32x4 red[NW][MT * RT][64];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const TileToken own = tile_token(p.plan, p.ids, blockIdx.x, 16 * MT, lane, p.tokens, p.num);
  const int id = own.id, token = static_cast<int>(own.t);
  const uint16_t *row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) row[m] = p.in + static_cast<int64_t>(__shfl(token, m * 16 + (lane & 15), 64)) * p.features;
  const int begin = blockIdx.y * p.slice, end = min(begin + p.slice, p.features);
  const int first = begin + wave * 64, kg = 16 * (lane >> 4);

  unsigned phase = 0;
  for (uint64_t left = __ballot(id >= 0); left != 0;) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const uint64_t mine = __ballot(id == cur);
    left &= ~mine;
    if (phase++ % gridDim.z != blockIdx.z) continue;
    f32x4 acc[MT][RT] = {};
    const uint16_t *w[RT];  // rank rows from `rank` on are computed from the last one and not kept
#pragma unroll
    for (int j = 0; j < RT; ++j)
      w[j] = p.pool + (static_cast<int64_t>(cur) * p.rank + min(j * 16 + (lane & 15), p.rank - 1)) * p.features;
    int k = first;
    for (; k + NW * 64 * (U - 1) + 64 <= end; k += NW * 64 * U) {
      ShrinkBlock<MT, RT, false, false> block[U];
#pragma unroll
      for (int u = 0; u < U; ++u) block[u].load(p, row, w, k + u * NW * 64 + kg, end);
      __builtin_amdgcn_sched_barrier(0);  // every load is on its way before the first product waits for one
#pragma unroll
      for (int u = 0; u < U; ++u) block[u].template multiply<E>(acc);
    }
    if constexpr (U > 1) {
      for (; k + 64 <= end; k += NW * 64) {
        ShrinkBlock<MT, RT, false, false> block;
        block.load(p, row, w, k + kg, end);
        block.template multiply<E>(acc);
      }
    }
    if (k < end) {
      ShrinkBlock<MT, RT, true, SMALL> block;
      block.load(p, row, w, k + kg, end);
      block.template multiply<E>(acc);
    }
    __syncthreads();  // the last adapter's sums are read
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < RT; ++j) red[wave][m * RT + j][lane] = acc[m][j];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * RT * 64; e += NW * 64) {
      const int l = e & 63, j = (e >> 6) % RT, m = (e >> 6) / RT;
      f32x4 s = red[0][m * RT + j][l];
#pragma unroll
      for (int n = 1; n < NW; ++n) s += red[n][m * RT + j][l];
      const int col = j * 16 + (l & 15);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = m * 16 + (l >> 4) * 4 + i;
        const int64_t t = __shfl(token, tok, 64);
        if (((mine >> tok) & 1) && col < p.rank) p.out[(blockIdx.y * p.tokens + t) * p.rank + col] = s[i];
      }
    }
  }
}

// one value of a rank vector: its slices in order, eight at a time on their way
__device__ __forceinline__ float sum_slices(const float *p, int slices, int64_t stride) {
  float s = 0.f;
  for (int s0 = 0; s0 < slices; s0 += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[min(s0 + i, slices - 1) * stride];
#pragma unroll
    for (int i = 0; i < 8; ++i) s += s0 + i < slices ? v[i] : 0.f;
  }
  return s;
}

// ====================================================================================
// expand: out[t][c] = base[t][c] + s_a sum_j (sum over slices of low[slice][t][j]) * w(c, j)
// w(c, j) = pool[a][c][j], or pool[a][j][c] (RMAJOR)
// Reads and writes 2 T O bytes each, which bounds it: 8192 x 14336, rank 32: 100 us (4.7 TB/s; 106 with the old values asked for only once the rank vectors were there).  A decode tile is bound by its adapters
// instead: 96 x 14336 with 48 of rank 16 (22 MB of pool, read about twice) 15 us.
// ====================================================================================
struct ExpandArgs {
  const float *low;
  const uint16_t *pool, *base;  // base may be null (zero) or out itself
  const float *scaling;         // null: 1
  const int *ids;
  Plan plan;
  uint16_t *out;
  int64_t tokens;
  int slices, features, rank, num, cols;  // cols: columns per workgroup, a multiple of 512
};

// A wave's step is 128 columns: operand f holds the columns c0 + 8 n + f, n = 0 .. 15.  D then leaves lane (n, lane group q), register i
// with the eight neighbours c0 + 8 n + 0 .. 7 of token 4 q + i over f, so that each of the four stores of a step writes 256 contiguous
// bytes of four tokens (tokens along the lanes instead, 64 bytes of sixteen a store: 119 against 103 us at 8192 x 14336, rank 32).
// Ends: a chunk of eight columns past the last takes the last eight, and its lanes write only what is theirs.  Likewise the ranks:
// `slot_rank` says which rank operand slot s stands for (-1: none, zero in the rank vector), so that the pool is always read in whole
// eights.  A rank past the last (RMAJOR) reads the last one again and meets such a zero.
__device__ __forceinline__ int slot_rank(int slot, int rank, bool rmajor) {
  const int first = slot & ~7, from = rmajor || rank < 8 ? first : min(first, rank - 8), r = from + (slot & 7);
  return r >= first && r < rank ? r : -1;
}

template <bool RMAJOR, bool SMALL>
__device__ __forceinline__ void pool_block(const ExpandArgs &p, int adapter, int lane, int c0, int j0, u32x4 (&f)[8]) {
  const int c = min(c0 + 8 * (lane & 15), max(p.features - 8, 0)), j = j0 + 8 * (lane >> 4);
  const uint16_t *w = p.pool + static_cast<int64_t>(adapter) * p.rank * p.features;
  const uint16_t *end = p.pool + static_cast<int64_t>(p.num) * p.rank * p.features;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (RMAJOR) {
      const uint16_t *at = w + static_cast<int64_t>(min(j + i, p.rank - 1)) * p.features + c;
      f[i] = SMALL ? load8_any(at, p.features - c, end) : load8(at);
    } else {
      const uint16_t *at = w + static_cast<int64_t>(min(c + i, p.features - 1)) * p.rank + (p.rank < 8 ? j : min(j, p.rank - 8));
      f[i] = SMALL ? load8_any(at, p.rank < 8 ? p.rank - j : 8, end) : load8(at);
    }
  }
}

// The tile's n-th distinct adapter is served by the workgroup of phase n % phases, tokens without one by phase 0.
template <typename E, int KT, int MT, bool RMAJOR, bool SMALL>
__device__ __forceinline__ void expand_tile(const ExpandArgs &p, int64_t tile, int columns, unsigned my_phase, unsigned phases,
                                            uint16_t (*s_hi)[KT * 32 + 8], uint16_t (*s_lo)[KT * 32 + 8]) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const TileToken own = tile_token(p.plan, p.ids, tile, 16 * MT, lane, p.tokens, p.num);
  const int id = own.id, token = static_cast<int>(own.t);
  uint64_t todo = __ballot(id >= 0), write = my_phase == 0 && p.base != p.out ? __ballot(id == -1) : 0;
  if (phases > 1) {
    unsigned phase = 0;
    uint64_t left = todo;
    todo = 0;
    while (left != 0) {
      const uint64_t same = __ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(left)));
      left &= ~same;
      if (phase++ % phases == my_phase) todo |= same;
    }
  }
  write |= todo;
  if (write == 0) return;
  const int begin = columns * p.cols, end = min(begin + p.cols, p.features);
  // All that the first step reads is on its way before anything waits: the rank vectors, which are needed first, then the pool's
  // operands and the columns' old values; later ones from the moment on that their predecessors are used up.
  const float scale = p.scaling != nullptr && id >= 0 ? p.scaling[id] : 1.f;
  constexpr int kMine = 2 * MT * KT;  // values per thread
  constexpr int kBatch = (MT == 1 ? 32 : 16) / kMine;  // slices on their way at once; many tokens have few
  const float *low[kMine];
#pragma unroll
  for (int n = 0; n < kMine; ++n) {
    const int e = threadIdx.x + 256 * n, tok = e / (KT * 32), j = e % (KT * 32);
    low[n] = p.low + static_cast<int64_t>(__shfl(token, tok, 64)) * p.rank + max(slot_rank(j, p.rank, RMAJOR), 0);
  }
  const int64_t stride = p.tokens * p.rank;
  float part[kBatch][kMine], v[kMine] = {};
  auto load_low = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int n = 0; n < kMine; ++n) part[i][n] = low[n][min(s0 + i, p.slices - 1) * stride];
  };
  load_low(0);
  __builtin_amdgcn_sched_barrier(0);

  u32x4 f[KT][8];
  auto load_pool = [&](uint64_t left, int c0) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
#pragma unroll
    for (int k = 0; k < KT; ++k) pool_block<RMAJOR, SMALL>(p, cur, lane, c0, k * 32, f[k]);
  };
  int c0 = begin + wave * 128;
  if (todo != 0 && c0 < end) load_pool(todo, c0);

  int my_id[MT][4];       // of the lane's four tokens per subtile
  int row[MT][4];         // they themselves; one that is not written here reads the first that is
  const int any = __builtin_ctzll(write);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = m * 16 + 4 * (lane >> 4) + i;
      my_id[m][i] = __shfl(id, tok, 64);
      row[m][i] = __shfl(token, ((write >> tok) & 1) ? tok : any, 64);
    }
  // the columns' old values travel a step ahead
  u32x4 base[MT][4], ahead[MT][4];
  auto load_base = [&](int c0, u32x4 (&v)[MT][4]) {
    const int c = min(c0 + 8 * (lane & 15), max(p.features - 8, 0));
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t *from = p.base + (static_cast<int64_t>(row[m][i]) * p.features + c);
        v[m][i] = SMALL ? load8_any(from, p.features - c, p.base + p.tokens * p.features) : load8(from);
      }
  };
  if (p.base == nullptr) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) base[m][i] = ahead[m][i] = u32x4{0u, 0u, 0u, 0u};
  } else if (c0 < end) {
    load_base(c0, base);
  }
  __builtin_amdgcn_sched_barrier(0);

  for (int s0 = 0;;) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int n = 0; n < kMine; ++n) v[n] += s0 + i < p.slices ? part[i][n] : 0.f;
    if ((s0 += kBatch) >= p.slices) break;
    load_low(s0);
  }
#pragma unroll
  for (int n = 0; n < kMine; ++n) {
    const int e = threadIdx.x + 256 * n, tok = e / (KT * 32), j = e % (KT * 32);
    const float s = __shfl(scale, tok, 64);
    __bf16 h, l;
    split1(((todo >> tok) & 1) && slot_rank(j, p.rank, RMAJOR) >= 0 ? s * v[n] : 0.f, h, l);
    s_hi[tok][j] = bits16(h);
    s_lo[tok][j] = bits16(l);
  }
  // only the LDS writes have to be done: the loads stay on their way
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  u32x4 hi[MT][KT], lo[MT][KT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      hi[m][k] = *reinterpret_cast<const u32x4 *>(&s_hi[m * 16 + (lane & 15)][k * 32 + (lane >> 4) * 8]);
      lo[m][k] = *reinterpret_cast<const u32x4 *>(&s_lo[m * 16 + (lane & 15)][k * 32 + (lane >> 4) * 8]);
    }
  f32x4 res[MT][8];
  uint64_t left = todo;
  while (c0 < end) {
    if (left == todo) {  // a new step
      if (p.base != nullptr && c0 + 512 < end) load_base(c0 + 512, ahead);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 8; ++i) res[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (left != 0) {
      const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      left &= ~__ballot(id == cur);
      if constexpr (RMAJOR) {
#pragma unroll
        for (int k = 0; k < KT; ++k) transpose8x8(f[k]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f32x4 acc[MT] = {};
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const Terms<E> terms(f[k][i]);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = mfma16_split<E, true>(terms, hi[m][k], lo[m][k], acc[m]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < 4; ++t) res[m][i][t] = my_id[m][t] == cur ? acc[m][t] : res[m][i][t];
      }
    }
    const bool done = left == 0;
    const int next = done ? c0 + 512 : c0;
    if (done) left = todo;
    if (left != 0 && next < end) load_pool(left, next);
    if (done) {
      const int c = c0 + 8 * (lane & 15), first = min(c, max(p.features - 8, 0));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((write >> (m * 16 + 4 * (lane >> 4) + i)) & 1)) continue;
          uint16_t *to = p.out + static_cast<int64_t>(row[m][i]) * p.features;
          E o[8];
          const E *old = reinterpret_cast<const E *>(&base[m][i]);
#pragma unroll
          for (int k = 0; k < 8; ++k) narrow(widen(old[k]) + res[m][k][i], o[k]);
          // a token without an adapter keeps its bits (-0 + 0 would be +0)
          const u32x4 sum = *reinterpret_cast<const u32x4 *>(o), bits = my_id[m][i] < 0 ? base[m][i] : sum;
          if (c + 8 <= p.features) {
            store8(to + c, bits);
          } else if (c < p.features) {
            uint64_t half[2] = {bits[0] | static_cast<uint64_t>(bits[1]) << 32, bits[2] | static_cast<uint64_t>(bits[3]) << 32};
#pragma unroll 1
            for (int k = c - first; k < min(8, p.features - first); ++k)
              to[first + k] = static_cast<uint16_t>((k < 4 ? half[0] : half[1]) >> (16 * (k & 3)));
          }
        }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) base[m][i] = ahead[m][i];
    }
    c0 = next;
  }
}

// grid: token tiles x column ranges x phases
template <typename E, int KT, int MT, bool SMALL>
__global__ __launch_bounds__(256, KT == 1 ? 2 : 1) void expand_kernel(ExpandArgs p) {
  // 16-byte aligned rows, neighbouring rows in different banks
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[16 * MT][KT * 32 + 8], s_lo[16 * MT][KT * 32 + 8];
  expand_tile<E, KT, MT, false, SMALL>(p, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, s_hi, s_lo);
}

// ====================================================================================
// prepare: the lists of a Plan, and where each adapter's work items of `per_item` blocks begin.  And B[a] [features][rank] transposed to
// [rank][features].
// One workgroup per adapter counts all ids for itself (T * 4 bytes out of L2), so nothing is exchanged; its sixteen waves own
// consecutive stretches of the tokens.  Two dependent walks of the ids: latency (2931 tokens 6.0 us, 8192 tokens and a 32 x 14336
// transpose 8.0 us; 8192 tokens of 64 adapters in any order 13 us, of 4096 adapters 125 us).
// ====================================================================================
struct PrepareArgs {
  const int *ids;
  const uint16_t *pool;
  uint16_t *transposed;
  Plan plan;
  int64_t tokens;
  int features, rank, num, per_item, lists;  // lists: workgroups of the first part, num + 1 or none
  int64_t pieces;                            // of the second part, dealt out over its workgroups
};

__device__ __forceinline__ int sum_1024(int v, int *scratch) {  // valid in every thread
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += scratch[w];
  return s;
}

// a == num: the tokens without an adapter
__device__ void list_tokens(const PrepareArgs &p, int a, int *hist, int *scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t stretch = ((p.tokens + 15) / 16 + 63) / 64 * 64, from = wave * stretch;
  const int64_t to = min(from + stretch, p.tokens);
  // the adapters of 256 tokens (num: none, -1: past the stretch), four loads on their way at once
  auto ids_of = [&](int64_t t0, int (&id)[4]) {
    int raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = p.ids[min(t0 + 64 * i + lane, p.tokens - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = t0 + 64 * i + lane >= to ? -1 : raw[i] >= 0 && raw[i] < p.num ? raw[i] : p.num;
  };
  for (int i = threadIdx.x; i <= p.num; i += 1024) hist[i] = 0;
  __syncthreads();
  int id[4], count = 0;
  for (int64_t t0 = from; t0 < to; t0 += 256) {
    ids_of(t0, id);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      count += __popcll(__ballot(id[i] == a));
      // one addition for each of the first few distinct ids, since a run would queue up on one address; what is left is mixed
      uint64_t left = __ballot(id[i] >= 0);
      for (int n = 0; n < 4 && left != 0; ++n) {
        const int cur = __builtin_amdgcn_readlane(id[i], __builtin_ctzll(left));
        const uint64_t same = __ballot(id[i] == cur);
        left &= ~same;
        if (lane == 0) atomicAdd(&hist[cur], __popcll(same));
      }
      if ((left >> lane) & 1) atomicAdd(&hist[id[i]], 1);
    }
  }
  __syncthreads();
  int blocks = 0, items = 0;
  for (int i = threadIdx.x; i < a; i += 1024) {
    const int b = (hist[i] + kBlock - 1) / kBlock;
    blocks += b;
    items += (b + p.per_item - 1) / p.per_item;
  }
  blocks = sum_1024(blocks, scratch);
  items = sum_1024(items, scratch);
  const int mine = hist[a], my_blocks = (mine + kBlock - 1) / kBlock;
  if (threadIdx.x == 0) {
    if (p.plan.items != nullptr) p.plan.item_base[a] = items;  // that of a == num is the end
    if (a == p.num) {
      p.plan.ends[0] = blocks;
      p.plan.ends[1] = blocks + my_blocks;
    }
  }
  if (mine == 0) return;
  for (int b = threadIdx.x; b < my_blocks; b += 1024) p.plan.owner[blocks + b] = a;
  if (p.plan.items != nullptr && a < p.num)
    for (int i = threadIdx.x, last = (my_blocks + p.per_item - 1) / p.per_item; i < last; i += 1024)
      p.plan.items[items + i] = int2{blocks + i * p.per_item, blocks + min((i + 1) * p.per_item, my_blocks)};
  int *order = p.plan.order + static_cast<int64_t>(blocks) * kBlock;
  __syncthreads();  // the last sum is read
  if (lane == 0) scratch[wave] = count;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < wave; ++w) at += scratch[w];
  for (int64_t t0 = from; t0 < to; t0 += 256) {
    if (stretch > 256) ids_of(t0, id);  // else they are still there
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool hit = id[i] == a;
      const uint64_t m = __ballot(hit);
      const int slot = at + __popcll(m & ((1ull << lane) - 1)), t = static_cast<int>(t0) + 64 * i + lane;
      if (hit) order[slot] = t;
      if (hit && slot == mine - 1)
        for (int k = mine; k < my_blocks * kBlock; ++k) order[k] = t | INT_MIN;
      at += __popcll(m);
    }
  }
}

// 64 features of one adapter's matrix
__device__ void transpose_rows(const PrepareArgs &p, int64_t piece, uint16_t *s) {
  const int per_adapter = (p.features + 63) / 64;
  const int64_t a = piece / per_adapter;
  const int f0 = static_cast<int>(piece % per_adapter) * 64, n = min(64, p.features - f0);
  const uint16_t *in = p.pool + (a * p.features + f0) * p.rank;
  for (int e = threadIdx.x; e < n * p.rank; e += 1024) s[e / p.rank * (p.rank + 1) + e % p.rank] = in[e];
  __syncthreads();
  uint16_t *out = p.transposed + a * p.features * p.rank + f0;
  for (int e = threadIdx.x; e < 64 * p.rank; e += 1024) {
    const int f = e & 63, j = e >> 6;
    if (f < n) out[static_cast<int64_t>(j) * p.features + f] = s[f * (p.rank + 1) + j];
  }
}

__global__ __launch_bounds__(1024) void prepare_kernel(PrepareArgs p) {
  __shared__ union {
    int hist[kMaxAdapters + 1];
    uint16_t rows[64 * (kMaxRank + 1)];
  } s;
  __shared__ int scratch[16];
  if (static_cast<int>(blockIdx.x) < p.lists) {
    list_tokens(p, blockIdx.x, s.hist, scratch);
    return;
  }
  for (int64_t piece = blockIdx.x - p.lists;;) {
    transpose_rows(p, piece, s.rows);
    piece += gridDim.x - p.lists;
    if (piece >= p.pieces) return;
    __syncthreads();  // the last piece is written
  }
}

// ====================================================================================
// pack: the scaled rank vectors of every block of 32 tokens as matrix operands: [block][16 ranks][hi, lo][lane][8 tokens]
// ====================================================================================
struct PackSide {
  const float *low;  // [slices][tokens][rank]
  uint16_t *packed;
  int slices;
};
struct PackArgs {
  PackSide side[2];
  const float *scaling;
  Plan plan;
  int64_t tokens;
  int rank, num;
};

__device__ __forceinline__ void pack_block(const PackArgs &p, const PackSide &side, int block) {
  if (block >= p.plan.ends[0]) return;
  const float scale = p.scaling != nullptr ? p.scaling[p.plan.owner[block]] : 1.f;
  const int tiles = (p.rank + 15) / 16;
  uint16_t *out = side.packed + static_cast<int64_t>(block) * tiles * 1024;
  // neighbouring threads take neighbouring ranks of one token
  for (int e = threadIdx.x; e < kBlock * tiles * 16; e += 256) {
    const int j = e % (tiles * 16), tok = e / (tiles * 16);
    const int t = p.plan.order[block * kBlock + tok];
    const float s = sum_slices(side.low + static_cast<int64_t>(t & INT_MAX) * p.rank + min(j, p.rank - 1), side.slices, p.tokens * p.rank);
    __bf16 h, l;
    split1(t >= 0 && j < p.rank ? scale * s : 0.f, h, l);
    const int at = (j >> 4) * 1024 + ((j & 15) + 16 * (tok >> 3)) * 8 + (tok & 7);
    out[at] = bits16(h);
    out[at + 512] = bits16(l);
  }
}

// the backward pass's `expand` and `pack` read the same rank vectors and nothing of each other: one launch
template <typename E, int KT, int MT, bool SMALL>
__global__ __launch_bounds__(256, KT == 1 ? 2 : 1) void expand_pack_kernel(ExpandArgs p, PackArgs q, int column_ranges, int tiles, int phases,
                                                          int blocks) {
  __shared__ __attribute__((aligned(16))) uint16_t s_hi[16 * MT][KT * 32 + 8], s_lo[16 * MT][KT * 32 + 8];
  const int b = blockIdx.x + gridDim.x * blockIdx.y;
  if (b < 2 * blocks) pack_block(q, b < blocks ? q.side[0] : q.side[1], b < blocks ? b : b - blocks);
  else {
    const int n = (b - 2 * blocks) / tiles;
    if (n >= column_ranges * phases) return;
    expand_tile<E, KT, MT, true, SMALL>(p, (b - 2 * blocks) % tiles, n % column_ranges, n / column_ranges, phases, s_hi, s_lo);
  }
}

// ====================================================================================
// wgrad: one work item's sums over its tokens of w[t] (x) z[t]: dA with z = x, dB (transposed) with z = dy
// Reads every activation of x and dy once per 64 ranks, rows of 256 bytes, and turns 8 x 8 blocks round in registers (the tokens are k
// here); the rank vectors come packed as operands, shared by all column groups out of L2.  8192 tokens, 4096 + 14336 columns, rank 32:
// 58 us (5.2 TB/s); with rank vectors put together in the kernel 117 us, 64 columns per wave 69 us.  A work item's partial sums go to
// `join` in fp32 (8 us there): items add up in a fixed order, no atomics.
// ====================================================================================
struct WgradSide {
  const uint16_t *z;       // activations [tokens][features]
  const uint16_t *packed;  // rank vectors
  float *part;             // [item][rank][features]
  void *grad;              // [num][rank][features], or [num][features][rank] (the second side)
  int features, groups;    // groups: workgroups along the features, 512 columns each
};
struct WgradArgs {
  WgradSide side[2];
  Plan plan;
  int64_t tokens;
  int rank, num, grad_type;
};

struct WgradTokens {  // a lane's eight tokens of a block
  int t[8];
  __device__ __forceinline__ void load(const int *order, int block, int lane) {
    const int *from = order + static_cast<int64_t>(block) * kBlock + 8 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from[i];
  }
};

template <typename E, int RT, bool SMALL>
struct WgradBlock {  // 32 tokens x 128 columns, and their rank vectors (zero for padding, whose rows are the adapter's own)
  u32x4 z[8], w[RT][2];
  __device__ __forceinline__ void load(const WgradSide &side, int64_t all, const WgradTokens &tokens, int block, int rank_tiles,
                                       int j0, int c, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t *at = side.z + static_cast<int64_t>(tokens.t[i] & INT_MAX) * side.features + c;
      z[i] = SMALL ? load8_any(at, side.features - c, side.z + all * side.features) : load8_once(at);
    }
    const uint16_t *from = side.packed + (static_cast<int64_t>(block) * rank_tiles + j0) * 1024 + lane * 8;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      w[j][0] = *reinterpret_cast<const u32x4 *>(from + min(j, rank_tiles - j0 - 1) * 1024);
      w[j][1] = *reinterpret_cast<const u32x4 *>(from + min(j, rank_tiles - j0 - 1) * 1024 + 512);
    }
  }
  __device__ __forceinline__ void multiply(f32x4 (&acc)[RT][8]) {
    transpose8x8(z);
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const Terms<E> terms(z[f]);
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[j][f] = mfma16_split<E, true>(terms, w[j][0], w[j][1], acc[j][f]);
    }
  }
};

// grid: column groups of both sides  x  work items (an upper bound; the rest leave at once)  x  64 ranks
template <typename E, int RT, bool SMALL>
__global__ __launch_bounds__(256, RT <= 2 ? 2 : 1) void wgrad_kernel(WgradArgs p) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int item = blockIdx.y;
  if (item >= p.plan.item_base[p.num]) return;
  const bool second = static_cast<int>(blockIdx.x) >= p.side[0].groups;
  const WgradSide side = second ? p.side[1] : p.side[0];
  const int c0 = (blockIdx.x - (second ? p.side[0].groups : 0)) * 512 + wave * 128;
  if (c0 >= side.features) return;
  const int first = __builtin_amdgcn_readfirstlane(p.plan.items[item].x), last = __builtin_amdgcn_readfirstlane(p.plan.items[item].y);
  // a lane past the last column computes the last eight once more, and stores the same values
  const int c = min(c0 + 8 * (lane & 15), max(side.features - 8, 0));
  const int rank_tiles = (p.rank + 15) / 16, j0 = blockIdx.z * 4;
  const int *order = p.plan.order;
  f32x4 acc[RT][8] = {};
  // while the products of one block run, the next block is on its way, and the one after's token numbers
  WgradTokens t0, t1;
  WgradBlock<E, RT, SMALL> even, odd;
  t0.load(order, first, lane);
  t1.load(order, min(first + 1, last - 1), lane);
  even.load(side, p.tokens, t0, first, rank_tiles, j0, c, lane);
  for (int b = first;;) {
    t0.load(order, min(b + 2, last - 1), lane);
    odd.load(side, p.tokens, t1, min(b + 1, last - 1), rank_tiles, j0, c, lane);
    __builtin_amdgcn_sched_barrier(0);
    even.multiply(acc);
    if (++b >= last) break;
    t1.load(order, min(b + 2, last - 1), lane);
    even.load(side, p.tokens, t0, min(b + 1, last - 1), rank_tiles, j0, c, lane);
    __builtin_amdgcn_sched_barrier(0);
    odd.multiply(acc);
    if (++b >= last) break;
  }
  float *out = side.part + static_cast<int64_t>(item) * p.rank * side.features + c;
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (j0 + j) * 16 + (lane >> 4) * 4 + i;
      if (row >= p.rank) continue;
      float *to = out + static_cast<int64_t>(row) * side.features;
      if (!SMALL || side.features >= 8) {
        *reinterpret_cast<f32x4_any *>(to) = f32x4{acc[j][0][i], acc[j][1][i], acc[j][2][i], acc[j][3][i]};
        *reinterpret_cast<f32x4_any *>(to + 4) = f32x4{acc[j][4][i], acc[j][5][i], acc[j][6][i], acc[j][7][i]};
      } else {
#pragma unroll
        for (int f = 0; f < 7; ++f)
          if (f < side.features) to[f] = acc[j][f][i];
      }
    }
}

// join: the sum of an adapter's work items in their order; zero for an adapter without tokens.  A workgroup takes 64 columns of
// 16 ranks: dA is written as it is read, dB turned round in LDS.  grid: column pieces of both sides x adapters x rank groups
__global__ __launch_bounds__(256) void join_kernel(WgradArgs p, int pieces) {
  __shared__ float s[64][17];
  const int a = blockIdx.y, j0 = blockIdx.z * 16;
  const bool second = static_cast<int>(blockIdx.x) >= pieces;
  const WgradSide side = second ? p.side[1] : p.side[0];
  const int c0 = (blockIdx.x - (second ? pieces : 0)) * 64, columns = min(64, side.features - c0), ranks = min(16, p.rank - j0);
  const int first = p.plan.item_base[a], items = p.plan.item_base[a + 1] - first;
  const int64_t size = static_cast<int64_t>(p.rank) * side.features;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float *part = side.part + first * size + min(c0 + lane, side.features - 1);
  float v[4] = {};
  for (int i0 = 0; i0 < items; i0 += 4) {
    float w[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        w[i][n] = part[min(i0 + i, items - 1) * size + static_cast<int64_t>(min(j0 + 4 * wave + n, p.rank - 1)) * side.features];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] += i0 + i < items ? w[i][n] : 0.f;
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int j = 4 * wave + n;
    if (second) s[lane][j] = v[n];
    else if (lane < columns && j < ranks)
      store1(side.grad, a * size + static_cast<int64_t>(j0 + j) * side.features + c0 + lane, p.grad_type, v[n]);
  }
  if (!second) return;
  __syncthreads();
  for (int e = threadIdx.x; e < columns * 16; e += 256)
    if ((e & 15) < ranks)
      store1(side.grad, a * size + static_cast<int64_t>(c0 + (e >> 4)) * p.rank + j0 + (e & 15), p.grad_type, s[e >> 4][e & 15]);
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
  NVTE_CHECK(tokens <= kMaxTokens, "up to ", kMaxTokens, " tokens per call, got ", tokens);
  return {static_cast<int64_t>(tokens), static_cast<int>(in), static_cast<int>(out), static_cast<int>(rank), static_cast<int>(num), t};
}

// Few tokens leave most CUs without a tile, so the features are cut into slices (a multiple of 64, at least 512) until about
// 768 workgroups run, three per CU; whoever reads the rank vectors adds the slices.  From 4096 tokens on a workgroup takes 32 tokens for one
// reading of the adapter (8192 x 14336, rank 32: 74 against 86 us with 16; 2048 x 4096, rank 16, within 2 %).
bool many_tokens(int64_t tokens) { return tokens >= 4096; }
int slice_of(int64_t tokens, int features) {
  const int64_t tiles = std::max<int64_t>(1, ceil_div(tokens, many_tokens(tokens) ? 32 : 16));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(768 / tiles, ceil_div(features, 512)));
  return static_cast<int>(round_up(ceil_div(features, static_cast<size_t>(want)), 64));
}
int num_slices(int64_t tokens, int features) { return static_cast<int>(ceil_div(features, slice_of(tokens, features))); }

// A decode tile's adapters go to workgroups of their own while there are too few of them: expand of 96 tokens, 48 adapters takes 15 us
// with up to 768, 17.5 with 448, 18.4 with 1024 (a second round of workgroups).
int phases_of(int64_t workgroups, int64_t tokens, int num) {
  const int64_t most = std::min<int64_t>(std::min<int64_t>(num, tokens), 16);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 768 / workgroups)));
}

// every list's last block may be partly filled
int64_t most_blocks(int64_t tokens, int num) { return tokens / kBlock + std::min<int64_t>(num + 1ll, tokens); }
int64_t tiles_of(const Plan &plan, int64_t tokens, int num, int size) {
  return plan.order != nullptr ? most_blocks(tokens, num) * kBlock / size : static_cast<int64_t>(ceil_div(tokens, size));
}

// Tokens are put in order of their adapters first where tiles would otherwise walk through many, and where listing them costs less than
// that: `prepare` reads all ids once for every adapter.  A forward pass of 4096 -> 4096, rank 16, ids in any order, in us with / without:
//   adapters   512 tokens    1024         2048         4096         8192
//   64         30 / 44       31 / 76      40 / 135     63 / 320     97 / 631
//   256        52 / 46       54 / 88      61 / 153     76 / 372     123 / 737
//   1024       88 / 52       115 / 98     133 / 162    153 / 380    183 / 762
//   4096       125 / 59      164 / 110    248 / 167    354 / 379    462 / 771
// Requests that lie back to back pay for nothing (2048 tokens of 64: 39 / 36; 4096 of 4096: 354 / 281); below 512 tokens both orders lose.
// A pass that lists the tokens anyway, for its weight gradients, follows the lists.
bool ordered(int64_t tokens, int num, bool listed) {
  return tokens >= 512 && num > 1 && num <= kMaxAdapters && (listed || tokens >= 2ll * num);
}

template <typename E, int RT, int MT, int NW, int U, bool SMALL = false>
void launch_shrink(const ShrinkArgs &p, int slices, hipStream_t stream) {
  const int64_t tiles = tiles_of(p.plan, p.tokens, p.num, 16 * MT);
  const int phases = p.plan.order != nullptr ? 1 : phases_of(tiles * slices, p.tokens, p.num);
  hipLaunchKernelGGL((shrink_kernel<E, RT, MT, NW, U, SMALL>), dim3(tiles, slices, phases), dim3(NW * 64), 0, stream, p);
  NVTE_CHECK_HIP(hipGetLastError());
}

template <typename E>
void shrink(const void *in, const void *pool, const int *ids, const Plan &plan, float *out, int64_t tokens, int features, int rank,
            int num, hipStream_t stream) {
  const ShrinkArgs p{static_cast<const uint16_t *>(in), static_cast<const uint16_t *>(pool), ids, plan, out, tokens, features, rank,
                     num, slice_of(tokens, features)};
  const int slices = num_slices(tokens, features);
  const bool many = many_tokens(tokens);
  if (features < 8) {
    launch_shrink<E, 8, 1, 4, 1, true>(p, slices, stream);
  } else if (rank <= 16) {
    many ? launch_shrink<E, 1, 2, 4, 1>(p, slices, stream) : launch_shrink<E, 1, 1, 4, 2>(p, slices, stream);
  } else if (rank <= 32) {
    many ? launch_shrink<E, 2, 2, 4, 1>(p, slices, stream) : launch_shrink<E, 2, 1, 4, 2>(p, slices, stream);
  } else if (rank <= 64) {
    many ? launch_shrink<E, 4, 2, 4, 1>(p, slices, stream) : launch_shrink<E, 4, 1, 4, 1>(p, slices, stream);
  } else {
    many ? launch_shrink<E, 8, 2, 4, 1>(p, slices, stream) : launch_shrink<E, 8, 1, 4, 1>(p, slices, stream);
  }
}

// Runs launch(KT, MT, SMALL) as integral constants: 32 ranks per operand, 16 tokens per tile.  32 tokens share one reading of the adapter
// from 1024 tokens on: whole forward passes in us, with 32 / with 16, 1024 x 4096 x 4096 rank 16 24.5 / 25.0, 2048 likewise 31.7 / 35.4,
// 4096 x 8192 x 8192 rank 32 70.5 / 75.1, 8192 x 4096 x 14336 rank 64 202 / 227; the other way at rank 64 of 4096 x 4096 x 4096 59 / 56 and
// four adapters of rank 16 in 8192 x 4096 x 14336 167 / 159.
template <typename Launch>
void expand_variant(int rank, int64_t tokens, bool small_features, bool small_rank, Launch &&launch) {
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  const bool many = tokens >= 1024;
  if (small_features) launch(Four(), One(), std::true_type());
  else if (small_rank) many ? launch(One(), Two(), std::true_type()) : launch(One(), One(), std::true_type());
  else if (rank <= 32) many ? launch(One(), Two(), std::false_type()) : launch(One(), One(), std::false_type());
  else if (rank <= 64) many ? launch(Two(), Two(), std::false_type()) : launch(Two(), One(), std::false_type());
  else launch(Four(), One(), std::false_type());
}

// columns per workgroup: 512 (a step of its four waves) until there are about 1024 workgroups
int columns_of(int64_t tiles, int features) {
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(ceil_div(features, 512), 1024 / tiles));
  return static_cast<int>(round_up(ceil_div(features, static_cast<size_t>(want)), 512));
}

template <typename E>
void expand(ExpandArgs p, hipStream_t stream) {
  expand_variant(p.rank, p.tokens, p.features < 8, p.rank < 8, [&](auto kt, auto mt, auto small) {
    const int64_t tiles = tiles_of(p.plan, p.tokens, p.num, 16 * mt());
    p.cols = columns_of(tiles, p.features);
    const int64_t ranges = ceil_div(p.features, p.cols);
    const int phases = p.plan.order != nullptr ? 1 : phases_of(tiles * ranges, p.tokens, p.num);
    hipLaunchKernelGGL((expand_kernel<E, kt(), mt(), small()>), dim3(tiles, ranges, phases), dim3(256), 0, stream, p);
    NVTE_CHECK_HIP(hipGetLastError());
  });
}

template <typename E>
void expand_and_pack(ExpandArgs p, const PackArgs &q, int64_t blocks, hipStream_t stream) {
  expand_variant(p.rank, p.tokens, p.features < 8, false, [&](auto kt, auto mt, auto small) {
    const int64_t tiles = tiles_of(p.plan, p.tokens, p.num, 16 * mt());
    p.cols = columns_of(tiles, p.features);
    const int64_t ranges = p.out != nullptr ? ceil_div(p.features, p.cols) : 0;
    const int phases = p.plan.order != nullptr ? 1 : phases_of(std::max<int64_t>(1, tiles * ranges), p.tokens, p.num);
    const int64_t all = 2 * blocks + tiles * ranges * phases, grid = std::min<int64_t>(all, 1 << 23);  // fewer than 2^32 threads along x
    if (all == 0) return;
    hipLaunchKernelGGL((expand_pack_kernel<E, kt(), mt(), small()>), dim3(grid, ceil_div(all, grid)), dim3(256), 0, stream, p, q, static_cast<int>(ranges),
                       static_cast<int>(tiles), phases, static_cast<int>(blocks));
    NVTE_CHECK_HIP(hipGetLastError());
  });
}

template <typename E>
void launch_wgrad(const WgradArgs &p, unsigned items, hipStream_t stream) {
  const dim3 grid(p.side[0].groups + p.side[1].groups, items, ceil_div(p.rank, 64));
  if (p.side[0].features < 8 || p.side[1].features < 8) hipLaunchKernelGGL((wgrad_kernel<E, 4, true>), grid, dim3(256), 0, stream, p);
  else if (p.rank <= 16) hipLaunchKernelGGL((wgrad_kernel<E, 1, false>), grid, dim3(256), 0, stream, p);
  else if (p.rank <= 32) hipLaunchKernelGGL((wgrad_kernel<E, 2, false>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((wgrad_kernel<E, 4, false>), grid, dim3(256), 0, stream, p);
  NVTE_CHECK_HIP(hipGetLastError());
}

// how many blocks of 32 tokens a work item sums: enough items for about eight waves per CU
int blocks_per_item(const Shape &s) {
  const int64_t columns = ceil_div(s.in, 512) + ceil_div(s.out, 512);
  const int64_t items = std::max<int64_t>(1, 512 / columns);
  return static_cast<int>(std::max<size_t>(2, ceil_div(ceil_div(s.tokens, kBlock), items)));
}
int64_t most_items(const Shape &s) {
  return most_blocks(s.tokens, s.num) / blocks_per_item(s) + std::min<int64_t>(s.num, s.tokens);
}

// one launch: the lists, if wanted, and B transposed, if given
void prepare(const Shape &s, const int *ids, const Plan &plan, bool lists, const void *b, uint16_t *transposed, hipStream_t stream) {
  const int64_t pieces = b != nullptr ? static_cast<int64_t>(s.num) * ceil_div(s.out, 64) : 0, first = lists ? s.num + 1 : 0;
  const PrepareArgs p{ids, static_cast<const uint16_t *>(b), transposed, plan, s.tokens, s.out, s.rank, s.num, blocks_per_item(s),
                      static_cast<int>(first), pieces};
  // a launch has fewer than 2^32 threads
  hipLaunchKernelGGL(prepare_kernel, dim3(first + std::min<int64_t>(pieces, 1 << 21)), dim3(1024), 0, stream, p);
  NVTE_CHECK_HIP(hipGetLastError());
}

struct Space {  // offsets into a workspace
  size_t at = 0;
  size_t take(size_t bytes) {
    const size_t here = at;
    at += round_up(bytes, 256);
    return here;
  }
};

struct ForwardWorkspace {
  size_t order, owner, ends, bytes;
  Plan plan(char *ws) const {
    return {reinterpret_cast<int *>(ws + order), reinterpret_cast<int *>(ws + owner), reinterpret_cast<int *>(ws + ends), nullptr,
            nullptr};
  }
};
ForwardWorkspace forward_workspace(int64_t tokens, int num) {
  if (!ordered(tokens, num, false)) return {};
  ForwardWorkspace w{};
  Space space;
  w.order = space.take(most_blocks(tokens, num) * kBlock * sizeof(int));
  w.owner = space.take(most_blocks(tokens, num) * sizeof(int));
  w.ends = space.take(2 * sizeof(int));
  w.bytes = space.at;
  return w;
}

struct BackwardWorkspace {
  size_t low, transposed, order, owner, ends, item_base, items, packed_a, packed_b, part_a, part_b, bytes;
  bool lists, wgrad;
  Plan plan(char *ws) const {
    if (!lists) return {};
    return {reinterpret_cast<int *>(ws + order), reinterpret_cast<int *>(ws + owner), reinterpret_cast<int *>(ws + ends),
            wgrad ? reinterpret_cast<int *>(ws + item_base) : nullptr, wgrad ? reinterpret_cast<int2 *>(ws + items) : nullptr};
  }
};
// Weight gradients take by far the most of it (a share of [rank][in + out] in fp32 for every work item), so a pass without them
// has a size of its own, in which `in` has no part.
BackwardWorkspace backward_workspace(const Shape &s, bool wgrad) {
  BackwardWorkspace w{};
  Space space;
  auto take = [&](size_t bytes) { return space.take(bytes); };
  w.wgrad = wgrad;
  w.lists = wgrad || ordered(s.tokens, s.num, false);
  w.low = take(static_cast<size_t>(num_slices(s.tokens, s.out)) * s.tokens * s.rank * sizeof(float));
  w.transposed = take(s.tokens > 0 ? static_cast<size_t>(s.num) * s.rank * s.out * 2 : 0);
  if (w.lists) {
    w.order = take(most_blocks(s.tokens, s.num) * kBlock * sizeof(int));
    w.owner = take(most_blocks(s.tokens, s.num) * sizeof(int));
    w.ends = take(2 * sizeof(int));
  }
  w.bytes = space.at;
  if (!wgrad) return w;
  w.item_base = take((static_cast<size_t>(s.num) + 1) * sizeof(int));
  w.items = take(most_items(s) * sizeof(int2));
  const size_t packed = static_cast<size_t>(most_blocks(s.tokens, s.num)) * ceil_div(s.rank, 16) * 2048;
  w.packed_a = take(packed);
  w.packed_b = take(packed);
  w.part_a = take(static_cast<size_t>(most_items(s)) * s.rank * s.in * sizeof(float));
  w.part_b = take(static_cast<size_t>(most_items(s)) * s.rank * s.out * sizeof(float));
  w.bytes = space.at;
  return w;
}

template <typename E>
void backward(const Shape &s, const void *x, const void *dy, const void *a, const void *b, const int *ids, const float *scaling,
              const float *low, const void *base_grad, void *dx, void *da, void *db, int grad_type, char *ws, hipStream_t stream) {
  const bool wgrad = da != nullptr;
  if (!wgrad && (dx == nullptr || s.tokens == 0)) return;
  const BackwardWorkspace w = backward_workspace(s, wgrad);
  float *up = reinterpret_cast<float *>(ws + w.low);
  uint16_t *bt = reinterpret_cast<uint16_t *>(ws + w.transposed);
  const Plan plan = w.plan(ws);
  prepare(s, ids, plan, w.lists, s.tokens > 0 ? b : nullptr, bt, stream);
  const Plan tiles = ordered(s.tokens, s.num, wgrad) ? plan : Plan{};
  const int64_t blocks = wgrad ? most_blocks(s.tokens, s.num) : 0;
  uint16_t *packed_a = reinterpret_cast<uint16_t *>(ws + w.packed_a), *packed_b = reinterpret_cast<uint16_t *>(ws + w.packed_b);
  if (s.tokens > 0) {
    shrink<E>(dy, bt, ids, tiles, up, s.tokens, s.out, s.rank, s.num, stream);
    const ExpandArgs e{up, static_cast<const uint16_t *>(a), static_cast<const uint16_t *>(base_grad), scaling, ids, tiles,
                       static_cast<uint16_t *>(dx), s.tokens, num_slices(s.tokens, s.out), s.in, s.rank, s.num, 0};
    const PackArgs q{{{up, packed_a, num_slices(s.tokens, s.out)}, {low, packed_b, num_slices(s.tokens, s.in)}}, scaling, plan,
                     s.tokens, s.rank, s.num};
    expand_and_pack<E>(e, q, blocks, stream);
  }
  if (!wgrad) return;
  WgradArgs p{};
  p.side[0] = {static_cast<const uint16_t *>(x), packed_a, reinterpret_cast<float *>(ws + w.part_a), da, s.in,
               static_cast<int>(ceil_div(s.in, 512))};
  p.side[1] = {static_cast<const uint16_t *>(dy), packed_b, reinterpret_cast<float *>(ws + w.part_b), db, s.out,
               static_cast<int>(ceil_div(s.out, 512))};
  p.plan = plan;
  p.tokens = s.tokens;
  p.rank = s.rank;
  p.num = s.num;
  p.grad_type = grad_type;
  const int64_t items = most_items(s);
  NVTE_CHECK(items <= 65535, "too many work items: ", items);
  if (items > 0) launch_wgrad<E>(p, static_cast<unsigned>(items), stream);
  const int columns = static_cast<int>(ceil_div(s.in, 64));
  hipLaunchKernelGGL(join_kernel, dim3(columns + ceil_div(s.out, 64), s.num, ceil_div(s.rank, 16)), dim3(256), 0, stream, p, columns);
  NVTE_CHECK_HIP(hipGetLastError());
}

}  // namespace
}  // namespace te

using namespace te;

extern "C" {

size_t nvte_amd_lora_num_slices(size_t tokens, size_t features) {
  return api_guard("nvte_amd_lora_num_slices", [&]() -> size_t {
    NVTE_CHECK(features >= 1 && features <= (1u << 24) && tokens <= kMaxTokens, "bad sizes ", tokens, " and ", features);
    return num_slices(static_cast<int64_t>(tokens), static_cast<int>(features));
  });
}

size_t nvte_amd_lora_forward_workspace_size(size_t tokens, size_t num_adapters) {
  return api_guard("nvte_amd_lora_forward_workspace_size", [&]() -> size_t {
    NVTE_CHECK(tokens <= kMaxTokens && num_adapters <= INT_MAX, "bad sizes ", tokens, " and ", num_adapters);
    return forward_workspace(static_cast<int64_t>(tokens), static_cast<int>(num_adapters)).bytes;
  });
}

void nvte_amd_lora_forward(const void *x, const void *a, const void *b, const int *adapter_ids, const float *scaling,
                           const void *base, void *out, float *low, size_t tokens, size_t in_features, size_t out_features,
                           size_t rank, size_t num_adapters, int dtype, void *workspace, size_t workspace_bytes,
                           hipStream_t stream) {
  api_guard("nvte_amd_lora_forward", [&] {
    const Shape s = shape_of(tokens, in_features, out_features, rank, num_adapters, dtype);
    if (s.tokens == 0) return;
    NVTE_CHECK(x && a && b && adapter_ids && out && low, "a required pointer is NULL");
    const ForwardWorkspace w = forward_workspace(s.tokens, s.num);
    NVTE_CHECK(w.bytes == 0 || (workspace != nullptr && workspace_bytes >= w.bytes), "workspace of ", workspace_bytes,
               " bytes, but ", w.bytes, " are needed");
    NVTE_CHECK(w.bytes == 0 || aligned16(workspace), "the workspace must be 16-byte aligned");
    char *ws = static_cast<char *>(workspace);
    Plan plan{};
    if (w.bytes != 0) {
      plan = w.plan(ws);
      prepare(s, adapter_ids, plan, true, nullptr, nullptr, stream);
    }
    const ExpandArgs p{low, static_cast<const uint16_t *>(b), static_cast<const uint16_t *>(base), scaling, adapter_ids, plan,
                       static_cast<uint16_t *>(out), s.tokens, num_slices(s.tokens, s.in), s.out, s.rank, s.num, 0};
    if (s.type == kNVTEBFloat16) {
      shrink<bf16_t>(x, a, adapter_ids, plan, low, s.tokens, s.in, s.rank, s.num, stream);
      expand<bf16_t>(p, stream);
    } else {
      shrink<f16_t>(x, a, adapter_ids, plan, low, s.tokens, s.in, s.rank, s.num, stream);
      expand<f16_t>(p, stream);
    }
  });
}

size_t nvte_amd_lora_backward_workspace_size(size_t tokens, size_t in_features, size_t out_features, size_t rank,
                                             size_t num_adapters) {
  return api_guard("nvte_amd_lora_backward_workspace_size", [&]() -> size_t {
    return backward_workspace(shape_of(tokens, in_features, out_features, rank, num_adapters, kNVTEBFloat16), true).bytes;
  });
}

size_t nvte_amd_lora_dgrad_workspace_size(size_t tokens, size_t out_features, size_t rank, size_t num_adapters) {
  return api_guard("nvte_amd_lora_dgrad_workspace_size", [&]() -> size_t {
    return backward_workspace(shape_of(tokens, 1, out_features, rank, num_adapters, kNVTEBFloat16), false).bytes;
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
    const size_t need = backward_workspace(s, da != nullptr).bytes;
    NVTE_CHECK(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace of ", workspace_bytes, " bytes, but ", need, " are needed");
    NVTE_CHECK(aligned16(workspace), "the workspace must be 16-byte aligned");
    char *ws = static_cast<char *>(workspace);
    if (s.type == kNVTEBFloat16)
      backward<bf16_t>(s, x, dy, a, b, adapter_ids, scaling, low, base_grad, dx, da, db, grad_dtype, ws, stream);
    else
      backward<f16_t>(s, x, dy, a, b, adapter_ids, scaling, low, base_grad, dx, da, db, grad_dtype, ws, stream);
  });
}

}  // extern "C"
