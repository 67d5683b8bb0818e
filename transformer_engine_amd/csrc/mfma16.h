// 16x16x32 matrix-instruction operands shared by lora.hip and moe_decode.hip (device code only).
//
// Operand registers: lane l of A holds row l % 16 and the eight consecutive k of group l / 16; B the same with columns.
// D: lane l holds column l % 16 and rows 4 * (l / 16) + i, i = 0..3.  All accumulation is fp32.
//
// An fp32 operand (a rank vector, a hidden activation) enters as two bf16 terms hi + lo = x (1 + e), |e| <= 2^-17: one
// rounded bf16 term alone would add an error as large as the final rounding of a bf16 result, and these kernels are bound
// by memory, so the second matrix instruction is free.  fp16 operands that meet such a pair are split the same way (11 bits
// fit two bf16 terms exactly), which keeps bf16's exponent range for products of small gradients; the lo * lo term
// (2^-17 of a product) is left out.  Non-finite values split as hi = x, lo = 0: a sum with one stays non-finite, but an Inf may meet the
// other operand's zero or opposite second term and become NaN.
#pragma once
#include <hip/hip_runtime.h>

#include "device_utils.h"

namespace te {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The matrix instructions ignore the lane mask, so what loops and branches around them depend on is made scalar, the wave's own
// number first.  And no branch skips one matrix instruction between others: where the skipped part writes other registers, this
// compiler (ROCm 7.2) counts the wait states of the joining block's reads along the long path only, and the short path reads a
// result before it is there.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <typename E>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma16<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma16<f16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ void split1(float v, __bf16 &hi, __bf16 &lo) {
  hi = static_cast<__bf16>(v);
  const float h = static_cast<float>(hi);
  lo = static_cast<__bf16>(__builtin_isfinite(h) ? v - h : 0.f);
}
__device__ __forceinline__ uint16_t bits16(__bf16 v) { return __builtin_bit_cast(uint16_t, v); }

// eight stored values as bf16 terms: the values themselves, or fp16 split in two
template <typename E>
struct Terms;
template <>
struct Terms<bf16_t> {
  static constexpr bool kTwo = false;
  u32x4 hi;
  __device__ __forceinline__ explicit Terms(u32x4 v) : hi(v) {}
};
template <>
struct Terms<f16_t> {
  static constexpr bool kTwo = true;
  u32x4 hi, lo;
  __device__ __forceinline__ explicit Terms(u32x4 v) {
    const f16x8 f = __builtin_bit_cast(f16x8, v);
    bf16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __bf16 a, b;
      split1(static_cast<float>(f[i]), a, b);
      h[i] = a;
      l[i] = b;
    }
    hi = __builtin_bit_cast(u32x4, h);
    lo = __builtin_bit_cast(u32x4, l);
  }
};

// c + (stored) x (hi + lo); SWAP: c + (hi + lo) x (stored)
template <typename E, bool SWAP = false>
__device__ __forceinline__ f32x4 mfma16_split(const Terms<E> &w, u32x4 hi, u32x4 lo, f32x4 c) {
  if constexpr (SWAP) {
    c = mfma16<bf16_t>(lo, w.hi, c);
    if constexpr (Terms<E>::kTwo) c = mfma16<bf16_t>(hi, w.lo, c);
    return mfma16<bf16_t>(hi, w.hi, c);
  } else {
    c = mfma16<bf16_t>(w.hi, lo, c);
    if constexpr (Terms<E>::kTwo) c = mfma16<bf16_t>(w.lo, hi, c);
    return mfma16<bf16_t>(w.hi, hi, c);
  }
}

// Eight 16-bit elements at any element address: the hardware takes unaligned 16-byte global accesses, so neither odd row
// lengths nor shifted storage need kernels of their own.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ u32x4 load8(const uint16_t *p) { return *reinterpret_cast<const u32x4_any *>(p); }
// for what is read once per call: does not displace what other workgroups share in L2
__device__ __forceinline__ u32x4 load8_once(const uint16_t *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
}
__device__ __forceinline__ void store8(uint16_t *p, u32x4 v) { *reinterpret_cast<u32x4_any *>(p) = v; }
// The ends of rows whose length is no multiple of the step: a lane whose eight elements would reach past the end takes the last
// eight instead and, where they are summed, has the `skip` that its neighbour holds already set to zero (in one operand at
// least).  This keeps the kernels small (instruction cache misses cost these short kernels more than the arithmetic: an expand kernel
// with element-wise ends had 32 KiB of code and ran 18 us on 6 MB).
__device__ __forceinline__ u32x4 without_head(u32x4 v, int skip) {
#pragma unroll
  for (int w = 0; w < 4; ++w) v[w] &= skip <= 2 * w ? 0xFFFFFFFFu : skip <= 2 * w + 1 ? 0xFFFF0000u : 0u;
  return v;
}
// Rows of fewer elements than a step (kernel variants of their own, SMALL): the first n, zeros after.  p .. end belongs to one array, so
// away from its end one access and a mask do.
__device__ __forceinline__ u32x4 load8_any(const uint16_t *p, int n, const uint16_t *end) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (n > 0 && p + 8 <= end) {
    v = load8(p);
#pragma unroll
    for (int w = 0; w < 4; ++w) v[w] &= n > 2 * w + 1 ? 0xFFFFFFFFu : n > 2 * w ? 0xFFFFu : 0u;
  } else {
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int i = 0; i < min(n, 8); ++i) {
      const uint64_t x = p[i];
      if (i < 4) lo |= x << (16 * i);
      else hi |= x << (16 * (i - 4));
    }
    v = u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32)};
  }
  return v;
}

// r[i] = eight columns of row i; on return r[c] = rows 0 .. 7 of column c: one v_perm per register, since a lane owns the block
__device__ __forceinline__ void transpose8x8(u32x4 (&r)[8]) {
  u32x4 o[8];
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      o[2 * w][p] = perm(r[2 * p + 1][w], r[2 * p][w], 0x05040100u);
      o[2 * w + 1][p] = perm(r[2 * p + 1][w], r[2 * p][w], 0x07060302u);
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = o[i];
}

}  // namespace te
