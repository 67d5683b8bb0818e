// Global gradient norm over a list of tensors, and clipping (include/transformer_engine/amd_ext.h).
//
//   n = sqrt(sum_i sum_e g_i[e]^2),   out_i = g_i * min(1, max_norm / (n + eps))
//
// Squares are summed in 64 bits: fp32 squares overflow from |g| = 1.8e19 and vanish below 1e-23, and v_fma_f64 runs at 64
// lanes per clock and CU, ten times what HBM delivers in bf16.  One workgroup sums one chunk into its own slot, the slots are
// added in index order: no atomics, the same bits every time.
// Both passes stream at HBM rate.  A list larger than the 256 MiB memory-side cache is read past the caches (1 GiB of bf16: 157 + 399 us
// so, 207 + 378 us with plain loads); keeping its last 128 to 240 MiB for a second pass that walks backwards gave 571 to 579 us.  A smaller
// list is read plainly and found again (56 tensors of 128 KiB: 6.4 against 7.5 us for the second pass).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "common.h"
#include "device_utils.h"
#include "transformer_engine/amd_ext.h"

namespace te {
namespace {

constexpr int kThreads = 512;
constexpr int kTensors = 128;              // per launch: the table travels as a kernel argument (< 4 KiB)
constexpr int64_t kMinChunk = 16384;       // elements; a multiple of every vector width
constexpr int64_t kChunks = 2048;          // chunks of a large list (plus one ragged end per tensor)
constexpr size_t kCached = 256ull << 20;    // bytes of gradients that the caches keep between the passes
constexpr int64_t kDirect = 512;           // up to this many slots every clipping workgroup adds them itself

struct Table {
  const void *in[kTensors];
  void *out[kTensors];
  int64_t numel[kTensors];
  uint32_t first_chunk[kTensors + 1];
  uint8_t in_type[kTensors], out_type[kTensors];
  int count;
};

struct Chunk {
  int tensor;
  int64_t begin, len;
};

__device__ __forceinline__ Chunk locate(const Table &t, uint32_t chunk, int64_t chunk_size) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid; else hi = mid;
  }
  Chunk c;
  c.tensor = lo;
  c.begin = static_cast<int64_t>(chunk - t.first_chunk[lo]) * chunk_size;
  c.len = min(t.numel[lo] - c.begin, chunk_size);
  return c;
}

// sum over the workgroup, valid in every thread; every lane adds in the same order each time
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += part[w];
  return s;
}

template <bool ONCE, typename V>
__device__ __forceinline__ V load_vec(const V *p) {
  if constexpr (ONCE) return __builtin_bit_cast(V, ld_stream<u32x4>(p));
  else return *p;
}

template <bool ONCE, typename T>
__device__ __forceinline__ double square_sum(const T *p, int64_t len) {
  double s0 = 0, s1 = 0;
  constexpr int V = 16 / sizeof(T);
  const int64_t head = min(len, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T)));
  for (int64_t i = threadIdx.x; i < head; i += kThreads) {
    const double v = widen(p[i]);
    s0 = __builtin_fma(v, v, s0);
  }
  p += head;
  len -= head;
  const int64_t nvec = len / V;
  constexpr int U = 4;  // 64 bytes per lane in flight
  struct alignas(16) Vec { T e[V]; };
  auto add = [&](const Vec &v) {
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      const double a = widen(v.e[k]), b = widen(v.e[k + 1]);
      s0 = __builtin_fma(a, a, s0);
      s1 = __builtin_fma(b, b, s1);
    }
  };
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * kThreads < nvec; i += U * kThreads) {
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_vec<ONCE>(reinterpret_cast<const Vec *>(p) + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) add(v[u]);
  }
  for (; i < nvec; i += kThreads) add(reinterpret_cast<const Vec *>(p)[i]);
  for (int64_t k = nvec * V + threadIdx.x; k < len; k += kThreads) {
    const double v = widen(p[k]);
    s1 = __builtin_fma(v, v, s1);
  }
  return s0 + s1;
}

template <typename T>
__device__ __forceinline__ double chunk_sum(const Table &t, const Chunk &c, bool once) {
  const T *p = static_cast<const T *>(t.in[c.tensor]) + c.begin;
  return once ? square_sum<true>(p, c.len) : square_sum<false>(p, c.len);
}

__global__ __launch_bounds__(kThreads) void square_sum_kernel(Table t, int64_t chunk_size, double *slots, bool once) {
  const Chunk c = locate(t, blockIdx.x, chunk_size);
  double s;
  switch (t.in_type[c.tensor]) {
    case kNVTEBFloat16: s = chunk_sum<bf16_t>(t, c, once); break;
    case kNVTEFloat16: s = chunk_sum<f16_t>(t, c, once); break;
    default: s = chunk_sum<float>(t, c, once); break;
  }
  s = block_sum(s);
  if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

__device__ __forceinline__ double slots_sum(const double *slots, int64_t n) {
  double s = 0;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) s += slots[i];
  return block_sum(s);
}

__global__ __launch_bounds__(kThreads) void add_slots_kernel(const double *slots, int64_t n, double *sum, float *norm) {
  const double s = slots_sum(slots, n);
  if (threadIdx.x == 0) {
    if (sum != nullptr) *sum = s;
    if (norm != nullptr) *norm = static_cast<float>(sqrt(s));
  }
}

template <bool ONCE, typename I, typename O>
__device__ __forceinline__ void scale_chunk(const I *in, O *out, int64_t len, float c) {
  constexpr int V = 16 / sizeof(I);
  const int64_t head = min(len, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) % 16 / sizeof(I)));
  struct alignas(16) Vec { I e[V]; };
  struct alignas(sizeof(O) * V < 16 ? sizeof(O) * V : 16) Res { O e[V]; };
  int64_t done = 0;
  if (reinterpret_cast<uintptr_t>(out + head) % alignof(Res) == 0) {
    for (int64_t i = threadIdx.x; i < head; i += kThreads) narrow(widen(in[i]) * c, out[i]);
    const int64_t nvec = (len - head) / V;
    auto scaled = [&](const Vec &v) {
      Res r;
#pragma unroll
      for (int k = 0; k < V; ++k) narrow(widen(v.e[k]) * c, r.e[k]);
      return r;
    };
    const Vec *vi = reinterpret_cast<const Vec *>(in + head);
    Res *vo = reinterpret_cast<Res *>(out + head);
    constexpr int U = 4;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < nvec; i += U * kThreads) {
      Vec v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load_vec<ONCE>(vi + i + u * kThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) vo[i + u * kThreads] = scaled(v[u]);
    }
    for (; i < nvec; i += kThreads) vo[i] = scaled(vi[i]);
    done = head + nvec * V;
  }
  // the ragged end, or everything where input and output are aligned differently
  for (int64_t i = done + threadIdx.x; i < len; i += kThreads) narrow(widen(in[i]) * c, out[i]);
}

template <bool ONCE, typename I>
__device__ __forceinline__ void scale_to(const Table &t, const Chunk &k, float c) {
  const I *in = static_cast<const I *>(t.in[k.tensor]) + k.begin;
  switch (t.out_type[k.tensor]) {
    case kNVTEBFloat16: scale_chunk<ONCE>(in, static_cast<bf16_t *>(t.out[k.tensor]) + k.begin, k.len, c); break;
    case kNVTEFloat16: scale_chunk<ONCE>(in, static_cast<f16_t *>(t.out[k.tensor]) + k.begin, k.len, c); break;
    default: scale_chunk<ONCE>(in, static_cast<float *>(t.out[k.tensor]) + k.begin, k.len, c); break;
  }
}

template <bool ONCE>
__global__ __launch_bounds__(kThreads) void clip_kernel(Table t, int64_t chunk_size, const double *slots, int64_t num_slots,
                                                        float max_norm, float eps, float *norm) {
  const double n = sqrt(slots_sum(slots, num_slots));
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm != nullptr) *norm = static_cast<float>(n);
  const double f = static_cast<double>(max_norm) / (n + static_cast<double>(eps));
  const float c = f > 1.0 ? 1.f : static_cast<float>(f);  // NaN stays NaN
  const Chunk k = locate(t, blockIdx.x, chunk_size);
  if (c == 1.f && t.in[k.tensor] == t.out[k.tensor]) return;  // in place and nothing to change
  switch (t.in_type[k.tensor]) {
    case kNVTEBFloat16: scale_to<ONCE, bf16_t>(t, k, c); break;
    case kNVTEFloat16: scale_to<ONCE, f16_t>(t, k, c); break;
    default: scale_to<ONCE, float>(t, k, c); break;
  }
}

// ------------------------------------------------------------------------------------------------ host
struct List {
  const void *const *in;
  void *const *out;  // null: no outputs
  const size_t *numel;
  const int *in_type, *out_type;
  size_t n;
};

int64_t chunk_size_of(const size_t *numel, size_t n) {
  uint64_t total = 0;
  for (size_t i = 0; i < n; ++i) total += numel[i];
  const int64_t c = static_cast<int64_t>(ceil_div(ceil_div(total, static_cast<size_t>(kChunks)), static_cast<size_t>(kMinChunk)));
  return std::max<int64_t>(1, c) * kMinChunk;
}

int64_t num_chunks(const size_t *numel, size_t n, int64_t chunk) {
  int64_t c = 0;
  for (size_t i = 0; i < n; ++i) c += static_cast<int64_t>(ceil_div(numel[i], static_cast<size_t>(chunk)));
  return c;
}

void check_list(const List &l, bool clips) {
  NVTE_CHECK(l.n == 0 || (l.in && l.numel && l.in_type), "a list of the gradients is NULL");
  NVTE_CHECK(l.n == 0 || !clips || (l.out && l.out_type), "outs or out_dtypes is NULL");
  for (size_t i = 0; i < l.n; ++i) {
    NVTE_CHECK(is_high_precision(static_cast<DType>(l.in_type[i])), "gradient ", i, " has dtype=",
               dtype_name(static_cast<DType>(l.in_type[i])), ", but expected float32, float16 or bfloat16");
    NVTE_CHECK(l.numel[i] == 0 || l.in[i] != nullptr, "gradient ", i, " has no data");
    const size_t align = dtype_bits(static_cast<DType>(l.in_type[i])) / 8;
    NVTE_CHECK(reinterpret_cast<uintptr_t>(l.in[i]) % align == 0, "gradient ", i, " is not aligned to its element");
    if (l.out == nullptr) continue;
    NVTE_CHECK(is_high_precision(static_cast<DType>(l.out_type[i])), "output ", i, " has dtype=",
               dtype_name(static_cast<DType>(l.out_type[i])), ", but expected float32, float16 or bfloat16");
    NVTE_CHECK(l.numel[i] == 0 || l.out[i] != nullptr, "output ", i, " has no data");
    const size_t oalign = dtype_bits(static_cast<DType>(l.out_type[i])) / 8;
    NVTE_CHECK(reinterpret_cast<uintptr_t>(l.out[i]) % oalign == 0, "output ", i, " is not aligned to its element");
    NVTE_CHECK(l.in[i] != l.out[i] || l.in_type[i] == l.out_type[i], "output ", i,
               " shares its gradient's memory but not its dtype");
  }
  if (l.out == nullptr) return;
  // an output may be its own gradient; any other overlap would be read or written by two workgroups at once
  struct Span {
    uintptr_t begin, end;
    bool out;
  };
  std::vector<Span> spans;
  spans.reserve(2 * l.n);
  for (size_t i = 0; i < l.n; ++i) {
    if (l.numel[i] == 0) continue;
    const uintptr_t o = reinterpret_cast<uintptr_t>(l.out[i]), g = reinterpret_cast<uintptr_t>(l.in[i]);
    spans.push_back({o, o + l.numel[i] * dtype_bits(static_cast<DType>(l.out_type[i])) / 8, true});
    if (g != o) spans.push_back({g, g + l.numel[i] * dtype_bits(static_cast<DType>(l.in_type[i])) / 8, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
  uintptr_t any_end = 0, out_end = 0;
  for (const Span &s : spans) {
    NVTE_CHECK(s.begin >= out_end && (!s.out || s.begin >= any_end),
               "an output overlaps another tensor of the call (an output may only be its own gradient)");
    any_end = std::max(any_end, s.end);
    if (s.out) out_end = std::max(out_end, s.end);
  }
}

template <typename Launch>
void for_tables(const List &l, int64_t chunk, Launch &&launch) {
  Table t;
  std::memset(&t, 0, sizeof(t));
  uint64_t chunks = 0, base = 0;
  auto flush = [&] {
    if (t.count == 0) return;
    t.first_chunk[t.count] = static_cast<uint32_t>(chunks);
    launch(t, static_cast<unsigned>(chunks), base);
    base += chunks;
    std::memset(&t, 0, sizeof(t));
    chunks = 0;
  };
  for (size_t i = 0; i < l.n; ++i) {
    if (l.numel[i] == 0) continue;
    t.in[t.count] = l.in[i];
    t.out[t.count] = l.out != nullptr ? l.out[i] : nullptr;
    t.numel[t.count] = static_cast<int64_t>(l.numel[i]);
    t.in_type[t.count] = static_cast<uint8_t>(l.in_type[i]);
    t.out_type[t.count] = static_cast<uint8_t>(l.out != nullptr ? l.out_type[i] : 0);
    t.first_chunk[t.count] = static_cast<uint32_t>(chunks);
    chunks += ceil_div(l.numel[i], static_cast<size_t>(chunk));
    if (++t.count == kTensors) flush();
  }
  flush();
}

bool read_once(const List &l) {
  size_t bytes = 0;
  for (size_t i = 0; i < l.n; ++i) bytes += l.numel[i] * (dtype_bits(static_cast<DType>(l.in_type[i])) / 8);
  return bytes > kCached;
}

void sum_squares(const List &l, int64_t chunk, double *slots, hipStream_t stream) {
  const bool once = read_once(l);
  for_tables(l, chunk, [&](const Table &t, unsigned grid, uint64_t base) {
    hipLaunchKernelGGL(square_sum_kernel, dim3(grid), dim3(kThreads), 0, stream, t, chunk, slots + base, once);
    NVTE_CHECK_HIP(hipGetLastError());
  });
}

void add_slots(const double *slots, int64_t n, double *sum, float *norm, hipStream_t stream) {
  hipLaunchKernelGGL(add_slots_kernel, dim3(1), dim3(kThreads), 0, stream, slots, n, sum, norm);
  NVTE_CHECK_HIP(hipGetLastError());
}

void clip(const List &l, int64_t chunk, const double *slots, int64_t num_slots, float max_norm, float eps, float *norm,
          hipStream_t stream) {
  bool any = false;
  const bool once = read_once(l);
  for_tables(l, chunk, [&](const Table &t, unsigned grid, uint64_t) {
    const auto kernel = once ? clip_kernel<true> : clip_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, stream, t, chunk, slots, num_slots, max_norm, eps, any ? nullptr : norm);
    NVTE_CHECK_HIP(hipGetLastError());
    any = true;
  });
  if (!any && norm != nullptr) add_slots(slots, num_slots, nullptr, norm, stream);  // nothing but empty tensors
}

void check_aligned(const char *what, const void *p, size_t align) {
  NVTE_CHECK(reinterpret_cast<uintptr_t>(p) % align == 0, what, " must be ", align, "-byte aligned");
}

void check_clip(float max_norm, float eps) {
  NVTE_CHECK(max_norm >= 0.f, "max_norm must not be negative or NaN, got ", max_norm);
  NVTE_CHECK(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
}

}  // namespace
}  // namespace te

using namespace te;

extern "C" {

size_t nvte_amd_grad_norm_workspace_size(const size_t *numels, size_t num_tensors) {
  return api_guard("nvte_amd_grad_norm_workspace_size", [&]() -> size_t {
    NVTE_CHECK(num_tensors == 0 || numels != nullptr, "numels is NULL");
    return static_cast<size_t>(num_chunks(numels, num_tensors, chunk_size_of(numels, num_tensors)) + 1) * sizeof(double);
  });
}

void nvte_amd_grad_norm(const void *const *grads, const size_t *numels, const int *dtypes, size_t num_tensors,
                        double *sum_of_squares, float *norm, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  api_guard("nvte_amd_grad_norm", [&] {
    const List l{grads, nullptr, numels, dtypes, nullptr, num_tensors};
    check_list(l, false);
    check_aligned("the workspace", workspace, sizeof(double));
    check_aligned("sum_of_squares", sum_of_squares, sizeof(double));
    check_aligned("norm", norm, sizeof(float));
    const int64_t chunk = chunk_size_of(numels, num_tensors), slots = num_chunks(numels, num_tensors, chunk);
    NVTE_CHECK(workspace != nullptr && workspace_bytes >= static_cast<size_t>(slots + 1) * sizeof(double),
               "workspace of ", workspace_bytes, " bytes, but ", (slots + 1) * sizeof(double), " are needed");
    double *w = static_cast<double *>(workspace);
    sum_squares(l, chunk, w, stream);
    add_slots(w, slots, sum_of_squares, norm, stream);
  });
}

void nvte_amd_clip_grad_norm(const void *const *grads, void *const *outs, const size_t *numels, const int *dtypes,
                             const int *out_dtypes, size_t num_tensors, float max_norm, float eps, float *norm,
                             void *workspace, size_t workspace_bytes, hipStream_t stream) {
  api_guard("nvte_amd_clip_grad_norm", [&] {
    const List l{grads, outs, numels, dtypes, out_dtypes, num_tensors};
    check_list(l, true);
    check_clip(max_norm, eps);
    check_aligned("the workspace", workspace, sizeof(double));
    check_aligned("norm", norm, sizeof(float));
    const int64_t chunk = chunk_size_of(numels, num_tensors), slots = num_chunks(numels, num_tensors, chunk);
    NVTE_CHECK(workspace != nullptr && workspace_bytes >= static_cast<size_t>(slots + 1) * sizeof(double),
               "workspace of ", workspace_bytes, " bytes, but ", (slots + 1) * sizeof(double), " are needed");
    double *w = static_cast<double *>(workspace);
    sum_squares(l, chunk, w, stream);
    if (slots <= kDirect) {
      clip(l, chunk, w, slots, max_norm, eps, norm, stream);
    } else {
      add_slots(w, slots, w + slots, nullptr, stream);
      clip(l, chunk, w + slots, 1, max_norm, eps, norm, stream);
    }
  });
}

void nvte_amd_clip_by_sum_of_squares(const void *const *grads, void *const *outs, const size_t *numels, const int *dtypes,
                                     const int *out_dtypes, size_t num_tensors, const double *sum_of_squares, float max_norm,
                                     float eps, float *norm, hipStream_t stream) {
  api_guard("nvte_amd_clip_by_sum_of_squares", [&] {
    const List l{grads, outs, numels, dtypes, out_dtypes, num_tensors};
    check_list(l, true);
    NVTE_CHECK(sum_of_squares != nullptr, "sum_of_squares is NULL");
    check_clip(max_norm, eps);
    check_aligned("sum_of_squares", sum_of_squares, sizeof(double));
    check_aligned("norm", norm, sizeof(float));
    clip(l, chunk_size_of(numels, num_tensors), sum_of_squares, 1, max_norm, eps, norm, stream);
  });
}

}  // extern "C"
