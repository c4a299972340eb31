// The norm of all gradients of a model together, and clipping by it.
//
//   norm = (sum over tensors and elements |g|^p)^(1/p), p = 1, 2 or infinity
//   coef = min(1, max_norm / (norm + 1e-6)),  g = g * coef (fp32 product, rounded once)
//
// The tensors' addresses and sizes travel in the kernel's parameters (up to 1600 tensors a
// launch), so nothing is copied to the device and a captured launch keeps its own table. The
// tensors are cut into chunks of 32 KB; a fixed grid walks the chunks, each CTA adds
// its own in 64 bits and writes one partial sum, and whoever needs the norm adds the partials in
// order: the same bits on every run. 64-bit sums of 64-bit squares: no gradient's square
// overflows or is lost, and HBM still bounds it (two 64-bit operations for each 2 or 4 bytes).
//
// Clipping reads the gradients a second time, from the last chunk to the first: what the norm's
// pass read last still sits in L2 (646 MB of fp32: 301 us, 311 us from the first chunk on), and
// with streaming loads and stores, since nothing of it is read again (306 us with plain ones).
// With a norm within the limit it reads and writes nothing. HBM bounds all of it: the norm reads
// 6.7 TB/s (96 us), norm and scaling together move 6.4 TB/s; a copy's measured rate is 6.54. Small
// sets are bound by the two launches and, with hundreds of tensors, by reading the table out of
// constant memory: 3 us for one tensor of 8192 elements, 16 us for 336 tensors of 35 MB.
#include <algorithm>
#include <vector>

#include "objective.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 32 * 1024;   // eight 16-byte vectors a thread
__host__ __device__ constexpr int64_t chunk_of(int e) { return kChunkBytes / e; }   // elements
// Of the scaling: vectors a thread has in flight. Eight need 127 registers for the 16-bit types
// (two CTAs an SM) and win 1 % at 646 MB, four win 15 % at 35 MB.
constexpr int kScaleVectors = 4;
// Tensors per launch. The large table stays under the 32 KB that parameters may take; filling and
// passing it costs the host 2 us a launch whatever it holds (one tensor: 18.8 us a call against
// 16.6 with the small one, 96 tensors 47.5 against 44.8; on the device 3.2 us against 3.0): 13 % of
// the smallest call, 6 % at 96 tensors, where the tensors themselves begin to cost more.
constexpr int kMaxTensors = 1600;
constexpr int kFewTensors = 96;
constexpr int kMaxGrid = 592;            // of the norm: 4 CTAs of 256 threads on each of 148 SMs
constexpr int kClipGrid = 2368;          // of the scaling: 16 on each, 4 of them at once

template <int K>
struct Table {
  void* ptr[K];
  int64_t size[K];                       // elements << 2 | dtype tag
  int32_t first[K];                      // the tensor's first chunk in this launch
  int32_t n, chunks;
};

struct Part {
  void* p;        // the chunk's first element
  int len, dtype;
};

template <int K>
__device__ __forceinline__ Part part_of(const Table<K>& t, int chunk) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {                      // the last tensor whose first chunk is <= chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  const int64_t size = t.size[lo] >> 2;
  const int dtype = static_cast<int>(t.size[lo] & 3);
  const int e = dtype == QB_F32 ? 4 : 2;
  const int64_t start = int64_t(chunk - t.first[lo]) * chunk_of(e);
  const int64_t left = size - start;
  return {static_cast<char*>(t.ptr[lo]) + start * e,
          static_cast<int>(left < chunk_of(e) ? left : chunk_of(e)), dtype};
}

// What a thread gathers of one norm: sum x^2 or sum |x| in 64 bits, or max |x| (a NaN stays).
template <int P> struct Sum {
  using type = double;
};
template <> struct Sum<0> {
  using type = float;
};
template <int P>
__device__ __forceinline__ void take(typename Sum<P>::type& acc, float x) {
  if constexpr (P == 2) acc = fma(static_cast<double>(x), static_cast<double>(x), acc);
  else if constexpr (P == 1) acc += static_cast<double>(fabsf(x));
  else asm("max.NaN.f32 %0, %1, %2;" : "=f"(acc) : "f"(acc), "f"(fabsf(x)));
}

template <int P>
__device__ __forceinline__ double join(double a, double b) {
  if (P != 0) return a + b;
  return a != a || b != b ? NAN : fmax(a, b);
}

template <int P>
__device__ __forceinline__ double block_join(double v, double* scratch) {
  if constexpr (P != 0) {
    return qb::block_sum64(v, scratch);
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) v = join<P>(v, scratch[w]);
    return v;
  }
}

template <typename T>
__device__ __forceinline__ int head_of(const T* p, int len) {
  const int past = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
  return min(len, ((16 - past) & 15) / static_cast<int>(sizeof(T)));
}

template <typename T, int P>
__device__ __forceinline__ void norm_part(typename Sum<P>::type& acc, const T* p, int len) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int U = kChunkBytes / 16 / kThreads;
  const int head = head_of(p, len), nvec = (len - head) / VE;
  qb::Vec16<T> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = threadIdx.x + u * kThreads;
    x[u].u = v < nvec ? *reinterpret_cast<const uint4*>(p + head + v * VE) : uint4{0, 0, 0, 0};
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < VE; ++e) take<P>(acc, qb::to_f(x[u].v[e]));
  for (int j = threadIdx.x; j < len - nvec * VE; j += kThreads)
    take<P>(acc, qb::to_f(p[j < head ? j : nvec * VE + j]));
}

template <int K, int P>
__global__ void __launch_bounds__(kThreads)
grad_norm_kernel(const __grid_constant__ Table<K> table, double* __restrict__ partials) {
  qb::release_next();
  __shared__ double scratch[32];
  typename Sum<P>::type acc = 0;
  for (int c = blockIdx.x; c < table.chunks; c += gridDim.x) {
    const Part part = part_of(table, c);
    if (part.dtype == QB_F32)
      norm_part<float, P>(acc, static_cast<const float*>(part.p), part.len);
    else if (part.dtype == QB_F16)
      norm_part<__half, P>(acc, static_cast<const __half*>(part.p), part.len);
    else
      norm_part<__nv_bfloat16, P>(acc, static_cast<const __nv_bfloat16*>(part.p), part.len);
  }
  const double all = block_join<P>(acc, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = all;
}

// The norm from the partials, the same in every thread of every CTA.
__device__ double total_norm(const double* partials, int n, int p, double* scratch) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    acc = p == 0 ? join<0>(acc, partials[i]) : acc + partials[i];
  acc = p == 0 ? block_join<0>(acc, scratch) : qb::block_sum64(acc, scratch);
  return p == 2 ? sqrt(acc) : acc;
}

__global__ void __launch_bounds__(kThreads)
grad_norm_total_kernel(const double* partials, int n, int p, float* __restrict__ norm) {
  qb::await_previous();
  __shared__ double scratch[32];
  const double v = total_norm(partials, n, p, scratch);
  if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

template <typename T>
__device__ __forceinline__ void scale_part(T* p, int len, float coef) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int U = kScaleVectors;
  const int head = head_of(p, len), nvec = (len - head) / VE;
#pragma unroll 1
  for (int v0 = threadIdx.x; v0 < nvec; v0 += U * kThreads) {
    qb::Vec16<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * kThreads;
      if (v < nvec) x[u].u = __ldcs(reinterpret_cast<const uint4*>(p + head + v * VE));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * kThreads;
      if (v < nvec) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[u].v[e] = qb::from_f<T>(qb::to_f(x[u].v[e]) * coef);
        __stcs(reinterpret_cast<uint4*>(p + head + v * VE), x[u].u);
      }
    }
  }
  for (int j = threadIdx.x; j < len - nvec * VE; j += kThreads) {
    T* q = p + (j < head ? j : nvec * VE + j);
    *q = qb::from_f<T>(qb::to_f(*q) * coef);
  }
}

template <int K>
__global__ void __launch_bounds__(kThreads)
grad_clip_kernel(const __grid_constant__ Table<K> table, const double* partials, int n, int p,
                 double max_norm, float* __restrict__ norm) {
  qb::await_previous();
  __shared__ double scratch[32];
  const double v = total_norm(partials, n, p, scratch);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(v);
  const double ratio = max_norm / (v + 1e-6);
  if (ratio >= 1.0) return;              // within the limit (a NaN goes on and spreads)
  const float coef = static_cast<float>(ratio);
  for (int c = table.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const Part part = part_of(table, c);
    if (part.dtype == QB_F32) scale_part(static_cast<float*>(part.p), part.len, coef);
    else if (part.dtype == QB_F16) scale_part(static_cast<__half*>(part.p), part.len, coef);
    else scale_part(static_cast<__nv_bfloat16*>(part.p), part.len, coef);
  }
}

struct Args {
  const uint64_t* ptrs;
  const int64_t* sizes;
  const uint8_t* dtypes;
  int64_t n;
};

int check(const char* what, const Args& a) {
  if (a.n < 0 || (a.n > 0 && (!a.ptrs || !a.sizes || !a.dtypes)))
    return qb::fail(QB_ERR_INVALID, "%s: null pointer", what);
  for (int64_t i = 0; i < a.n; ++i) {
    const int e = qb::elem_size(a.dtypes[i]);
    if (e == 0) return qb::fail(QB_ERR_INVALID, "%s: unsupported dtype %d", what, a.dtypes[i]);
    if (a.sizes[i] < 0 || a.sizes[i] > (int64_t(1) << 40))
      return qb::fail(QB_ERR_INVALID, "%s: bad size", what);
    if (a.sizes[i] > 0 && (!a.ptrs[i] || a.ptrs[i] % e))
      return qb::fail(QB_ERR_INVALID, "%s: null or misaligned tensor %lld", what, (long long)i);
  }
  return QB_OK;
}

// Two tensors that share memory: their elements would count twice, and be scaled by two CTAs at
// once.
int check_overlap(const char* what, const Args& a) {
  std::vector<std::pair<uint64_t, uint64_t>> spans;
  spans.reserve(a.n);
  bool sorted = true;
  for (int64_t i = 0; i < a.n; ++i) {
    if (a.sizes[i] == 0) continue;
    const uint64_t end = a.ptrs[i] + a.sizes[i] * qb::elem_size(a.dtypes[i]);
    sorted = sorted && (spans.empty() || spans.back().first <= a.ptrs[i]);
    spans.emplace_back(a.ptrs[i], end);
  }
  if (!sorted) std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second)
      return qb::fail(QB_ERR_INVALID, "%s: two gradients share memory", what);
  return QB_OK;
}

// Calls launch(table, grid of at most `most` CTAs) for the tensors from *at on that fit one table,
// and moves *at past them.
template <int K, typename F>
int launch_table(const Args& a, int64_t* at, int most, F&& launch) {
  Table<K> t;
  t.n = 0;
  int64_t chunks = 0;
  for (; *at < a.n && t.n < K; ++*at) {
    const int64_t size = a.sizes[*at];
    if (size == 0) continue;
    const int64_t chunk = chunk_of(qb::elem_size(a.dtypes[*at])), c = (size + chunk - 1) / chunk;
    if (chunks + c > 0x7fff0000) break;           // more than 1.7e13 elements: the next launch's
    t.ptr[t.n] = reinterpret_cast<void*>(a.ptrs[*at]);
    t.size[t.n] = size << 2 | a.dtypes[*at];
    t.first[t.n] = static_cast<int32_t>(chunks);
    chunks += c;
    ++t.n;
  }
  t.chunks = static_cast<int32_t>(chunks);
  if (t.n == 0) return QB_OK;
  return launch(t, static_cast<int>(std::min<int64_t>(chunks, most)));
}

template <typename F>
int launch_all(const Args& a, int most, F&& launch) {
  for (int64_t at = 0; at < a.n;) {
    const int64_t left = a.n - at;
    const int rc = left <= kFewTensors ? launch_table<kFewTensors>(a, &at, most, launch)
                                       : launch_table<kMaxTensors>(a, &at, most, launch);
    if (rc) return rc;
  }
  return QB_OK;
}

int norm_partials(const Args& a, int p, double* partials, int64_t capacity, int64_t* used,
                  cudaStream_t stream) {
  *used = 0;
  return launch_all(a, kMaxGrid, [&](const auto& t, int grid) {
    if (*used + grid > capacity)
      return qb::fail(QB_ERR_INVALID, "grad_norm: workspace of %lld sums is too small",
                      (long long)capacity);
    double* out = partials + *used;
    *used += grid;
    using Tab = std::decay_t<decltype(t)>;
    constexpr int K = sizeof(Tab::size) / sizeof(int64_t);
    if (p == 2) grad_norm_kernel<K, 2><<<grid, kThreads, 0, stream>>>(t, out);
    else if (p == 1) grad_norm_kernel<K, 1><<<grid, kThreads, 0, stream>>>(t, out);
    else grad_norm_kernel<K, 0><<<grid, kThreads, 0, stream>>>(t, out);
    return qb::check_launch("grad_norm");
  });
}

int check_norm(const char* what, const Args& a, int p, const void* workspace, const void* norm) {
  if (int rc = check(what, a)) return rc;
  if (p < 0 || p > 2)
    return qb::fail(QB_ERR_INVALID, "%s: norm of order 1, 2 or 0 (infinity)", what);
  if (!workspace || !norm) return qb::fail(QB_ERR_INVALID, "%s: null pointer", what);
  return QB_OK;
}

}  // namespace

extern "C" int64_t qb_grad_norm_workspace(int64_t n_tensors) {
  if (n_tensors < 0) return 0;
  return (n_tensors / kMaxTensors + 2) * kMaxGrid;
}

extern "C" int qb_grad_norm(const uint64_t* ptrs, const int64_t* sizes, const uint8_t* dtypes,
                            int64_t n_tensors, int order, double* workspace,
                            int64_t workspace_doubles, float* norm, cudaStream_t stream) {
  const Args a{ptrs, sizes, dtypes, n_tensors};
  if (int rc = check_norm("grad_norm", a, order, workspace, norm)) return rc;
  int64_t used = 0;
  if (int rc = norm_partials(a, order, workspace, workspace_doubles, &used, stream)) return rc;
  qb::launch_after(grad_norm_total_kernel, 1, kThreads, stream, workspace, static_cast<int>(used),
                   order, norm);
  return qb::check_launch("grad_norm");
}

extern "C" int qb_grad_clip(const uint64_t* ptrs, const int64_t* sizes, const uint8_t* dtypes,
                            int64_t n_tensors, int order, const double* max_norm,
                            double* workspace, int64_t workspace_doubles, float* norm,
                            cudaStream_t stream) {
  const Args a{ptrs, sizes, dtypes, n_tensors};
  if (int rc = check_norm("grad_clip", a, order, workspace, norm)) return rc;
  if (!max_norm || !(*max_norm >= 0))
    return qb::fail(QB_ERR_INVALID, "grad_clip: max_norm must be a number of at least 0");
  try {
    if (int rc = check_overlap("grad_clip", a)) return rc;
  } catch (...) {
    return qb::fail(QB_ERR_INVALID, "grad_clip: out of host memory");
  }
  int64_t used = 0;
  if (int rc = norm_partials(a, order, workspace, workspace_doubles, &used, stream)) return rc;
  if (used == 0) return qb_grad_norm(ptrs, sizes, dtypes, 0, order, workspace, workspace_doubles,
                                     norm, stream);
  const double limit = *max_norm;
  float* out = norm;                     // the first launch writes it
  return launch_all(a, kClipGrid, [&](const auto& t, int grid) {
    using Tab = std::decay_t<decltype(t)>;
    constexpr int K = sizeof(Tab::size) / sizeof(int64_t);
    // directly behind the last norm launch; a further table's launch waits for the one before
    if (out)
      qb::launch_after(grad_clip_kernel<K>, grid, kThreads, stream, t, workspace,
                       static_cast<int>(used), order, limit, out);
    else
      grad_clip_kernel<K><<<grid, kThreads, 0, stream>>>(t, workspace, static_cast<int>(used),
                                                         order, limit, out);
    out = nullptr;
    return qb::check_launch("grad_clip");
  });
}
