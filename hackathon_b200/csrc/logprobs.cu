// Log-probabilities of chosen tokens (and the entropy of each row's distribution) from rows of
// materialised logits, forward and backward.
//
// With temperature T, c = log2(e) / T and a row's maximum m:
//   y_j = (z_j - m) c,  e_j = 2^y_j,  s = sum e_j,  t = sum e_j y_j
//   logp = (z_label - m) / T - ln s          H = ln s - ln2 t / s
//   dz_j = (1/T) [ g (1{j = label} - p_j) - g_H p_j (ln p_j + H) ],  p_j = e_j / s
//        = e_j (A + B y_j) + (g / T) 1{j = label}
//   with A = -(g + g_H (H - ln s)) / (T s),  B = -g_H ln2 / (T s)
// Sums and maxima are fp32. The maximum is subtracted before the scale: z c - m c in one fused
// multiply-add would save an operation, but leaves the rounding of m c in every y, which grows with
// |m| / T, and makes a certain token's log-probability something near 0 instead of 0.
//
// A banned token (a logit of -inf, or so low that y is) has e = 0 and no e y term: y is held above
// kLowest, where 2^y is 0 and y stays finite. Rows need no other care: one of equal lowest values
// is the uniform distribution, one of -inf alone, with +inf or with NaN is NaN, as the formula is.
#include <cooperative_groups.h>

#include "qb_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr float kLowest = -1e5f;

__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Row r of the logits: [outer, inner, vocab] with element strides so, si.
struct Rows {
  int64_t inner, so, si;
  __device__ __forceinline__ int64_t offset(int64_t r) const {
    return (r / inner) * so + (r % inner) * si;
  }
};

// max, sum 2^(y), sum 2^(y) y of a set of elements, y relative to m.
struct Stat {
  float m, s, t;
};

// From one maximum to a larger one (from -inf, with s = t = 0, too).
__device__ __forceinline__ void rescale(Stat& a, float m, float c) {
  const float d = fmaxf((a.m - m) * c, kLowest);
  const float f = ex2(d);
  a.t = (a.t + a.s * d) * f;
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, c);
  rescale(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ Stat warp_merge(Stat st, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
               __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = merge(st, other, c);
  }
  return st;
}

template <typename T, bool ENT>
__device__ __forceinline__ void add(Stat& st, const float* z, int n, float c) {
  float m = z[0];
#pragma unroll
  for (int e = 1; e < n; ++e) m = max_nan(m, z[e]);
  if (m == -INFINITY) return;    // all banned: nothing to add, and no maximum to subtract
  if (m > st.m) rescale(st, m, c);
#pragma unroll
  for (int e = 0; e < n; ++e) {
    float y = (z[e] - st.m) * c;
    if (ENT) y = max_nan(y, kLowest);
    const float x = ex2(y);
    st.s += x;
    if (ENT) st.t += x * y;
  }
}

// One CTA per row, or a cluster of CTAs when there are few rows: each takes every CS-th vector
// block of the row, the cluster's first CTA merges.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const T* __restrict__ logits, Rows rows, int vocab,
                      const int64_t* __restrict__ target, float inv_t,
                      float* __restrict__ logp, float* __restrict__ entropy,
                      float2* __restrict__ stats) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int U = 4;
  __shared__ Stat warp_stat[32];
  __shared__ Stat cta_stat;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / cs;
  const T* z = logits + rows.offset(row);
  const float c = inv_t * kLog2e;
  const int tid = rank * kThreads + threadIdx.x, nthreads = cs * kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // scalars before the first 16-byte boundary and after the last, vectors between
  const int head = min(vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15)
                                               / sizeof(T)));
  const int nvec = (vocab - head) / VE;
  const T* body = z + head;

  auto cluster_merge = [&](Stat st) {
    st = warp_merge(st, c);
    if (lane == 0) warp_stat[warp] = st;
    __syncthreads();
    if (warp == 0) {
      st = lane < kThreads / 32 ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
      st = warp_merge(st, c);
      if (lane == 0) cta_stat = st;
    }
    if (cs == 1) {
      __syncthreads();
      return cta_stat;
    }
    cluster.sync();
    Stat all = *cluster.map_shared_rank(&cta_stat, 0);
    for (int k = 1; k < cs; ++k) all = merge(all, *cluster.map_shared_rank(&cta_stat, k), c);
    cluster.sync();            // nobody leaves, or writes again, while another still reads
    return all;
  };

  Stat st{-INFINITY, 0.f, 0.f};
  for (int v = tid; v < nvec; v += U * nthreads) {
    qb::Vec16<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * nthreads < nvec)
        x[u].u = __ldg(reinterpret_cast<const uint4*>(body + int64_t(v + u * nthreads) * VE));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v + u * nthreads < nvec) {
        float f[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = qb::to_f(x[u].v[e]);
        add<T, ENT>(st, f, VE, c);
      }
    }
  }
  for (int j = tid; j < vocab - nvec * VE; j += nthreads) {
    const int col = j < head ? j : nvec * VE + j;
    const float f = qb::to_f(z[col]);
    add<T, ENT>(st, &f, 1, c);
  }
  st = cluster_merge(st);
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t label = target[row];
    const float log_s = logf(st.s);
    float lp = 0.f;
    if (label >= 0 && label < vocab) lp = (qb::to_f(z[label]) - st.m) * inv_t - log_s;
    logp[row] = lp;
    if (ENT) entropy[row] = log_s - kLn2 * (st.t / st.s);
    stats[row] = make_float2(st.m, st.s);
  }
}

// ---------------------------------------------------------------------------------------------
// backward: elementwise given the row's (m, s, H); one CTA per (row, tile of columns)

constexpr int kBwdThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
token_logprobs_bwd_kernel(const T* __restrict__ logits, Rows rows, int vocab, int tiles,
                          const int64_t* __restrict__ target, float inv_t,
                          const float2* __restrict__ stats, const float* __restrict__ entropy,
                          const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                          T* __restrict__ dlogits) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int U = 4;
  const int64_t row = blockIdx.x / tiles;
  const int tile = blockIdx.x % tiles;
  const T* z = logits + rows.offset(row);
  T* dz = dlogits + row * vocab;
  const int64_t label = target[row];
  const bool labelled = label >= 0 && label < vocab;
  const float g = labelled && g_logp ? g_logp[row] : 0.f;
  const float gh = g_ent ? g_ent[row] : 0.f;
  const float2 ms = stats[row];
  const float c = inv_t * kLog2e, k = inv_t / ms.y;
  const float log_s = logf(ms.y);
  const float A = -(g + (g_ent ? gh * (entropy[row] - log_s) : 0.f)) * k;
  const float B = -gh * kLn2 * k;
  const float hot = g * inv_t;
  const bool zero = g == 0.f && gh == 0.f;   // e.g. a prompt's positions: nothing to read

  auto value = [&](float zf, int col) -> float {
    if (zero) return 0.f;
    const float y = max_nan((zf - ms.x) * c, kLowest);
    const float x = ex2(y);
    const float d = x * fmaf(B, y, A);
    return col == label && labelled ? d + hot : d;
  };

  const int head = min(vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dz) & 15)) & 15)
                                               / sizeof(T)));
  const int nvec = (vocab - head) / VE;
  const bool vec_in = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  const int v0 = tile * (kBwdThreads * U);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + u * kBwdThreads + threadIdx.x;
    if (v < nvec) {
      const int col = head + v * VE;
      float f[VE];
      if (!zero) {
        if (vec_in) {
          qb::load16<T>(z + col, f);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) f[e] = qb::to_f(z[col + e]);
        }
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = value(f[e], col + e);
      qb::store16<T>(dz + col, f);
    }
  }
  if (tile == 0) {
    for (int j = threadIdx.x; j < vocab - nvec * VE; j += kBwdThreads) {
      const int col = j < head ? j : nvec * VE + j;
      dz[col] = qb::from_f<T>(value(zero ? 0.f : qb::to_f(z[col]), col));
    }
  }
}

int check(const char* what, const void* logits, int64_t rows, int64_t inner, int64_t vocab,
          const int64_t* target, float temperature, const void* stats) {
  if (rows < 0 || vocab <= 0 || vocab > 0x3fffffff || inner <= 0 || rows % inner != 0)
    return qb::fail(QB_ERR_INVALID, "%s: bad shape (%lld rows of %lld, groups of %lld)", what,
                    (long long)rows, (long long)vocab, (long long)inner);
  if (!(temperature >= 1e-6f && temperature <= 1e6f))
    return qb::fail(QB_ERR_INVALID, "%s: temperature %g is not in 1e-6 .. 1e6", what,
                    (double)temperature);
  if (rows > 0 && (!logits || !target || !stats))
    return qb::fail(QB_ERR_INVALID, "%s: null pointer", what);
  return QB_OK;
}

}  // namespace

extern "C" int qb_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t inner,
                                 int64_t stride_outer, int64_t stride_inner, int64_t vocab,
                                 const int64_t* target, float temperature, float* logp,
                                 float* entropy, float* stats, cudaStream_t stream) {
  if (int rc = check("token_logprobs", logits, rows, inner, vocab, target, temperature, stats))
    return rc;
  if (rows == 0) return QB_OK;
  if (!logp) return qb::fail(QB_ERR_INVALID, "token_logprobs: null pointer");
  int cs = 1;
  while (cs < 8 && rows * cs < 296 && vocab / cs > 8 * kThreads) cs *= 2;
  if (rows * cs > 0x7fffffff) return qb::fail(QB_ERR_INVALID, "token_logprobs: too many rows");
  const Rows r{inner, stride_outer, stride_inner};
  const float inv_t = 1.f / temperature;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cs));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(cs), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  QB_DISPATCH_FLOAT(dtype, T, {
    auto* lp = static_cast<const T*>(logits);
    auto* st = reinterpret_cast<float2*>(stats);
    if (entropy)
      cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, lp, r, (int)vocab, target, inv_t,
                         logp, entropy, st);
    else
      cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, lp, r, (int)vocab, target, inv_t,
                         logp, entropy, st);
  });
  return qb::check_launch("token_logprobs");
}

extern "C" int qb_token_logprobs_bwd(const void* logits, int dtype, int64_t rows, int64_t inner,
                                     int64_t stride_outer, int64_t stride_inner, int64_t vocab,
                                     const int64_t* target, float temperature,
                                     const float* stats, const float* entropy,
                                     const float* g_logp, const float* g_entropy, void* dlogits,
                                     cudaStream_t stream) {
  if (int rc = check("token_logprobs_bwd", logits, rows, inner, vocab, target, temperature, stats))
    return rc;
  if (rows == 0) return QB_OK;
  if (!dlogits || (g_entropy && !entropy))
    return qb::fail(QB_ERR_INVALID, "token_logprobs_bwd: null pointer");
  const Rows r{inner, stride_outer, stride_inner};
  QB_DISPATCH_FLOAT(dtype, T, {
    constexpr int kTile = kBwdThreads * 4 * (16 / sizeof(T));
    const int64_t tiles = (vocab + kTile - 1) / kTile;
    if (rows * tiles > 0x7fffffff)
      return qb::fail(QB_ERR_INVALID, "token_logprobs_bwd: too many rows");
    token_logprobs_bwd_kernel<T><<<static_cast<unsigned>(rows * tiles), kBwdThreads, 0, stream>>>(
        static_cast<const T*>(logits), r, (int)vocab, (int)tiles, target, 1.f / temperature,
        reinterpret_cast<const float2*>(stats), entropy, g_logp, g_entropy,
        static_cast<T*>(dlogits));
  });
  return qb::check_launch("token_logprobs_bwd");
}
