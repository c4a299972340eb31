// Preference loss over pairs of sequences (paired log ratios), forward and backward.
//
//   s_i = sum_t mask_it (logp_it - ref_it)   [/ max(n_i, 1)]   [- ref_i]
//   D_k = s_k - s_{P+k}      (rows 0 .. P-1 preferred, P .. 2P-1 rejected)     u = beta D - margin
//   sigmoid  (1 - eps) softplus(-u) + eps softplus(u)      hinge  max(0, 1 - u)
//   ipo      (D - 1 / (2 beta))^2                          loss = sum_k L_k / denominator
//   dlogp_it = mask_it * (+ | -) L'(D_k) / denominator [/ max(n_i, 1)]
//
// A difference of two long sums: terms and sums are 64-bit, so what the pair differs by is not
// lost in them. Masked places are skipped, not multiplied by zero: whatever they hold (a NaN of a
// padded position) does not count. Reads 4 + 4 + 1 bytes a token, writes 4: at the sizes of a
// batch latency bounds it (forward 4.5 us for 8 x 512 tokens, 6.4 us for 62 x 16383, backward 1.6
// and 2.5 us), and before that the host, whose part of a loss and its gradient is about 112 us, 69
// of them an empty autograd function's.
#include "objective.cuh"

namespace {

using qb::kObjChunk;
using qb::kObjPerThread;
using qb::kObjThreads;

struct Record {
  double sum;
  int64_t count;
};

template <typename T>
__global__ void __launch_bounds__(kObjThreads)
preference_rows_kernel(const T* __restrict__ logp, const T* __restrict__ ref,
                       const uint8_t* __restrict__ mask, int64_t cols, int chunks,
                       Record* __restrict__ records) {
  qb::release_next();
  __shared__ double scratch[64];
  const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
  const int64_t c0 = int64_t(blockIdx.x % static_cast<unsigned>(chunks)) * kObjChunk + threadIdx.x;
  const int left = static_cast<int>(cols - c0 < kObjChunk ? cols - c0 : kObjChunk);
  logp += row * cols + c0;
  if (ref) ref += row * cols + c0;
  if (mask) mask += row * cols + c0;
  float a[kObjPerThread], b[kObjPerThread];
  bool on[kObjPerThread];
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k) {
    const int j = k * kObjThreads;
    on[k] = j < left && (!mask || mask[j]);
    a[k] = j < left ? qb::to_f(logp[j]) : 0.f;
    b[k] = ref && j < left ? qb::to_f(ref[j]) : 0.f;
  }
  double sum = 0.0;
  int count = 0;
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k) {
    if (on[k]) {
      sum += static_cast<double>(a[k]) - static_cast<double>(b[k]);
      ++count;
    }
  }
  const unsigned n = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(count));
  double both[2] = {sum, threadIdx.x % 32 == 0 ? static_cast<double>(n) : 0.0};
  qb::block_sums64<true>(both, scratch);
  if (threadIdx.x == 0) records[blockIdx.x] = Record{both[0], static_cast<int64_t>(both[1])};
}

// NaN in, NaN out: fabs keeps it, and log1p(exp()) carries it.
__device__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }
__device__ double sigmoid(double x) {
  const double e = exp(-fabs(x));
  return (x >= 0 ? 1.0 : e) / (1.0 + e);
}

// One CTA: a group of lanes per pair, the rows' records added in a fixed order.
__global__ void __launch_bounds__(1024)
preference_pairs_kernel(const Record* records, int chunks, int lanes, int64_t pairs,
                        const void* __restrict__ ref_row, bool ref_row_double,
                        qb_preference_config cfg, const double* __restrict__ denom_dev,
                        float* __restrict__ loss, float* __restrict__ rewards,
                        float* __restrict__ coef) {
  qb::await_previous();
  __shared__ double scratch[32];
  const double denom = denom_dev ? *denom_dev
                                 : cfg.denominator > 0 ? cfg.denominator : double(pairs);
  const int sub = threadIdx.x % lanes, group = threadIdx.x / lanes, groups = blockDim.x / lanes;
  double total = 0.0;
  for (int64_t p0 = 0; p0 < pairs; p0 += groups) {     // whole warps go round together
    const int64_t p = p0 + group;
    double s[2] = {0.0, 0.0}, n[2] = {0.0, 0.0};
    if (p < pairs) {
      for (int k = sub; k < chunks; k += lanes) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Record rec = records[(p + h * pairs) * chunks + k];
          s[h] += rec.sum;
          n[h] += static_cast<double>(rec.count);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = qb::group_sum64(s[h], lanes);
      n[h] = qb::group_sum64(n[h], lanes);
    }
    if (p >= pairs || sub != 0) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = p + h * pairs;
      n[h] = cfg.length_normalized ? fmax(n[h], 1.0) : 1.0;
      s[h] = s[h] / n[h] - (!ref_row ? 0.0
                            : ref_row_double ? static_cast<const double*>(ref_row)[row]
                                             : static_cast<const float*>(ref_row)[row]);
      rewards[row] = static_cast<float>(cfg.beta * s[h]);
    }
    const double d = s[0] - s[1], u = cfg.beta * d - cfg.margin;
    double slope;    // dL/dD
    if (cfg.loss_type == 0) {
      const double eps = cfg.label_smoothing;
      total += (1.0 - eps) * softplus(-u) + (eps > 0 ? eps * softplus(u) : 0.0);
      slope = cfg.beta * (eps * sigmoid(u) - (1.0 - eps) * sigmoid(-u));
    } else if (cfg.loss_type == 1) {
      total += u != u ? u : fmax(0.0, 1.0 - u);
      slope = u < 1.0 ? -cfg.beta : u != u ? u : 0.0;   // u may be +inf
    } else {
      const double off = d - 0.5 / cfg.beta;
      total += off * off;
      slope = 2.0 * off;
    }
    coef[p] = static_cast<float>(slope / (denom * n[0]));
    coef[p + pairs] = static_cast<float>(-slope / (denom * n[1]));
  }
  double all[1] = {total};
  qb::block_sums64<true>(all, scratch);
  if (threadIdx.x == 0) *loss = static_cast<float>(all[0] / denom);
}

template <typename T>
__global__ void __launch_bounds__(kObjThreads)
preference_bwd_kernel(const uint8_t* __restrict__ mask, const float* __restrict__ coef,
                      const float* __restrict__ g, int64_t cols, int chunks,
                      T* __restrict__ grad) {
  const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
  const int64_t c0 = int64_t(blockIdx.x % static_cast<unsigned>(chunks)) * kObjChunk + threadIdx.x;
  const int left = static_cast<int>(cols - c0 < kObjChunk ? cols - c0 : kObjChunk);
  grad += row * cols + c0;
  if (mask) mask += row * cols + c0;
  const T v = qb::from_f<T>(coef[row] * *g), zero = qb::from_f<T>(0.f);
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k) {
    const int j = k * kObjThreads;
    if (j < left) grad[j] = !mask || mask[j] ? v : zero;
  }
}

int check(const char* what, int64_t pairs, int64_t cols) {
  if (pairs <= 0 || cols <= 0)
    return qb::fail(QB_ERR_INVALID, "%s: bad shape (%lld pairs of %lld)", what, (long long)pairs,
                    (long long)cols);
  if (pairs > 0x3fffffff || (cols + kObjChunk - 1) / kObjChunk > 0x7fffffff / (2 * pairs))
    return qb::fail(QB_ERR_INVALID, "%s: too large", what);
  return QB_OK;
}

int chunks_of(int64_t cols) { return static_cast<int>((cols + kObjChunk - 1) / kObjChunk); }

}  // namespace

extern "C" int64_t qb_preference_config_size(void) { return sizeof(qb_preference_config); }

extern "C" int64_t qb_preference_workspace(int64_t pairs, int64_t cols) {
  if (check("preference", pairs, cols) != QB_OK) return 0;
  return 2 * pairs * chunks_of(cols) * static_cast<int64_t>(sizeof(Record));
}

extern "C" int qb_preference_fwd(const void* logp, const void* ref, int dtype,
                                 const uint8_t* mask, const void* ref_row, int ref_row_double,
                                 int64_t pairs, int64_t cols, const qb_preference_config* cfg,
                                 const double* denominator, float* loss, float* rewards,
                                 float* coef, void* workspace, cudaStream_t stream) {
  if (int rc = check("preference", pairs, cols)) return rc;
  if (!logp || !cfg || !loss || !rewards || !coef || !workspace)
    return qb::fail(QB_ERR_INVALID, "preference: null pointer");
  if (ref && ref_row) return qb::fail(QB_ERR_INVALID, "preference: two references");
  if (cfg->loss_type < 0 || cfg->loss_type > 2 || !(cfg->beta > 0) ||
      !(cfg->label_smoothing >= 0 && cfg->label_smoothing < 0.5) || cfg->margin != cfg->margin)
    return qb::fail(QB_ERR_INVALID, "preference: bad loss type, beta, label smoothing or margin");
  const int chunks = chunks_of(cols);
  auto* records = static_cast<Record*>(workspace);
  QB_DISPATCH_FLOAT(dtype, T, {
    preference_rows_kernel<T><<<static_cast<unsigned>(2 * pairs * chunks), kObjThreads, 0,
                                stream>>>(static_cast<const T*>(logp),
                                          static_cast<const T*>(ref), mask, cols, chunks, records);
  });
  if (int rc = qb::check_launch("preference")) return rc;
  const int lanes = qb::lanes_per_row(chunks);
  qb::launch_after(preference_pairs_kernel, 1, qb::adding_threads(pairs, lanes), stream, records,
                   chunks, lanes, pairs, ref_row, ref_row_double != 0, *cfg, denominator, loss,
                   rewards, coef);
  return qb::check_launch("preference");
}

extern "C" int qb_preference_bwd(const uint8_t* mask, const float* coef, const float* g,
                                 int64_t pairs, int64_t cols, void* grad, int dtype,
                                 cudaStream_t stream) {
  if (int rc = check("preference_bwd", pairs, cols)) return rc;
  if (!coef || !g || !grad) return qb::fail(QB_ERR_INVALID, "preference_bwd: null pointer");
  const int chunks = chunks_of(cols);
  QB_DISPATCH_FLOAT(dtype, T, {
    preference_bwd_kernel<T><<<static_cast<unsigned>(2 * pairs * chunks), kObjThreads, 0,
                               stream>>>(mask, coef, g, cols, chunks, static_cast<T*>(grad));
  });
  return qb::check_launch("preference_bwd");
}
