// Clipped policy objective with a KL term over masked [rows, cols] log-probabilities, forward
// and backward.
//
//   l = logp - old,  r = e^l,  d = ref - logp,  k3 = e^d - d - 1
//   L = -min(min(r, delta) A, clamp(r, 1 - lo, 1 + hi) A) + kl k3
//   dL/dlogp = (-A r where the unclipped term is the smaller one, else 0) + kl (1 - e^d)
//   token:     sum mask L / denominator            (default: the number of unmasked tokens)
//   sequence:  sum_i (sum_t mask L / max(n_i, 1)) / denominator    (default: the rows)
//
// The gradient jumps where r crosses a border, so the side is that of the exact l against the
// border's logarithm B, not of a rounded r. Rounding keeps the order: the fp32 difference says
// which side it is wherever it is not B's own rounding, and there the 64-bit difference does. k3
// cancels for small d: below |d| = 1/2 it is summed as its Taylor series. The forward writes each
// token's dL/dlogp (fp32, unnormalised) when a gradient will be asked for; the backward multiplies
// it by g and the row's weight. Sums are 64-bit, in a fixed order. Masked places are skipped,
// whatever they hold.
//
// Latency bounds it at the sizes of a batch: forward 4.8 us for 16 x 333 tokens, 6.9 us for 8 x
// 32768, backward 1.4 and 1.7 us. 512 x 4096 tokens without a reference (27 MB with the gradient)
// take 13.9 us. The rows' launch executes 127 instructions a warp for 32 tokens, 7.4 us of the
// issue slots, which are 55 % busy: 64 registers allow four CTAs on an SM, so the 1024 CTAs go in
// 1.7 waves, and a CTA's loads, arithmetic and sums follow one another (16 columns a thread
// instead of 8 spill registers: 16 us). The total's launch adds its own latency. Backward 2.9 us
// (5.9 TB/s).
#include <cmath>

#include "objective.cuh"

namespace {

using qb::kObjChunk;
using qb::kObjPerThread;
using qb::kObjThreads;

// What the kernels take of qb_policy_config.
struct Params {
  double log_low, log_high, log_delta;   // the borders of r as logarithms
  float log_low32, log_high32, log_delta32;
  float low, high, delta, kl_coef;
  double denominator;
  bool sequence;
};

struct Record {
  double loss, kl;
  int32_t count, low, high, pad;
};

// e^d - 1 - d and e^d - 1, to the relative precision of fp32 also where they cancel.
__device__ __forceinline__ void kl_terms(float d, float& k3, float& em1) {
  if (fabsf(d) < 0.5f) {
    // sum_{n >= 2} d^n / n! to n = 10: the rest is below 2^-24 of the first
    float p = 1.f / 3628800.f;
    p = fmaf(p, d, 1.f / 362880.f);
    p = fmaf(p, d, 1.f / 40320.f);
    p = fmaf(p, d, 1.f / 5040.f);
    p = fmaf(p, d, 1.f / 720.f);
    p = fmaf(p, d, 1.f / 120.f);
    p = fmaf(p, d, 1.f / 24.f);
    p = fmaf(p, d, 1.f / 6.f);
    p = fmaf(p, d, 0.5f);
    k3 = p * d * d;
    em1 = fmaf(p * d, d, d);
  } else {
    em1 = expm1f(d);
    k3 = em1 - d;
  }
}

template <typename T>
__global__ void __launch_bounds__(kObjThreads)
policy_rows_kernel(const T* __restrict__ logp, const T* __restrict__ old,
                   const T* __restrict__ ref, const float* __restrict__ adv, int64_t adv_row,
                   int64_t adv_col, const uint8_t* __restrict__ mask, int64_t cols, int chunks,
                   Params par, Record* __restrict__ records,
                   float* __restrict__ unit) {
  qb::release_next();
  __shared__ double scratch[96];
  const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
  const int64_t c0 = int64_t(blockIdx.x % static_cast<unsigned>(chunks)) * kObjChunk + threadIdx.x;
  const int64_t at = row * cols + c0;
  const int left = static_cast<int>(cols - c0 < kObjChunk ? cols - c0 : kObjChunk);
  logp += at;
  old = old ? old + at : logp;           // the policy itself: l = 0
  if (ref) ref += at;
  if (mask) mask += at;
  if (unit) unit += at;
  adv += row * adv_row + c0 * adv_col;
  const float adv_one = adv_col == 0 ? *adv : 0.f;
  float lp[kObjPerThread], lo[kObjPerThread], lr[kObjPerThread], av[kObjPerThread];
  bool on[kObjPerThread];
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k) {
    const int j = k * kObjThreads;
    const bool in = j < left;
    on[k] = in && (!mask || mask[j]);
    lp[k] = in ? qb::to_f(logp[j]) : 0.f;
    lo[k] = in ? qb::to_f(old[j]) : 0.f;
    lr[k] = in && ref ? qb::to_f(ref[j]) : 0.f;
    av[k] = adv_col == 0 ? adv_one : in ? adv[j * adv_col] : 0.f;
  }
  double loss = 0.0, kl = 0.0;
  int count = 0, low = 0, high = 0;
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k) {
    float g = 0.f;
    if (on[k]) {
      const float l = lp[k] - lo[k], a = av[k];       // the 64-bit difference, rounded once
      bool below = l < par.log_low32, above = l > par.log_high32, past = l > par.log_delta32;
      if (l == par.log_low32 || l == par.log_high32 || l == par.log_delta32) {
        const double exact = static_cast<double>(lp[k]) - static_cast<double>(lo[k]);
        below = exact < par.log_low;
        above = exact > par.log_high;
        past = exact > par.log_delta;
      }
      const float r = expf(l);
      const float first = fminf(r, par.delta), held = fminf(fmaxf(r, par.low), par.high);
      float term = -fminf(first * a, held * a);
      if (r != r || a != a) term = r * a;
      const bool live = !past && (!(below || above) || (below && a > 0.f) || (above && a < 0.f));
      g = live ? -a * r : 0.f;
      if (ref) {
        float k3, em1;
        kl_terms(lr[k] - lp[k], k3, em1);
        if (par.kl_coef != 0.f) {          // 0 of an overflowed k3 is nothing
          term = fmaf(par.kl_coef, k3, term);
          g = fmaf(-par.kl_coef, em1, g);
        }
        kl += k3;
      }
      loss += term;
      ++count;
      low += below && a < 0.f;
      high += above && a > 0.f;
    }
    if (unit && k * kObjThreads < left) unit[k * kObjThreads] = g;
  }
  // the three counts of a warp (at most 2^8 each) in one integer, then of the chunk in one exact
  // double (at most 2^11 each)
  const unsigned counts = __reduce_add_sync(0xffffffffu, count + (low << 10) + (high << 20));
  const double packed = threadIdx.x % 32 == 0 ? (counts & 1023) + (counts >> 10 & 1023) * 65536.0
                                                    + (counts >> 20) * 4294967296.0 : 0.0;
  double sums[3] = {loss, kl, packed};
  if (ref) {
    qb::block_sums64<true>(sums, scratch);
  } else {
    double two[2] = {loss, packed};
    qb::block_sums64<true>(two, scratch);
    sums[0] = two[0], sums[2] = two[1];
  }
  if (threadIdx.x == 0) {
    const int64_t p = static_cast<int64_t>(sums[2]);
    records[blockIdx.x] = Record{sums[0], sums[1], static_cast<int32_t>(p & 0xffff),
                                 static_cast<int32_t>((p >> 16) & 0xffff),
                                 static_cast<int32_t>(p >> 32), 0};
  }
}
static_assert(kObjPerThread * 32 < 1024, "a warp's counts are packed in ten bits each");

// One CTA: a group of lanes per row, the records added in a fixed order. stats: tokens, mean k3,
// the shares of the tokens held by the lower and by the upper border. weight: one number (token),
// or one per row.
__global__ void __launch_bounds__(1024)
policy_total_kernel(const Record* records, int chunks, int lanes, int64_t rows,
                    Params par, const double* __restrict__ denom_dev, float* __restrict__ loss,
                    float* __restrict__ stats, float* __restrict__ weight) {
  qb::await_previous();
  __shared__ double scratch[160];
  double total = 0.0, kl = 0.0, count = 0.0, low = 0.0, high = 0.0;
  const bool given = denom_dev || par.denominator > 0;
  const double asked = denom_dev ? *denom_dev : par.denominator;
  const double per = given ? asked : double(rows);          // sequence mode
  const int sub = threadIdx.x % lanes, group = threadIdx.x / lanes, groups = blockDim.x / lanes;
  for (int64_t r0 = 0; r0 < rows; r0 += groups) {           // whole warps go round together
    const int64_t r = r0 + group;
    double row_loss = 0.0, row_count = 0.0;
    if (r < rows) {
      for (int k = sub; k < chunks; k += lanes) {
        const Record rec = records[r * chunks + k];
        row_loss += rec.loss;
        kl += rec.kl;
        row_count += rec.count;
        low += rec.low;
        high += rec.high;
      }
    }
    count += row_count;
    if (!par.sequence) {
      total += row_loss;
      continue;
    }
    row_loss = qb::group_sum64(row_loss, lanes);
    row_count = qb::group_sum64(row_count, lanes);
    if (r < rows && sub == 0) {
      const double each = fmax(row_count, 1.0);
      total += row_loss / each;
      weight[r] = static_cast<float>(1.0 / (each * per));
    }
  }
  double all[5] = {total, kl, count, low, high};
  qb::block_sums64<true>(all, scratch);
  if (threadIdx.x >= 32) return;
  // a lane each for the five quotients
  const double tokens = fmax(all[2], 1.0);
  const double denom = par.sequence ? per : given ? asked : tokens;
  const int k = threadIdx.x;
  const float q = static_cast<float>((k == 0 ? all[0] : k == 1 ? 1.0 : k == 2 ? all[1]
                                      : k == 3 ? all[3] : all[4]) / (k < 2 ? denom : tokens));
  if (k == 0) {
    *loss = q;
    stats[0] = static_cast<float>(all[2]);
  } else if (k == 1) {
    if (!par.sequence) weight[0] = q;
  } else if (k < 5) {
    stats[k - 1] = q;
  }
}

template <typename T>
__global__ void __launch_bounds__(kObjThreads)
policy_bwd_kernel(const float* __restrict__ unit, const float* __restrict__ weight,
                  int64_t weight_row, const float* __restrict__ g, int64_t cols, int chunks,
                  T* __restrict__ grad) {
  const int64_t row = blockIdx.x / static_cast<unsigned>(chunks);
  const int64_t c0 = int64_t(blockIdx.x % static_cast<unsigned>(chunks)) * kObjChunk + threadIdx.x;
  const int left = static_cast<int>(cols - c0 < kObjChunk ? cols - c0 : kObjChunk);
  unit += row * cols + c0;
  grad += row * cols + c0;
  const float w = weight[row * weight_row] * *g;
  float v[kObjPerThread];
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k)
    v[k] = k * kObjThreads < left ? unit[k * kObjThreads] : 0.f;
#pragma unroll
  for (int k = 0; k < kObjPerThread; ++k)
    // a token without a gradient (masked, or held by the clip) has none whatever g is
    if (k * kObjThreads < left)
      grad[k * kObjThreads] = qb::from_f<T>(v[k] == 0.f ? 0.f : v[k] * w);
}

int check(const char* what, int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0)
    return qb::fail(QB_ERR_INVALID, "%s: bad shape (%lld x %lld)", what, (long long)rows,
                    (long long)cols);
  if (rows > 0x7fffffff || (cols + kObjChunk - 1) / kObjChunk > 0x7fffffff / rows)
    return qb::fail(QB_ERR_INVALID, "%s: too large", what);
  return QB_OK;
}

int chunks_of(int64_t cols) { return static_cast<int>((cols + kObjChunk - 1) / kObjChunk); }

}  // namespace

extern "C" int64_t qb_policy_config_size(void) { return sizeof(qb_policy_config); }

extern "C" int64_t qb_policy_workspace(int64_t rows, int64_t cols) {
  if (check("policy", rows, cols) != QB_OK) return 0;
  return rows * chunks_of(cols) * static_cast<int64_t>(sizeof(Record));
}

extern "C" int qb_policy_fwd(const void* logp, const void* old_logp, const void* ref, int dtype,
                             const float* advantages, int64_t adv_row_stride,
                             int64_t adv_col_stride, const uint8_t* mask, int64_t rows,
                             int64_t cols, const qb_policy_config* cfg,
                             const double* denominator, float* loss, float* stats,
                             float* weight, float* unit_grad, void* workspace,
                             cudaStream_t stream) {
  if (int rc = check("policy", rows, cols)) return rc;
  if (!logp || !advantages || !cfg || !loss || !stats || !weight || !workspace)
    return qb::fail(QB_ERR_INVALID, "policy: null pointer");
  if (!(cfg->clip_low >= 0 && cfg->clip_low <= 1) || !(cfg->clip_high >= 0) ||
      (cfg->delta != 0 && !(cfg->delta > 1 + cfg->clip_high)) ||
      cfg->reduction < 0 || cfg->reduction > 1 || cfg->kl_coef != cfg->kl_coef)
    return qb::fail(QB_ERR_INVALID, "policy: bad clip range, delta, KL coefficient or reduction");
  const int chunks = chunks_of(cols);
  auto* records = static_cast<Record*>(workspace);
  Params par;
  par.log_low = log1p(-cfg->clip_low);        // -inf for a lower border of 0
  par.log_high = log1p(cfg->clip_high);
  par.log_delta = cfg->delta > 0 ? log(cfg->delta) : INFINITY;
  par.log_low32 = static_cast<float>(par.log_low);
  par.log_high32 = static_cast<float>(par.log_high);
  par.log_delta32 = static_cast<float>(par.log_delta);
  par.low = static_cast<float>(1.0 - cfg->clip_low);
  par.high = static_cast<float>(1.0 + cfg->clip_high);
  par.delta = cfg->delta > 0 ? static_cast<float>(cfg->delta) : INFINITY;
  par.kl_coef = static_cast<float>(cfg->kl_coef);
  par.denominator = cfg->denominator;
  par.sequence = cfg->reduction == 1;
  QB_DISPATCH_FLOAT(dtype, T, {
    policy_rows_kernel<T><<<static_cast<unsigned>(rows * chunks), kObjThreads, 0, stream>>>(
        static_cast<const T*>(logp), static_cast<const T*>(old_logp), static_cast<const T*>(ref),
        advantages, adv_row_stride, adv_col_stride, mask, cols, chunks, par, records, unit_grad);
  });
  if (int rc = qb::check_launch("policy")) return rc;
  const int lanes = qb::lanes_per_row(chunks);
  qb::launch_after(policy_total_kernel, 1, qb::adding_threads(rows, lanes), stream, records,
                   chunks, lanes, rows, par, denominator, loss, stats, weight);
  return qb::check_launch("policy");
}

extern "C" int qb_policy_bwd(const float* unit_grad, const float* weight,
                             int64_t weight_row_stride, const float* g, int64_t rows,
                             int64_t cols, void* grad, int dtype, cudaStream_t stream) {
  if (int rc = check("policy_bwd", rows, cols)) return rc;
  if (!unit_grad || !weight || !g || !grad)
    return qb::fail(QB_ERR_INVALID, "policy_bwd: null pointer");
  const int chunks = chunks_of(cols);
  QB_DISPATCH_FLOAT(dtype, T, {
    policy_bwd_kernel<T><<<static_cast<unsigned>(rows * chunks), kObjThreads, 0, stream>>>(
        unit_grad, weight, weight_row_stride, g, cols, chunks, static_cast<T*>(grad));
  });
  return qb::check_launch("policy_bwd");
}
