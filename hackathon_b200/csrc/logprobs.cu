// Log-probabilities of chosen tokens (and the entropy of each row's distribution) from rows of
// materialised logits, forward and backward.
//
// With temperature T, c = log2(e) / T and a row's maximum m:
//   d_j = z_j - m,  e_j = 2^(c d_j),  s = sum e_j,  t = sum e_j d_j
//   logp = d_label / T - ln s                H = ln s - t / (s T)
//   dz_j = (1/T) [ g (1{j = label} - p_j) - g_H p_j (ln p_j + H) ],  p_j = e_j / s
//        = e_j (A + B d_j) for j != label,  A = -(g + g_H (H - ln s)) / (T s),  B = -g_H / (T^2 s)
//        = e_j (A' + B d_j) + (g / T) (s - e_j) / s  at the label,  A' = -g_H (H - ln s) / (T s)
// The label's 1 - p is taken from s before any product is rounded: g / T and -g p / T, each rounded
// by itself, leave an error of 2^-24 g / T, which is 4 % of a gradient with 1 - p = 2^-20.
// Sums and maxima are fp32. The maximum is subtracted before the scale: z c - m c in one fused
// multiply-add would save an operation, but leaves the rounding of m c in every exponent, which
// grows with |m| / T, and makes a certain token's log-probability something near 0 instead of 0.
//
// A banned token (a logit of -inf) has e = 0 and no e d term: d is held at -300 T, where e is 0 and
// every product with d finite. Rows need no other care: one of equal lowest values is the uniform
// distribution, one of -inf alone, with +inf or with NaN is NaN, as the formula is.
#include <algorithm>
#include <cstring>

#include "qb_common.cuh"

namespace {

// 128 threads and 8 KB a batch: many small CTAs on an SM are each at another point of their row, so
// loads and exponentials overlap (4096 x 152064 bf16: 189 us, 205 us with 512 threads and as many
// bytes an SM in flight; with the entropy 196 and 227).
constexpr int kFwdThreads = 128;
constexpr int kFwdVectors = 4;         // 16-byte vectors per thread and batch
constexpr int64_t kFwdCtas = 8 * 148;  // CTAs aimed at: eight on an SM (registers allow 9 or 10)
constexpr float kLog2e = 1.4426950408889634f;

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

// ---------------------------------------------------------------------------------------------
// Two fp32 values in one 64-bit register: one issue slot for two additions or multiplications.

using Pair = unsigned long long;

__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void halves(Pair p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes of logits: pair k of them less m, in fp32, and their maximum (a NaN stays one). The
// 16-bit types are widened inside the subtraction (one instruction for both).
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  uint4 u;
  __device__ __forceinline__ Pair less(int k, float m) const {
    const Pair z = k == 0 ? pair(__uint_as_float(u.x), __uint_as_float(u.y))
                          : pair(__uint_as_float(u.z), __uint_as_float(u.w));
    return add2(z, pair(-m, -m));
  }
  __device__ __forceinline__ float top() const {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)),
                   max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ uint32_t none() { return 0xff800000u; }   // -inf
};
template <typename H2>
__device__ __forceinline__ H2 word_as(uint32_t w) {
  H2 h;
  memcpy(&h, &w, 4);
  return h;
}
template <typename H2> struct Vec16Bit {
  static constexpr int N = 8;
  uint4 u;
  __device__ __forceinline__ uint32_t word(int k) const {
    return k == 0 ? u.x : k == 1 ? u.y : k == 2 ? u.z : u.w;
  }
  __device__ __forceinline__ uint16_t low(int k) const { return word(k) & 0xffffu; }
  __device__ __forceinline__ uint16_t high(int k) const { return word(k) >> 16; }
  __device__ __forceinline__ float top() const {
    const H2 m = __hmax2_nan(__hmax2_nan(word_as<H2>(u.x), word_as<H2>(u.y)),
                             __hmax2_nan(word_as<H2>(u.z), word_as<H2>(u.w)));
    return max_nan(qb::to_f(m.x), qb::to_f(m.y));
  }
};
template <> struct Vec<__nv_bfloat16> : Vec16Bit<__nv_bfloat162> {
  __device__ __forceinline__ Pair less(int k, float m) const {
    float lo, hi;
    asm("add.rn.f32.bf16 %0, %1, %2;" : "=f"(lo) : "h"(low(k)), "f"(-m));
    asm("add.rn.f32.bf16 %0, %1, %2;" : "=f"(hi) : "h"(high(k)), "f"(-m));
    return pair(lo, hi);
  }
  static __device__ __forceinline__ uint32_t none() { return 0xff80ff80u; }
};
template <> struct Vec<__half> : Vec16Bit<__half2> {
  __device__ __forceinline__ Pair less(int k, float m) const {
    float lo, hi;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(lo) : "h"(low(k)), "f"(-m));
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(hi) : "h"(high(k)), "f"(-m));
    return pair(lo, hi);
  }
  static __device__ __forceinline__ uint32_t none() { return 0xfc00fc00u; }
};

// max, sum 2^(d c), sum 2^(d c) d of a set of elements, d relative to m.
struct Stat {
  float m, s, t;
};

// c, and the d below which nothing is left of e.
struct Scale {
  float c, low;
  __device__ __forceinline__ explicit Scale(float inv_t) : c(inv_t * kLog2e), low(-300.f / inv_t) {}
};

// From one maximum to a larger one (from -inf, with s = t = 0, too).
__device__ __forceinline__ void rescale(Stat& a, float m, Scale c) {
  const float d = fmaxf(a.m - m, c.low);
  const float f = ex2(d * c.c);
  a.t = (a.t + a.s * d) * f;
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ Stat merge(Stat a, Stat b, Scale c) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, c);
  rescale(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ Stat warp_merge(Stat st, Scale c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
               __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = merge(st, other, c);
  }
  return st;
}

// U vectors of a thread: one maximum and at most one rescaling for all of them, and sums of their
// own that join the thread's at the end. (Added one by one, a thread that holds the row's top token
// rounds every term at that one's last place: 2.6e-7 instead of 1.2e-7 in the gradient of 999 rows
// of 50001, at the same time.)
template <typename T, bool ENT, int U>
__device__ __forceinline__ void add_vectors(Stat& st, const Vec<T> (&x)[U], Scale c) {
  float m = x[0].top();
#pragma unroll
  for (int u = 1; u < U; ++u) m = max_nan(m, x[u].top());
  if (m == -INFINITY) return;    // all banned: nothing to add, and no maximum to subtract
  if (m > st.m) rescale(st, m, c);
  const Pair cc = pair(c.c, c.c);
  Pair s = pair(0.f, 0.f), t = pair(0.f, 0.f);
  float lo, hi;
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int k = 0; k < Vec<T>::N / 2; ++k) {
      const Pair d = x[u].less(k, st.m);
      halves(mul2(d, cc), lo, hi);
      const Pair e = pair(ex2(lo), ex2(hi));
      s = add2(s, e);
      if (ENT) {
        halves(d, lo, hi);
        t = fma2(e, pair(max_nan(lo, c.low), max_nan(hi, c.low)), t);
      }
    }
  }
  halves(s, lo, hi);
  st.s += lo + hi;
  halves(t, lo, hi);
  st.t += lo + hi;
}

template <bool ENT>
__device__ __forceinline__ void add_one(Stat& st, float z, Scale c) {
  if (z == -INFINITY) return;
  if (z > st.m) rescale(st, z, c);
  const float d = max_nan(z - st.m, c.low);
  const float e = ex2(d * c.c);
  st.s += e;
  if (ENT) st.t += e * d;
}

// What bounds it: HBM, and right behind it the power limit (a loop of seconds runs at 990 of 1000 W
// and 1755 MHz: 204 us where a burst takes 189). The XU's exponentials need three quarters of HBM's
// time; moving a quarter of them to the FMA pipes (a polynomial) was slower, 209 us in the loop.
//
// One CTA per (row, span of the vocabulary): batches of kFwdVectors vectors a thread, the next one
// requested before the present one is added up. The CTA's record goes to `partials`, or, where
// one span is the whole row, straight to the outputs.
struct Outputs {
  const int64_t* target;
  float* logp;
  float* entropy;      // NULL: not asked for
  float2* stats;
};

template <typename T>
__device__ __forceinline__ void finish(const Outputs& out, int64_t row, const T* z, int vocab,
                                       float inv_t, Stat st) {
  const int64_t label = out.target[row];
  const float log_s = logf(st.s);
  float lp = 0.f;
  if (label >= 0 && label < vocab) lp = (qb::to_f(z[label]) - st.m) * inv_t - log_s;
  out.logp[row] = lp;
  if (out.entropy) out.entropy[row] = log_s - inv_t * (st.t / st.s);
  out.stats[row] = make_float2(st.m, st.s);
}

template <typename T, bool ENT>
__global__ void __launch_bounds__(kFwdThreads)
token_logprobs_kernel(const T* __restrict__ logits, Rows rows, int vocab, int spans, int batches,
                      float inv_t, Outputs out, float4* __restrict__ partials) {
  constexpr int VE = Vec<T>::N;
  constexpr int U = kFwdVectors;
  __shared__ Stat warp_stat[kFwdThreads / 32];
  qb::release_next();
  const int64_t row = blockIdx.x / spans;
  const int span = blockIdx.x % spans;
  const T* z = logits + rows.offset(row);
  const Scale c(inv_t);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // scalars before the first 16-byte boundary and after the last (the first span takes them),
  // vectors between; a thread past the end adds banned tokens
  const int head = min(vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15)
                                               / sizeof(T)));
  const int nvec = (vocab - head) / VE;
  const T* body = z + head;
  const uint4 none = {Vec<T>::none(), Vec<T>::none(), Vec<T>::none(), Vec<T>::none()};
  const int first = span * batches * (kFwdThreads * U) + threadIdx.x;
  const int end = min(nvec, first + batches * (kFwdThreads * U));
  auto load = [&](Vec<T>(&x)[U], int v) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u].u = v + u * kFwdThreads < end
                   ? __ldg(reinterpret_cast<const uint4*>(body + int64_t(v + u * kFwdThreads) * VE))
                   : none;
  };
  Stat st{-INFINITY, 0.f, 0.f};
  Vec<T> x[U], next[U];
  load(x, first);
  for (int v = first; v < end; v += U * kFwdThreads) {
    load(next, v + U * kFwdThreads);
    add_vectors<T, ENT, U>(st, x, c);
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = next[u];
  }
  if (span == 0 && static_cast<int>(threadIdx.x) < vocab - nvec * VE) {
    const int j = threadIdx.x;
    add_one<ENT>(st, qb::to_f(z[j < head ? j : nvec * VE + j]), c);
  }
  st = warp_merge(st, c);
  if (lane == 0) warp_stat[warp] = st;
  __syncthreads();
  if (warp != 0) return;
  st = lane < kFwdThreads / 32 ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
  st = warp_merge(st, c);
  if (lane != 0) return;
  if (spans == 1) finish(out, row, z, vocab, inv_t, st);
  else partials[blockIdx.x] = make_float4(st.m, st.s, st.t, 0.f);
}

// A warp per row: the row's records, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256)
token_logprobs_merge_kernel(const T* __restrict__ logits, Rows rows, int64_t n, int vocab,
                            int spans, float inv_t, Outputs out, const float4* partials) {
  qb::await_previous();
  const int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= n) return;
  const int lane = threadIdx.x & 31;
  const Scale c(inv_t);
  Stat st{-INFINITY, 0.f, 0.f};
  for (int k = lane; k < spans; k += 32) {
    const float4 p = partials[row * spans + k];
    st = merge(st, Stat{p.x, p.y, p.z}, c);
  }
  st = warp_merge(st, c);
  if (lane == 0) finish(out, row, logits + rows.offset(row), vocab, inv_t, st);
}

// ---------------------------------------------------------------------------------------------
// backward: elementwise given the row's (m, s, H); one CTA per (row, tile of columns). HBM bounds
// it: 4096 x 152064 bf16 in 380 us, 6.55 TB/s of reads and writes; 400 us with the entropy's
// gradient. Four vectors a thread instead of eight: 424 us.

constexpr int kThreads = 256;
constexpr int kVectors = 8;            // per thread, all requested at once: 32 KB of logits a CTA

__device__ __forceinline__ uint32_t packed(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &h, 4);
  return w;
}
__device__ __forceinline__ uint32_t packed(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &h, 4);
  return w;
}

// The row's numbers, and dlogits of one element or one vector, and of the target's.
struct RowGrad {
  float m, a, b;
  Scale c;
  float s, hot, a_hot;   // of the target's element: s, g / T, A'
  __device__ __forceinline__ float target(float z) const {
    const float d = max_nan(z - m, c.low);
    const float e = ex2(d * c.c);
    return fmaf(hot, (s - e) / s, e * fmaf(b, d, a_hot));
  }
  __device__ __forceinline__ float one(float z) const {
    const float d = max_nan(z - m, c.low);
    return ex2(d * c.c) * fmaf(b, d, a);
  }
  __device__ __forceinline__ void two(Pair less, float& lo, float& hi) const {
    float x, y;
    halves(less, x, y);
    const Pair d = pair(max_nan(x, c.low), max_nan(y, c.low));
    halves(mul2(d, pair(c.c, c.c)), x, y);
    halves(mul2(pair(ex2(x), ex2(y)), fma2(pair(b, b), d, pair(a, a))), lo, hi);
  }
  __device__ __forceinline__ uint4 vec(const Vec<float>& x) const {
    float f[4];
    two(x.less(0, m), f[0], f[1]);
    two(x.less(1, m), f[2], f[3]);
    return {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
            __float_as_uint(f[3])};
  }
  template <typename T>
  __device__ __forceinline__ uint4 vec(const Vec<T>& x) const {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo, hi;
      two(x.less(k, m), lo, hi);
      w[k] = packed(lo, hi, T());
    }
    return {w[0], w[1], w[2], w[3]};
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
token_logprobs_bwd_kernel(const T* __restrict__ logits, Rows rows, int vocab, int tiles,
                          const int64_t* __restrict__ target, float inv_t,
                          const float2* __restrict__ stats, const float* __restrict__ entropy,
                          const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                          T* __restrict__ dlogits) {
  constexpr int VE = Vec<T>::N;
  constexpr int U = kVectors;
  const int64_t row = blockIdx.x / tiles;
  const int tile = blockIdx.x % tiles;
  const T* z = logits + rows.offset(row);
  T* dz = dlogits + row * vocab;
  const int64_t label = target[row];
  const bool labelled = label >= 0 && label < vocab;
  const float g = labelled && g_logp ? g_logp[row] : 0.f;
  const float gh = g_ent ? g_ent[row] : 0.f;
  const bool zero = g == 0.f && gh == 0.f;   // e.g. a prompt's positions: nothing to read

  // scalars before the first 16-byte boundary of the gradient and after its last
  const int head = min(vocab, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dz) & 15)) & 15)
                                               / sizeof(T)));
  const int nvec = (vocab - head) / VE;
  const int v0 = tile * (kThreads * U) + threadIdx.x;
  if (zero) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * kThreads < nvec)
        *reinterpret_cast<uint4*>(dz + head + int64_t(v0 + u * kThreads) * VE) = {0, 0, 0, 0};
    if (tile == 0)
      for (int j = threadIdx.x; j < vocab - nvec * VE; j += kThreads)
        dz[j < head ? j : nvec * VE + j] = qb::from_f<T>(0.f);
    return;
  }
  const bool vec_in =
      ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  Vec<T> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + u * kThreads;
    if (v < nvec) {
      const T* p = z + head + int64_t(v) * VE;
      if (vec_in) {
        x[u].u = __ldg(reinterpret_cast<const uint4*>(p));
      } else {
        T f[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = p[e];
        memcpy(&x[u].u, f, 16);
      }
    }
  }
  const float2 ms = stats[row];
  const float k = inv_t / ms.y, log_s = logf(ms.y);
  const float ent = g_ent ? gh * (entropy[row] - log_s) : 0.f;
  const RowGrad grad{ms.x, -(g + ent) * k, -gh * inv_t * k, Scale(inv_t),
                     ms.y, g * inv_t,      -ent * k};
  // the target's element is rewritten by the thread that wrote its vector
  const int hot_col = labelled ? static_cast<int>(label) : -1;
  const int hot_vec = hot_col >= head && hot_col < head + nvec * VE ? (hot_col - head) / VE : -1;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + u * kThreads;
    if (v < nvec) *reinterpret_cast<uint4*>(dz + head + int64_t(v) * VE) = grad.vec(x[u]);
  }
  if (hot_vec >= 0 && hot_vec / (kThreads * U) == tile &&
      hot_vec % kThreads == static_cast<int>(threadIdx.x))
    dz[hot_col] = qb::from_f<T>(grad.target(qb::to_f(z[hot_col])));
  if (tile == 0) {
    for (int j = threadIdx.x; j < vocab - nvec * VE; j += kThreads) {
      const int col = j < head ? j : nvec * VE + j;
      const float zc = qb::to_f(z[col]);
      dz[col] = qb::from_f<T>(col == hot_col ? grad.target(zc) : grad.one(zc));
    }
  }
}

// Spans of a row and batches of a span: rows are cut into kFwdCtas / rows spans, down to a batch a
// CTA; from half of kFwdCtas rows on that is 1, whole rows and no merging launch. Cutting evens
// out the last wave but pays a reduction and a record for each span. Whole against cut, 151936
// bf16 with the entropy: 593 rows 41.6 us, 40.0 in 3 spans; 700 42.5, 44.0; 789 50.8, 47.4; 888
// 50.5, 56.4 in 2; 1000 58.2, 59.9; 1183 65.3, 65.8. 999 rows of 50001 fp32 take 33 us whole and
// 36 to 38 in 4 to 9 spans; 148 rows of 151936 bf16 14.7 us in 8 spans, 17.7 us in 2.
struct Spans {
  int64_t spans, batches;
};
Spans spans_of(int64_t rows, int64_t vocab, int e) {
  const int64_t batch = int64_t(kFwdThreads) * kFwdVectors * (16 / e);
  const int64_t all = (vocab + batch - 1) / batch;
  const int64_t want = std::min(all, std::max<int64_t>(1, kFwdCtas / rows));
  const int64_t batches = (all + want - 1) / want;
  return {(all + batches - 1) / batches, batches};
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

extern "C" int64_t qb_token_logprobs_workspace(int64_t rows, int64_t vocab, int dtype) {
  const int e = qb::elem_size(dtype);
  if (rows <= 0 || vocab <= 0 || e == 0) return 0;
  const int64_t spans = spans_of(rows, vocab, e).spans;
  return spans > 1 ? rows * spans * static_cast<int64_t>(sizeof(float4)) : 0;
}

extern "C" int qb_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t inner,
                                 int64_t stride_outer, int64_t stride_inner, int64_t vocab,
                                 const int64_t* target, float temperature, float* logp,
                                 float* entropy, float* stats, void* workspace,
                                 cudaStream_t stream) {
  if (int rc = check("token_logprobs", logits, rows, inner, vocab, target, temperature, stats))
    return rc;
  if (rows == 0) return QB_OK;
  const Rows r{inner, stride_outer, stride_inner};
  const float inv_t = 1.f / temperature;
  const Outputs out{target, logp, entropy, reinterpret_cast<float2*>(stats)};
  auto* partials = static_cast<float4*>(workspace);
  QB_DISPATCH_FLOAT(dtype, T, {
    const Spans sp = spans_of(rows, vocab, sizeof(T));
    if (!logp || (sp.spans > 1 && !workspace))
      return qb::fail(QB_ERR_INVALID, "token_logprobs: null pointer");
    if (rows > 0x7fffffff / sp.spans)
      return qb::fail(QB_ERR_INVALID, "token_logprobs: too many rows");
    const auto* z = static_cast<const T*>(logits);
    const unsigned grid = static_cast<unsigned>(rows * sp.spans);
    const int spans = static_cast<int>(sp.spans), batches = static_cast<int>(sp.batches);
    if (entropy)
      token_logprobs_kernel<T, true><<<grid, kFwdThreads, 0, stream>>>(
          z, r, (int)vocab, spans, batches, inv_t, out, partials);
    else
      token_logprobs_kernel<T, false><<<grid, kFwdThreads, 0, stream>>>(
          z, r, (int)vocab, spans, batches, inv_t, out, partials);
    if (int rc = qb::check_launch("token_logprobs")) return rc;
    if (spans > 1)
      qb::launch_after(token_logprobs_merge_kernel<T>, static_cast<unsigned>((rows + 7) / 8), 256,
                       stream, z, r, rows, (int)vocab, spans, inv_t, out, partials);
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
    constexpr int64_t kTile = int64_t(kThreads) * kVectors * Vec<T>::N;
    const int64_t tiles = (vocab + kTile - 1) / kTile;
    if (rows > 0x7fffffff / tiles)
      return qb::fail(QB_ERR_INVALID, "token_logprobs_bwd: too many rows");
    token_logprobs_bwd_kernel<T><<<static_cast<unsigned>(rows * tiles), kThreads, 0, stream>>>(
        static_cast<const T*>(logits), r, (int)vocab, (int)tiles, target, 1.f / temperature,
        reinterpret_cast<const float2*>(stats), entropy, g_logp, g_entropy,
        static_cast<T*>(dlogits));
  });
  return qb::check_launch("token_logprobs_bwd");
}
