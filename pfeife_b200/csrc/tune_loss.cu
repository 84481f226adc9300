// Losses on the log-probabilities of given tokens: a preference loss over pairs of sequences and a clipped policy
// loss over sampled tokens, forward and backward.
//
// Both take logits z [N, T, V] (any strides, V innermost) and a label for each row; a row whose label is the ignored
// one or outside the vocabulary does not count: its logits are not read, and its gradient is zero.
// The forward passes over a row once and keeps M and s = sum 2^(k z - M), k = log2(e) / temperature, M the largest
// k z rounded up to an integer: log p = ln 2 (k z_label - M - log2 s).
// A preference subtracts sums over thousands of tokens from one another, which show what is off by the same little
// part in every row (rewards of sequences of 1024 tokens were 3e-5 off).  So parts of a row are joined between
// integers, by powers of two, which are exact; and each lane has a fraction of its own between its reference and
// the integer, since 16-bit logits lie on a grid on which the exponential's errors would be the same in every row.
// What follows is a few operations per row, done in 64 bits by one thread: those differences, and a KL estimate
// exp(d) - d - 1, which loses d^2 / 2 next to 1.
// The backward passes over it again: dz = g (onehot - p) with p = 2^(k z - M) / s and g what the loss has for the
// row's log-probability, so that only M, s and g are kept.
#include "common.cuh"
#include "api.h"

namespace pf {

constexpr double LN2 = 0.693147180559945309417;
// ex2.approx cuts its last bits off: it is low by this part of its value on average (over 2^20 arguments of one
// binade), and so is s.  A single probability hides that in its rounding, a sum over a sequence does not.  The
// backward divides such values by such sums, where it cancels.
constexpr double EXP2_LOW = 5.06e-8;

struct Logits {                    // z [N, T, V]
  const void* at;
  const long long* labels;         // [N * T]
  long long n, t;                  // strides in elements
  long long rows, ignore;
  int T, V;
  float k;                         // log2(e) / temperature
  __device__ __forceinline__ long long row(long long r) const {
    const long long s = r / T;
    return s * n + (r - s * T) * t;
  }
  __device__ __forceinline__ bool counts(long long label) const {
    return label >= 0 && label < V && label != ignore;
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (M, s) of two parts of a row, with integers M; a part without a finite element is (-inf, 0), or (-inf, NaN) when it holds a NaN,
// which no maximum shows: the sums are always added, and -inf counts as 0 where it is subtracted.
__device__ __forceinline__ void part_merge(float& m, float& s, float m2, float s2) {
  const float mm = fmaxf(m, m2), sub = mm == -INFINITY ? 0.f : mm;
  s = s * exp2_fast(m - sub) + s2 * exp2_fast(m2 - sub);
  m = mm;
}

// What a loss makes of a row, in 64 bits.
struct PolicyRow {
  const float *old, *ref, *adv;    // ref null: no reference
  long long adv_n, adv_t;          // strides of the advantages
  float low, high, kl;
  double inv_temperature;
  float *logp, *coef;              // coef: of the row's own term, before the mean
  float4* terms;                   // (term, KL, clipped, counted)
  __device__ __forceinline__ void operator()(const Logits& z, long long r, bool counted, double lp) const {
    if (!counted) {
      logp[r] = coef[r] = 0.f;
      terms[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      return;
    }
    const long long n = r / z.T;
    const double a = adv[n * adv_n + (r - n * z.T) * adv_t], ratio = exp(lp - (double)old[r]);
    const double lo = 1.0 - (double)low, hi = 1.0 + (double)high;
    const double free = ratio * a, held = fmin(fmax(ratio, lo), hi) * a;
    const bool clipped = free > held;
    double term = clipped ? -held : -free, c = clipped ? 0.0 : -free, each = 0.0;
    if (ref) {
      const double d = (double)ref[r] - lp, e = expm1(d);
      each = e - d;
      term += kl * each;
      c -= kl * e;
    }
    logp[r] = (float)lp;
    coef[r] = (float)(c * inv_temperature);
    terms[r] = make_float4((float)term, (float)each, clipped ? 1.f : 0.f, 1.f);
  }
};
struct PreferenceRow {
  double* logp;
  __device__ __forceinline__ void operator()(const Logits&, long long r, bool counted, double lp) const {
    logp[r] = counted ? lp : 0.0;
  }
};

// One pass over each row that counts.  THREADS threads a row: whole CTAs, or warps that share a CTA of 256.
template <typename T, int THREADS, typename Row>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
row_fwd_kernel(const Logits z, float2* __restrict__ stats, const Row finish) {
  after_previous();
  constexpr int W = THREADS / 32, VN = 16 / sizeof(T), U = 4;
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  static_assert(ROWS == 1 || W == 1, "rows that share a CTA are a warp each");
  __shared__ float smax[W], ssum[W];
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (row >= z.rows) return;
  const int tid = threadIdx.x % THREADS;
  const long long label = z.labels[row];
  if (!z.counts(label)) {
    if (tid == 0) finish(z, row, false, 0.0);
    return;
  }
  const T* x = static_cast<const T*>(z.at) + z.row(row);
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(z.V, mis ? VN - mis : 0), nvec = (z.V - head) / VN;
  const float k = z.k, fraction = (threadIdx.x & 31) * (1.f / 32);
  float m = -INFINITY, s = 0.f;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  for (int i0 = tid; i0 < nvec; i0 += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * THREADS < nvec) q[u] = __ldg(xv + i0 + u * THREADS);
    float lm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * THREADS < nvec) {
        const T* e = reinterpret_cast<const T*>(&q[u]);
#pragma unroll
        for (int j = 0; j < VN; ++j) lm = fmaxf(lm, to_f32<T>(e[j]));
      }
    // a NaN does not move the maximum but reaches the sum below; parts that are -inf so far subtract 0, which
    // leaves their exponentials at zero
    const float mm = fmaxf(m, ceilf(lm * k) + fraction), sub = mm == -INFINITY ? 0.f : mm;
    if (mm > m) s *= exp2_fast(m - sub);
    float a = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * THREADS < nvec) {
        const T* e = reinterpret_cast<const T*>(&q[u]);
#pragma unroll
        for (int j = 0; j < VN; ++j) a += exp2_fast(fmaf(to_f32<T>(e[j]), k, -sub));
      }
    s += a;
    m = mm;
  }
  // the elements before the first and after the last vector (at most 2 (VN - 1))
  for (int i = tid; i < z.V - nvec * VN; i += THREADS) {
    const float v = to_f32<T>(x[i < head ? i : nvec * VN + i]);
    const float mm = fmaxf(m, ceilf(v * k) + fraction), sub = mm == -INFINITY ? 0.f : mm;
    s = s * exp2_fast(m - sub) + exp2_fast(fmaf(v, k, -sub));
    m = mm;
  }
  if (m > -INFINITY) {
    const float whole = ceilf(m);
    s *= exp2f(m - whole);
    m = whole;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    part_merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if (W > 1) {
    const int w = tid >> 5, l = tid & 31;
    if (l == 0) { smax[w] = m; ssum[w] = s; }
    __syncthreads();
    if (w > 0) return;
    m = l < W ? smax[l] : -INFINITY;
    s = l < W ? ssum[l] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      part_merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  }
  if (tid == 0) {
    stats[row] = make_float2(m, s);
    const double lp = LN2 * ((double)to_f32<T>(x[label]) * (double)k - (double)m) - log((double)s) - EXP2_LOW;
    finish(z, row, true, lp);
  }
}

// sums over a CTA of 1024 threads, for its first warp
__device__ __forceinline__ double cta_sum(double v, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Means over the rows that count: out = (loss, KL, clipped, one over their number).
__global__ void __launch_bounds__(1024)
policy_mean_kernel(const float4* __restrict__ terms, float* __restrict__ loss, float* __restrict__ kl,
                   float* __restrict__ clipped, float* __restrict__ inv, long long rows) {
  after_previous();
  __shared__ double scratch[32];
  double t = 0.0, e = 0.0, c = 0.0, n = 0.0;
#pragma unroll 4
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    const float4 v = terms[r];
    t += v.x; e += v.y; c += v.z; n += v.w;
  }
  t = cta_sum(t, scratch);
  e = cta_sum(e, scratch);
  c = cta_sum(c, scratch);
  n = cta_sum(n, scratch);
  if (threadIdx.x == 0) {
    const double one = 1.0 / (n > 0.0 ? n : 1.0);
    *loss = (float)(t * one);
    *kl = (float)(e * one);
    *clipped = (float)(c * one);
    *inv = (float)one;
  }
}

// Rewards of the sequences, the mean loss over the pairs and what a sequence's log-probability gets of it.
__global__ void __launch_bounds__(1024)
preference_kernel(const double* __restrict__ logp, const float* __restrict__ ref, float* __restrict__ rewards,
                  double* __restrict__ sums, float* __restrict__ loss, float* __restrict__ coef, int N, int T,
                  float beta, float smoothing) {
  after_previous();
  __shared__ double scratch[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int n = warp; n < N; n += 32) {
    double t = 0.0;
#pragma unroll 4
    for (int i = lane; i < T; i += 32) t += logp[(long long)n * T + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) {
      const double reward = (double)beta * (t - (double)ref[n]);
      sums[n] = reward;
      rewards[n] = (float)reward;
    }
  }
  __syncthreads();
  const int P = N / 2;
  double total = 0.0;
  for (int p = threadIdx.x; p < P; p += 1024) {
    const double m = sums[p] - sums[P + p], e = exp(-fabs(m)), near = log1p(e);
    // -log sig(m) and -log sig(-m), sig(-m) and sig(m), none of which overflows
    const double lp = near + fmax(-m, 0.0), lm = near + fmax(m, 0.0);
    const double big = 1.0 / (1.0 + e), small = e / (1.0 + e);
    total += smoothing < 1.f ? (1.0 - (double)smoothing) * lp : 0.0;      // 0 x inf is not 0
    total += smoothing > 0.f ? (double)smoothing * lm : 0.0;
    const double c = -(double)beta / P * ((1.0 - (double)smoothing) * (m > 0.0 ? small : big) -
                                          (double)smoothing * (m > 0.0 ? big : small));
    coef[p] = (float)c;
    coef[P + p] = (float)-c;
  }
  total = cta_sum(total, scratch);
  if (threadIdx.x == 0) *loss = (float)(total / P);
}

// dz = g (onehot - p), g = coef[row / per] * gout * inv (inv null: 1).  THREADS threads a row; with 256 the grid is
// (row, slab of the row).
template <typename T, int THREADS>
__global__ void __launch_bounds__(256)
row_bwd_kernel(const Logits z, const float2* __restrict__ stats, const float* __restrict__ coef,
               const float* __restrict__ gout, const float* __restrict__ inv, T* __restrict__ dz, int per) {
  after_previous();
  constexpr int VN = 16 / sizeof(T), UNROLL = THREADS < 128 ? 1 : THREADS < 256 ? 2 : 4;
  const long long row = (long long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (row >= z.rows) return;
  const T* x = static_cast<const T*>(z.at) + z.row(row);
  T* d = dz + row * z.V;
  const long long label = z.labels[row];
  const bool counted = z.counts(label);
  const float g = counted ? coef[row / per] * gout[0] * (inv ? inv[0] : 1.f) : 0.f;
  const int first = blockIdx.y * THREADS + threadIdx.x % THREADS, step = gridDim.y * THREADS;
  const int mis = (int)((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
  const int head = min(z.V, mis ? VN - mis : 0), nvec = (z.V - head) / VN, rest = z.V - nvec * VN;
  if (g == 0.f) {                    // a row that does not count, or whose ratio is held by the clipping
    for (int i = first; i < nvec; i += step) reinterpret_cast<uint4*>(d + head)[i] = make_uint4(0, 0, 0, 0);
    for (int i = first; i < rest; i += step) d[i < head ? i : nvec * VN + i] = from_f32<T>(0.f);
    return;
  }
  const float2 st = stats[row];
  const float M = st.x == -INFINITY ? 0.f : st.x, q = -g / st.y, k = z.k;
  auto grad = [&](float v, int i) { return fmaf(exp2_fast(fmaf(v, k, -M)), q, i == label ? g : 0.f); };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) != 0) {
    for (int i = first; i < z.V; i += step) d[i] = from_f32<T>(grad(to_f32<T>(x[i]), i));
    return;
  }
#pragma unroll UNROLL
  for (int i = first; i < nvec; i += step) {
    const uint4 in = __ldg(reinterpret_cast<const uint4*>(x + head) + i);
    const T* e = reinterpret_cast<const T*>(&in);
    uint4 o;
    T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int j = 0; j < VN; ++j) oe[j] = from_f32<T>(grad(to_f32<T>(e[j]), head + i * VN + j));
    reinterpret_cast<uint4*>(d + head)[i] = o;
  }
  for (int k2 = first; k2 < rest; k2 += step) {
    const int i = k2 < head ? k2 : nvec * VN + k2;
    d[i] = from_f32<T>(grad(to_f32<T>(x[i]), i));
  }
}

}  // namespace pf

using namespace pf;

#define PF_DISPATCH3(dtype, ...)                               \
  switch (dtype) {                                             \
    case PF_F32: { using T = float; __VA_ARGS__; } break;       \
    case PF_F16: { using T = __half; __VA_ARGS__; } break;      \
    case PF_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
    default: return -1;                                        \
  }

namespace {

int logits_of(Logits& z, const void* at, const void* labels, long long N, int T, int V, long long n, long long t,
              long long ignore, float inv_temperature, int dtype) {
  if (dtype != PF_F32 && dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (reinterpret_cast<uintptr_t>(at) % (dtype == PF_F32 ? 4 : 2)) return -2;
  if (N < 0 || T < 0 || V < 1 || N * T > 0x7fffffffll) return -3;
  z = {at, (const long long*)labels, n, t, N * T, ignore, T, V, 1.44269504088896341f * inv_temperature};
  return 0;
}

template <typename Row>
int rows_fwd(const Logits& z, void* stats, const Row& finish, int dtype, int sm_count, cudaStream_t st) {
#define PF_ROWS(THREADS)                                                                                   \
  after(row_fwd_kernel<T, THREADS, Row>, (unsigned)(THREADS < 256 ? (z.rows + 7) / 8 : z.rows),             \
        THREADS < 256 ? 256 : THREADS, 0, st)(z, (float2*)stats, finish)
  PF_DISPATCH3(dtype, {
    if (z.V <= 1024) PF_ROWS(32);
    else if (z.rows <= sm_count && z.V > 8192) PF_ROWS(1024);
    else PF_ROWS(256);
  });
#undef PF_ROWS
  return 0;
}

}  // namespace

// logits [N, T, V] with strides (n, t); labels int64 [N, T]; ref fp32 [N] -> loss, rewards fp32 [N], and for the
// backward stats (two floats a row) and coef fp32 [N].  scratch: doubles [N * T + N].  N is even: the chosen
// sequences, then the rejected ones.
PF_API int pf_preference_fwd(const void* logits, const void* labels, const void* ref, void* loss, void* rewards,
                             void* stats, void* coef, void* scratch, long long N, int T, int V, long long n,
                             long long t, long long ignore_index, float beta, float smoothing, int dtype,
                             int sm_count, void* stream) {
  Logits z;
  const int code = logits_of(z, logits, labels, N, T, V, n, t, ignore_index, 1.f, dtype);
  if (code) return code;
  if (N < 2 || N % 2) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  double* logp = (double*)scratch;
  if (z.rows) {
    const int c = rows_fwd(z, stats, PreferenceRow{logp}, dtype, sm_count, st);
    if (c) return c;
  }
  after(preference_kernel, 1, 1024, 0, st)(logp, (const float*)ref, (float*)rewards, logp + z.rows, (float*)loss,
                                           (float*)coef, (int)N, T, beta, smoothing);
  PF_CHECK_LAUNCH();
  return 0;
}

// actions int64, old and ref (null: none) fp32 [N, T], adv fp32 with strides -> loss, kl, clipped, inv (one over the
// number of rows that count), logp and coef fp32 [N, T], stats two floats a row.  scratch: four floats a row.
PF_API int pf_policy_fwd(const void* logits, const void* actions, const void* old, const void* ref, const void* adv,
                         void* loss, void* kl, void* clipped, void* inv, void* logp, void* coef, void* stats,
                         void* scratch, long long N, int T, int V, long long n, long long t, long long adv_n,
                         long long adv_t, long long ignore_index, float low, float high, float kl_coef,
                         float inv_temperature, int dtype, int sm_count, void* stream) {
  Logits z;
  const int code = logits_of(z, logits, actions, N, T, V, n, t, ignore_index, inv_temperature, dtype);
  if (code) return code;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const PolicyRow finish{(const float*)old, (const float*)ref, (const float*)adv, adv_n, adv_t, low, high, kl_coef,
                         (double)inv_temperature, (float*)logp, (float*)coef, (float4*)scratch};
  if (z.rows) {
    const int c = rows_fwd(z, stats, finish, dtype, sm_count, st);
    if (c) return c;
  }
  after(policy_mean_kernel, 1, 1024, 0, st)((const float4*)scratch, (float*)loss, (float*)kl, (float*)clipped,
                                            (float*)inv, z.rows);
  PF_CHECK_LAUNCH();
  return 0;
}

// dlogits [N, T, V] packed.  coef: one value for `per` rows; gout: the loss's gradient; inv may be null.
PF_API int pf_token_loss_bwd(const void* logits, const void* labels, const void* stats, const void* coef,
                             const void* gout, const void* inv, void* dlogits, long long N, int T, int V,
                             long long n, long long t, long long ignore_index, int per, float inv_temperature,
                             int dtype, int sm_count, void* stream) {
  Logits z;
  const int code = logits_of(z, logits, labels, N, T, V, n, t, ignore_index, inv_temperature, dtype);
  if (code) return code;
  if (z.rows == 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  long long slabs = 8ll * sm_count / z.rows;
  const long long most = (V + 2047) / 2048;
  if (slabs > most) slabs = most;
  if (slabs < 1) slabs = 1;
#define PF_BWD(THREADS, GRID)                                                                             \
  after(row_bwd_kernel<T, THREADS>, GRID, 256, 0, st)(z, (const float2*)stats, (const float*)coef,         \
                                                      (const float*)gout, (const float*)inv, (T*)dlogits, per)
  PF_DISPATCH3(dtype, {
    if (V / (16 / (int)sizeof(T)) <= 64) PF_BWD(32, (unsigned)((z.rows + 7) / 8));
    else PF_BWD(256, dim3((unsigned)z.rows, (unsigned)slabs));
  });
#undef PF_BWD
  PF_CHECK_LAUNCH();
  return 0;
}
