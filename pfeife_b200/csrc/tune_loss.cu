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
// Where |M| is 2^22 or more (a row that a mask of the type's lowest value has left nothing, say), k z - M has lost what
// the softmax is made of, and there may be no M: such a part of a row is passed over once more, with its largest z in
// the place of M, sum 2^(k (z - M)), which has a minus to tell it.
// The backward passes over it again: dz = g (onehot - p) with p = 2^(k z - M) / s and g what the loss has for the
// row's log-probability, so that only M, s and g are kept.
#include "common.cuh"
#include "api.h"

namespace pf {

constexpr double LN2 = 0.693147180559945309417;
// ex2.approx cuts its last bits off: one exponential is low by 5.1e-8 of its value on average over all fractions, and s
// by this part (over 2048 rows of 32000 normal logits, bf16 and fp32 alike; a row's own s is off by 4e-8 around that).
// A single probability hides it in its rounding, a sum over a sequence does not.  The backward divides such values by
// such sums, where it cancels.  What is left, a row on average: below 1e-8 over normal logits; -2.5e-8 for a word that has
// all the probability, since what comes out above 0 is cut off; and k's 24 bits, a temperature that is off by 1.3e-8:
// 1.3e-8 (mean of z - z_label), 8e-8 for words taken at random among logits of 2.5 sigma.  The reference's sum over a
// thousand such rows, some 1e4, is fp32: half a step of it is 5e-7 a row.
constexpr double EXP2_LOW = 3.7e-8;

constexpr float FAR = 4194304.f;

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

// M in powers of two, in its far form too
__device__ __forceinline__ double reference(const Logits& z, float2 stat) {
  return stat.y < 0.f ? (double)z.k * (double)stat.x : (double)stat.x;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(i/32 - 1), which a lane's sum is multiplied by to get from its reference to the integer (exp2f would be as
// low as ex2.approx is); lane 0 has an integer
__constant__ float FRACTION_SCALE[32] = {
    1.000000000f, 0.510948574f, 0.522136891f, 0.533570200f, 0.545253866f, 0.557193371f, 0.569394317f, 0.581862429f,
    0.594603558f, 0.607623680f, 0.620928906f, 0.634525479f, 0.648419777f, 0.662618322f, 0.677127773f, 0.691954941f,
    0.707106781f, 0.722590403f, 0.738413073f, 0.754582214f, 0.771105413f, 0.787990423f, 0.805245166f, 0.822877739f,
    0.840896415f, 0.859309649f, 0.878126080f, 0.897354538f, 0.917004043f, 0.937083817f, 0.957603281f, 0.978572062f};

// (M, s) of two parts of a row, with integers M; a part without a finite element is (-inf, 0), or (-inf, NaN) when it
// holds a NaN, which no maximum shows: the sums are always added, and -inf counts as 0 where it is subtracted.
__device__ __forceinline__ void part_merge(float& m, float& s, float m2, float s2) {
  const float mm = fmaxf(m, m2), sub = mm == -INFINITY ? 0.f : mm;
  s = s * exp2_fast(m - sub) + s2 * exp2_fast(m2 - sub);
  m = mm;
}

// 16 bytes of a row: its largest value, and its values two by two in fp32.  16-bit maxima are taken two at a time
// before anything is widened, as fp32 sums and products are: ten instructions a value became five.  What is left are
// the loads: without its exponentials, 16 a cycle and SM, the pass takes 38 us for 41 (2787 of 4096 rows of 32000
// bf16; 27 at the copy rate).  Batches of 4 vectors and twelve CTAs an SM take 41 too, the next batch in registers
// 42 and several in shared memory 54.
template <typename T> struct Words;
template <> struct Words<float> {
  static constexpr int PAIRS = 2;
  static __device__ __forceinline__ uint4 none() {
    return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
  }
  template <int U> static __device__ __forceinline__ float most(const uint4 (&q)[U]) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(q[u].x), __uint_as_float(q[u].y))),
                fmaxf(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
    return m;
  }
  static __device__ __forceinline__ uint64_t pair(const uint4& q, int j) {
    return f2_pack(__uint_as_float(j ? q.z : q.x), __uint_as_float(j ? q.w : q.y));
  }
};
template <typename T2> __device__ __forceinline__ T2 word_of(const uint4& q, int j) {
  const uint32_t w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
  return *reinterpret_cast<const T2*>(&w);
}
template <typename T2, int U> __device__ __forceinline__ T2 most_words(const uint4 (&q)[U]) {
  T2 m = word_of<T2>(q[0], 0);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = __hmax2(m, word_of<T2>(q[u], j));      // the other one of a NaN
  return m;
}
template <> struct Words<__half> {
  static constexpr int PAIRS = 4;
  static __device__ __forceinline__ uint4 none() {
    return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
  }
  template <int U> static __device__ __forceinline__ float most(const uint4 (&q)[U]) {
    const float2 m = __half22float2(most_words<__half2>(q));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint64_t pair(const uint4& q, int j) {
    const float2 v = __half22float2(word_of<__half2>(q, j));
    return f2_pack(v.x, v.y);
  }
};
template <> struct Words<__nv_bfloat16> {
  static constexpr int PAIRS = 4;
  static __device__ __forceinline__ uint4 none() {
    return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  }
  template <int U> static __device__ __forceinline__ float most(const uint4 (&q)[U]) {
    const float2 m = __bfloat1622float2(most_words<__nv_bfloat162>(q));
    return fmaxf(m.x, m.y);
  }
  static __device__ __forceinline__ uint64_t pair(const uint4& q, int j) {
    const uint32_t w = word_of<uint32_t>(q, j);
    return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};

constexpr int ROW_BATCH = 8;       // vectors that a thread of a CTA takes at a time
constexpr int ROW_THREADS = 128;   // of a part of a row
constexpr int ROW_CTAS = 8;        // such CTAs an SM

template <bool B> struct Flag { static constexpr bool value = B; };

// One pass over each row that counts: M and s of its gridDim.y parts, and the label's logit to `at_label`.  THREADS
// threads a part: CTAs of their own, or 8 or 32 lanes (of whole rows) that share one of 256.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS < 64 ? 256 : THREADS, THREADS == ROW_THREADS ? ROW_CTAS : 1)
row_fwd_kernel(const Logits z, float2* __restrict__ parts, float* __restrict__ at_label) {
  after_previous();
  constexpr int W = THREADS / 32, VN = 16 / sizeof(T), U = W > 1 ? ROW_BATCH : 4;
  constexpr int ROWS = W > 1 ? 1 : 256 / THREADS;
  __shared__ float smax[W > 1 ? W : 1], ssum[W > 1 ? W : 1];
  const long long row = (long long)blockIdx.x * ROWS + (W > 1 ? 0 : threadIdx.x / THREADS);
  if (row >= z.rows) return;
  const int tid = threadIdx.x % THREADS;
  const long long label = z.labels[row];
  if (!z.counts(label)) return;
  const T* x = static_cast<const T*>(z.at) + z.row(row);
  const int part = W > 1 ? blockIdx.y : 0, n_parts = W > 1 ? gridDim.y : 1;
  const float mine = tid == 0 && part == 0 ? to_f32<T>(x[label]) : 0.f;
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(z.V, mis ? VN - mis : 0), nvec = (z.V - head) / VN;
  const float k = z.k, fraction = (threadIdx.x & 31) * (1.f / 32);
  float m = -FAR, s = 0.f;                           // a reference below would have sums that are infinite
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const uint64_t k2 = f2_pack(k, k);
  // A batch of vectors from i0 on, all before `end` or some.
  auto add = [&](auto whole, int i0, int end) {
    constexpr bool ALL = decltype(whole)::value;
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {                    // -inf behind the end, which adds nothing
      if (!ALL) q[u] = Words<T>::none();
      if (ALL || i0 + u * THREADS < end) q[u] = __ldg(xv + i0 + u * THREADS);
    }
    // a NaN does not move the maximum but reaches the sum below
    const float mm = fmaxf(m, ceilf(Words<T>::most(q) * k) + fraction);
    if (mm > m) s *= exp2_fast(m - mm);
    const uint64_t minus2 = f2_pack(-mm, -mm);
    uint64_t sums[2] = {0, 0};                       // two zeros each
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ALL || i0 + u * THREADS < end)
#pragma unroll
        for (int j = 0; j < Words<T>::PAIRS; ++j) {
          float a, b;
          f2_unpack(fma2(Words<T>::pair(q[u], j), k2, minus2), a, b);
          sums[j & 1] = add2(sums[j & 1], f2_pack(exp2_fast(a), exp2_fast(b)));
        }
    float a, b;
    f2_unpack(add2(sums[0], sums[1]), a, b);
    s += a + b;
    m = mm;
  };
  const int begin = (int)((long long)nvec * part / n_parts), end = (int)((long long)nvec * (part + 1) / n_parts);
  int i0 = begin + tid;
  for (; i0 + (U - 1) * THREADS < end; i0 += U * THREADS) add(Flag<true>{}, i0, end);
  if (i0 < end) add(Flag<false>{}, i0, end);
  // the elements before the first and after the last vector (at most 2 (VN - 1))
  for (int i = tid; part == 0 && i < z.V - nvec * VN; i += THREADS) {
    const float v = to_f32<T>(x[i < head ? i : nvec * VN + i]);
    const float mm = fmaxf(m, ceilf(v * k) + fraction);
    s = s * exp2_fast(m - mm) + exp2_fast(fmaf(v, k, -mm));
    m = mm;
  }
  {                                                  // to the integer above, by the lane's own power where it is that
    const float whole = ceilf(m), down = m - whole;
    s *= down == fraction - 1.f ? FRACTION_SCALE[threadIdx.x & 31] : exp2f(down);
    m = whole;
  }
  // the lanes of a row; others of the warp may have left, or have more to add
  const unsigned lanes =
      THREADS >= 32 ? 0xffffffffu : ((1u << (THREADS & 31)) - 1) << (threadIdx.x & 31 & ~(THREADS - 1));
#pragma unroll
  for (int o = (THREADS < 32 ? THREADS : 32) / 2; o > 0; o >>= 1)
    part_merge(m, s, __shfl_xor_sync(lanes, m, o), __shfl_xor_sync(lanes, s, o));
  if constexpr (W > 1) {
    const int w = tid >> 5, l = tid & 31;
    if (l == 0) { smax[w] = m; ssum[w] = s; }
    __syncthreads();
    m = smax[l % W];
    s = ssum[l % W];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1)
      part_merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  }
  if (!(fabsf(m) < FAR)) {                           // all threads of the part
    const int from = head + begin * VN, to = head + end * VN, most = part == 0 ? z.V - nvec * VN : 0;
    auto each = [&](auto f) {
      for (int i = from + tid; i < to; i += THREADS) f(to_f32<T>(x[i]));
      for (int i = tid; i < most; i += THREADS) f(to_f32<T>(x[i < head ? i : nvec * VN + i]));
    };
    float top = -INFINITY, sum = 0.f;
    each([&](float v) { top = fmaxf(top, v); });
#pragma unroll
    for (int o = (THREADS < 32 ? THREADS : 32) / 2; o > 0; o >>= 1)
      top = fmaxf(top, __shfl_xor_sync(lanes, top, o));
    if (W > 1) {
      __syncthreads();                               // both have been read
      if ((tid & 31) == 0) smax[tid >> 5] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, smax[w]);
    }
    m = top;                                         // -inf: a part without a finite element, its sum 0 or NaN
    if (top > -INFINITY) {
      each([&](float v) { sum += exp2_fast((v - top) * k); });
#pragma unroll
      for (int o = (THREADS < 32 ? THREADS : 32) / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
      if (W > 1) {
        if ((tid & 31) == 0) ssum[tid >> 5] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += ssum[w];
      }
      s = -sum;
    }
  }
  if (tid == 0) {
    parts[row * n_parts + part] = make_float2(m, s);
    if (part == 0) at_label[row] = mine;
  }
}

// What follows is one launch: a cluster of CTAs shares the rows, leaves sums in `scratch`, and the first CTA joins
// them in their order.  (A thread of each row's CTA doing its row's part kept that CTA: 48 us for 42 with the pass.)
// Beyond some thousand rows the 64-bit arithmetic of a row each takes longer than another launch: CTAs that are no
// cluster, and one that joins (65536 rows of 256: 38 -> 18 us with the pass).
constexpr int TAIL_THREADS = 512, TAIL_CTAS = 8, TAIL_ONE = 512, TAIL_MANY = 8192, TAIL_MOST = 296;
enum { WHOLE, SHARE, JOIN };       // one launch, or the first and the second of two

// What the forward's pass over the rows has left: joined for the backward, and a row's log-probability.
struct Rows {
  const float2* parts;             // [rows][n_parts]
  const float* at_label;
  float2* stats;                   // [rows]
  int n_parts;
  __device__ __forceinline__ float2 join(const Logits& z, long long r) const {
    float2 v = parts[r * n_parts];
    for (int i = 1; i < n_parts; ++i) {
      const float2 w = parts[r * n_parts + i];
      if (!(v.y < 0.f) && !(w.y < 0.f)) {
        part_merge(v.x, v.y, w.x, w.y);
      } else {                                       // the sum with the greater reference takes the other one
        const double d = reference(z, w) - reference(z, v);
        const float2 less = d > 0.0 ? v : w;
        if (d > 0.0) v = w;
        v.y += copysignf(exp2f(-fabsf((float)d)), v.y) * fabsf(less.y);
      }
    }
    return v;
  }
};
__device__ __forceinline__ double log_prob(const Logits& z, float2 stat, float at_label) {
  // the far form's largest exponentials are 2^0, which is exact
  const double low = stat.y < 0.f ? 0.0 : EXP2_LOW;
  const double l = LN2 * ((double)at_label * (double)z.k - reference(z, stat)) - log(fabs((double)stat.y)) - low;
  return l > 0.0 ? 0.0 : l;          // a row of one word by 1e-7; a NaN stays
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct PolicyArgs {
  const float *old, *ref, *adv;    // ref null: no reference
  long long adv_n, adv_t;          // strides of the advantages
  double low, high, kl, inv_temperature;
  float *logp, *coef;              // coef: of the row's own term, before the mean
  float *loss, *mean_kl, *clipped, *inv;
};
template <int STEP>
__global__ void __launch_bounds__(TAIL_THREADS)
policy_tail_kernel(const Logits z, const Rows rows, const PolicyArgs p, double* __restrict__ scratch, int ctas) {
  after_previous();
  __shared__ double part[4][TAIL_THREADS / 32];
  double sums[4] = {};                               // terms, KL, clipped, counted
  for (long long r = (long long)blockIdx.x * TAIL_THREADS + threadIdx.x; STEP != JOIN && r < z.rows;
       r += (long long)ctas * TAIL_THREADS) {
    // all at once, whether the row counts (its statistics are written only then) or not
    const long long n = r / z.T, label = z.labels[r];
    const float2 stat = rows.join(z, r);
    const float logit = rows.at_label[r], old = p.old[r], ref = p.ref ? p.ref[r] : 0.f;
    const float adv = p.adv[n * p.adv_n + (r - n * z.T) * p.adv_t];
    if (!z.counts(label)) {
      p.logp[r] = p.coef[r] = 0.f;
      continue;
    }
    rows.stats[r] = stat;
    const double lp = log_prob(z, stat, logit), a = adv, ratio = exp(lp - (double)old);
    const double lo = 1.0 - p.low, hi = 1.0 + p.high;
    const double free = ratio * a, held = fmin(fmax(ratio, lo), hi) * a;
    const bool clipped = free > held;
    double term = clipped ? -held : -free, c = clipped ? 0.0 : -free, each = 0.0;
    if (p.ref) {
      const double d = (double)ref - lp, e = expm1(d);
      each = e == INFINITY ? e : e - d;
      if (p.kl != 0.0) {                             // 0 x inf is not 0
        term += p.kl * each;
        c -= p.kl * e;
      }
    }
    p.logp[r] = (float)lp;
    p.coef[r] = (float)(c * p.inv_temperature);
    sums[0] += term; sums[1] += each; sums[2] += clipped ? 1.0 : 0.0; sums[3] += 1.0;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double total = 0.0;                                // threads 0 to 3: of the CTA, then of all
  if (STEP != JOIN) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[i] = warp_sum64(sums[i]);
      if (lane == 0) part[i][warp] = sums[i];
    }
    __syncthreads();
    if (threadIdx.x < 4) {
#pragma unroll
      for (int w = 0; w < TAIL_THREADS / 32; ++w) total += part[threadIdx.x][w];
      if (ctas > 1) scratch[blockIdx.x * 4 + threadIdx.x] = total;
    }
    __syncwarp();
    if (STEP == SHARE) return;
    if (ctas > 1) cluster_sync();
  }
  if (blockIdx.x > 0 || warp > 0) return;
  if (ctas > 1) {                                    // eight lanes for each sum
    total = 0.0;
    for (int c = lane >> 2; c < ctas; c += 8) total += __ldcg(scratch + c * 4 + (lane & 3));
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  const double count = __shfl_sync(0xffffffffu, total, 3), one = 1.0 / (count > 0.0 ? count : 1.0);
  float* const to[4] = {p.loss, p.mean_kl, p.clipped, p.inv};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane == i) *to[i] = (float)(i == 3 ? one : total * one);
}

// Rewards of the sequences, the mean loss over the pairs and what a sequence's log-probability gets of it.  Warps
// share the sequences; where there are more warps than sequences, several sum parts of one.
template <int STEP>
__global__ void __launch_bounds__(TAIL_THREADS)
preference_tail_kernel(const Logits z, const Rows rows, const float* __restrict__ ref, float* __restrict__ rewards,
                       float* __restrict__ loss, float* __restrict__ coef, double* __restrict__ scratch, int N,
                       double beta, double smoothing, int ctas) {
  after_previous();
  const int warps = ctas * (TAIL_THREADS / 32), warp = blockIdx.x * (TAIL_THREADS / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, parts = max(1, min(warps / N, (z.T + 31) / 32)), items = N * parts;
  for (int i = warp; STEP != JOIN && i < items; i += warps) {
    const int n = i / parts, part = i - n * parts;
    double t = 0.0;
    for (long long j = part * 32 + lane; j < z.T; j += parts * 32) {
      const long long r = (long long)n * z.T + j, label = z.labels[r];
      const float2 stat = rows.join(z, r);           // written where the row counts
      const float logit = rows.at_label[r];
      if (z.counts(label)) {
        rows.stats[r] = stat;
        t += log_prob(z, stat, logit);
      }
    }
    t = warp_sum64(t);
    if (lane == 0) scratch[i] = t;
  }
  if (STEP == SHARE) return;
  __syncwarp();
  if (STEP == WHOLE) {
    if (ctas > 1) cluster_sync();
    else __syncthreads();
  }
  if (blockIdx.x > 0) return;
  __shared__ double shared[TAIL_THREADS / 32];
  auto reward = [&](int n) {
    double t = 0.0;
    for (int i = 0; i < parts; ++i) t += __ldcg(scratch + n * parts + i);
    return beta * (t - (double)ref[n]);
  };
  const int P = N / 2;
  double total = 0.0;
  for (int p = threadIdx.x; p < P; p += TAIL_THREADS) {
    const double chosen = reward(p), rejected = reward(P + p);
    rewards[p] = (float)chosen;
    rewards[P + p] = (float)rejected;
    const double m = chosen - rejected, e = exp(-fabs(m)), near = log1p(e);
    // -log sig(m) and -log sig(-m), sig(-m) and sig(m), none of which overflows
    const double lp = near + fmax(-m, 0.0), lm = near + fmax(m, 0.0);
    const double big = 1.0 / (1.0 + e), small = e / (1.0 + e);
    total += smoothing < 1.0 ? (1.0 - smoothing) * lp : 0.0;      // 0 x inf is not 0
    total += smoothing > 0.0 ? smoothing * lm : 0.0;
    const double c = -beta / P * ((1.0 - smoothing) * (m > 0.0 ? small : big) - smoothing * (m > 0.0 ? big : small));
    coef[p] = (float)c;
    coef[P + p] = (float)-c;
  }
  total = warp_sum64(total);
  if (lane == 0) shared[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int w = 0; w < TAIL_THREADS / 32; ++w) total += shared[w];
    *loss = (float)(total / P);
  }
}

// dz = g (onehot - p), g = coef[row / per] * gout * inv (inv null: 1).  THREADS threads a row; where they are whole
// CTAs the grid is (row, slab of the row).
template <typename T, int THREADS>
__global__ void __launch_bounds__(256)
row_bwd_kernel(const Logits z, const float2* __restrict__ stats, const float* __restrict__ coef,
               const float* __restrict__ gout, const float* __restrict__ inv, T* __restrict__ dz, int per,
               long long dz_row) {
  after_previous();
  constexpr int VN = 16 / sizeof(T), UNROLL = THREADS < 32 ? 2 : 4;
  // the last rows first: the forward has read them last, and what L2 still holds of them is read from there
  const long long row = z.rows - 1 - ((long long)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS);
  if (row < 0) return;
  const T* x = static_cast<const T*>(z.at) + z.row(row);
  T* d = dz + row * dz_row;
  const long long label = z.labels[row];
  const bool counted = z.counts(label);
  const float g = counted ? coef[row / per] * gout[0] * (inv ? inv[0] : 1.f) : 0.f;
  const int first = blockIdx.y * THREADS + threadIdx.x % THREADS, step = gridDim.y * THREADS;
  const int mis = (int)((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
  const int head = min(z.V, mis ? VN - mis : 0), nvec = (z.V - head) / VN, rest = z.V - nvec * VN;
  if (g == 0.f) {                    // a row that does not count, or whose ratio is held by the clipping
    for (int i = first; i < nvec; i += step) __stcs(reinterpret_cast<uint4*>(d + head) + i, make_uint4(0, 0, 0, 0));
    for (int i = first; i < rest; i += step) d[i < head ? i : nvec * VN + i] = from_f32<T>(0.f);
    return;
  }
  const float2 st = stats[row];
  const float M = st.x == -INFINITY ? 0.f : st.x, q = -g / fabsf(st.y), k = z.k;
  if (st.y < 0.f) {
    for (int i = first; i < z.V; i += step)
      d[i] = from_f32<T>(fmaf(exp2_fast((to_f32<T>(x[i]) - M) * k), q, i == label ? g : 0.f));
    return;
  }
  auto grad = [&](float v, int i) { return fmaf(exp2_fast(fmaf(v, k, -M)), q, i == label ? g : 0.f); };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) != 0) {
    for (int i = first; i < z.V; i += step) d[i] = from_f32<T>(grad(to_f32<T>(x[i]), i));
    return;
  }
#pragma unroll UNROLL
  for (int i = first; i < nvec; i += step) {
    const uint4 in = __ldcs(reinterpret_cast<const uint4*>(x + head) + i);
    const T* e = reinterpret_cast<const T*>(&in);
    uint4 o;
    T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int j = 0; j < VN; ++j) oe[j] = from_f32<T>(grad(to_f32<T>(e[j]), head + i * VN + j));
    __stcs(reinterpret_cast<uint4*>(d + head) + i, o);
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
              long long ignore, double inv_temperature, int dtype) {
  if (dtype != PF_F32 && dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (reinterpret_cast<uintptr_t>(at) % (dtype == PF_F32 ? 4 : 2)) return -2;
  if (N < 0 || T < 0 || V < 1 || N * T > 0x7fffffffll) return -3;
  z = {at, (const long long*)labels, n, t, N * T, ignore, T, V, (float)(1.44269504088896341 * inv_temperature)};
  return 0;
}

// Lanes of a row in the forward, 0: CTAs.  What a short row costs beside its values is the same for all lanes that
// it keeps, so many short rows get few (microseconds with 8, 32 lanes and CTAs of 128, with what follows, bf16:
// 65536 rows of 256 18, 24 and 53; 16384 of 1000 16, 18 and 23; 16384 of 1500 to 2049 with 32 lanes 23 to 25 and
// with CTAs 57 to 59; 16384 of 8192 54 and 69; 4096 of 16384 36 and 35).  Few rows take a warp each, or CTAs.
int row_lanes(long long rows, int V, int sm_count) {
  if (V <= 1024) return rows >= 32ll * sm_count ? 8 : 32;
  return V <= 8192 && rows >= 16ll * sm_count ? 32 : 0;
}
// The same for the backward, by the vectors of a row (65536 rows of 256 bf16: 17 us with 8 lanes, 29 with 32; 16384
// of 1500 24 with 32 lanes, 43 with CTAs of 256; 8192 of 4096 31 either way; 64 of 256 2.7 with 8 lanes, 2.1 with 32).
int back_lanes(long long rows, int nvec, int sm_count) {
  if (nvec <= 64) return rows >= 32ll * sm_count ? 8 : 32;
  return nvec <= 256 && rows >= 4ll * sm_count ? 32 : 0;
}

// Parts of a row: enough for the CTAs that the SMs hold, but no more than batches, so that a part has a batch or, since
// they are equal, somewhat less (16 rows of 32000 fp32: 7.7 us in one part, 6.1 in 8; four times as many are slower by
// 1 to 3 us where rows fill the SMs as they are).
int row_parts(long long rows, int V, int dtype, int sm_count) {
  const int batch = ROW_THREADS * ROW_BATCH * (dtype == PF_F32 ? 4 : 8);
  if (rows == 0 || row_lanes(rows, V, sm_count)) return 1;
  long long n = ROW_CTAS * (long long)sm_count / rows;
  const int most = (V + batch - 1) / batch;
  if (n > most) n = most;
  return n < 1 ? 1 : (int)n;
}

// CTAs that share the rows behind the pass.
int tail_ctas(long long rows) {
  if (rows <= TAIL_ONE) return 1;
  if (rows <= TAIL_MANY) return TAIL_CTAS;
  const long long n = (rows + TAIL_THREADS - 1) / TAIL_THREADS;
  return n < TAIL_MOST ? (int)n : TAIL_MOST;
}
// Scratch of a forward: the cluster's sums (a preference: of up to as many parts of sequences as it has warps), the
// parts of the rows and the logits at the labels.
struct Scratch {
  double* sums;
  float2* parts;
  float* at_label;
  long long doubles;
  Scratch(void* at, long long N, long long rows, int n_parts) {
    const long long warps = (long long)tail_ctas(rows) * (TAIL_THREADS / 32), n = N > warps ? N : warps;
    sums = (double*)at;
    parts = (float2*)(sums + n);
    at_label = (float*)(parts + rows * n_parts);
    doubles = n + rows * n_parts + (rows + 1) / 2;
  }
};

int rows_fwd(const Logits& z, const Scratch& s, int n_parts, int dtype, int sm_count, cudaStream_t st) {
  if (z.rows == 0) return 0;
  const int lanes = row_lanes(z.rows, z.V, sm_count);
  const dim3 grid(lanes == 0 ? (unsigned)z.rows : (unsigned)((z.rows * lanes + 255) / 256), n_parts);
  PF_DISPATCH3(dtype, {
    if (lanes == 8) after(row_fwd_kernel<T, 8>, grid, 256, 0, st)(z, s.parts, s.at_label);
    else if (lanes == 32) after(row_fwd_kernel<T, 32>, grid, 256, 0, st)(z, s.parts, s.at_label);
    else after(row_fwd_kernel<T, ROW_THREADS>, grid, ROW_THREADS, 0, st)(z, s.parts, s.at_label);
  });
  return 0;
}

// The launches behind the rows: `whole`, one CTA or a cluster, or `share` and `join`.
template <typename... P, typename... A>
void tail(void (*whole)(P...), void (*share)(P...), void (*join)(P...), long long rows, cudaStream_t st,
          const A&... args) {
  const int ctas = tail_ctas(rows);
  if (rows > TAIL_MANY) {
    after(share, ctas, TAIL_THREADS, 0, st)(args..., ctas);
    after(join, 1, TAIL_THREADS, 0, st)(args..., ctas);
    return;
  }
  auto l = after(whole, ctas, TAIL_THREADS, 0, st);
  cudaLaunchAttribute cluster;
  if (ctas > 1) {
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = ctas;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    l.cfg.attrs = &cluster;
    l.cfg.numAttrs = 1;
  }
  l(args..., ctas);
}

}  // namespace

// Doubles of scratch that a forward needs.
PF_API int pf_token_loss_scratch(long long N, int T, int V, int dtype, int sm_count) {
  const long long rows = N * T, n = Scratch(nullptr, N, rows, row_parts(rows, V, dtype, sm_count)).doubles;
  return n > 0x7fffffffll ? -3 : (int)n;
}

// logits [N, T, V] with strides (n, t); labels int64 [N, T]; ref fp32 [N] -> loss, rewards fp32 [N], and for the
// backward stats (two floats a row) and coef fp32 [N].  N is even: the chosen sequences, then the rejected ones.
PF_API int pf_preference_fwd(const void* logits, const void* labels, const void* ref, void* loss, void* rewards,
                             void* stats, void* coef, void* scratch, long long N, int T, int V, long long n,
                             long long t, long long ignore_index, double beta, double smoothing, int dtype,
                             int sm_count, void* stream) {
  Logits z;
  int code = logits_of(z, logits, labels, N, T, V, n, t, ignore_index, 1.0, dtype);
  if (code) return code;
  if (N < 2 || N % 2) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int n_parts = row_parts(z.rows, V, dtype, sm_count);
  const Scratch s(scratch, N, z.rows, n_parts);
  if ((code = rows_fwd(z, s, n_parts, dtype, sm_count, st))) return code;
  const Rows rows{s.parts, s.at_label, (float2*)stats, n_parts};
  tail(preference_tail_kernel<WHOLE>, preference_tail_kernel<SHARE>, preference_tail_kernel<JOIN>, z.rows, st, z, rows,
       (const float*)ref, (float*)rewards, (float*)loss, (float*)coef, s.sums, (int)N, beta, smoothing);
  PF_CHECK_LAUNCH();
  return 0;
}

// actions int64, old and ref (null: none) fp32 [N, T], adv fp32 with strides -> loss, kl, clipped, inv (one over the
// number of rows that count), logp and coef fp32 [N, T], stats two floats a row.
PF_API int pf_policy_fwd(const void* logits, const void* actions, const void* old, const void* ref, const void* adv,
                         void* loss, void* kl, void* clipped, void* inv, void* logp, void* coef, void* stats,
                         void* scratch, long long N, int T, int V, long long n, long long t, long long adv_n,
                         long long adv_t, long long ignore_index, double low, double high, double kl_coef,
                         double inv_temperature, int dtype, int sm_count, void* stream) {
  Logits z;
  int code = logits_of(z, logits, actions, N, T, V, n, t, ignore_index, inv_temperature, dtype);
  if (code) return code;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const PolicyArgs p{(const float*)old, (const float*)ref, (const float*)adv, adv_n, adv_t, low, high, kl_coef,
                     inv_temperature, (float*)logp, (float*)coef, (float*)loss, (float*)kl, (float*)clipped,
                     (float*)inv};
  const int n_parts = row_parts(z.rows, V, dtype, sm_count);
  const Scratch s(scratch, N, z.rows, n_parts);
  if ((code = rows_fwd(z, s, n_parts, dtype, sm_count, st))) return code;
  const Rows rows{s.parts, s.at_label, (float2*)stats, n_parts};
  tail(policy_tail_kernel<WHOLE>, policy_tail_kernel<SHARE>, policy_tail_kernel<JOIN>, z.rows, st, z, rows, p, s.sums);
  PF_CHECK_LAUNCH();
  return 0;
}

// dlogits: rows of V values, dlogits_row apart.  coef: one value for `per` rows; gout: the loss's gradient; inv may
// be null.  Rows that lie to 16 bytes as the logits' do are written by vectors, others element by element.
PF_API int pf_token_loss_bwd(const void* logits, const void* labels, const void* stats, const void* coef,
                             const void* gout, const void* inv, void* dlogits, long long dlogits_row,
                             long long N, int T, int V, long long n, long long t, long long ignore_index, int per,
                             double inv_temperature, int dtype, int sm_count, void* stream) {
  Logits z;
  const int code = logits_of(z, logits, labels, N, T, V, n, t, ignore_index, inv_temperature, dtype);
  if (code) return code;
  if (z.rows == 0) return 0;
  if (dlogits_row < V) return -3;
  if (reinterpret_cast<uintptr_t>(dlogits) % (dtype == PF_F32 ? 4 : 2)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  long long slabs = 8ll * sm_count / z.rows;
  const long long most = (V + 2047) / 2048;
  if (slabs > most) slabs = most;
  if (slabs < 1) slabs = 1;
#define PF_BWD(THREADS, GRID)                                                                             \
  after(row_bwd_kernel<T, THREADS>, GRID, 256, 0, st)(z, (const float2*)stats, (const float*)coef,         \
                                                      (const float*)gout, (const float*)inv, (T*)dlogits, per,  \
                                                      dlogits_row)
  PF_DISPATCH3(dtype, {
    const int lanes = back_lanes(z.rows, V / (16 / (int)sizeof(T)), sm_count);
    if (lanes == 8) PF_BWD(8, (unsigned)((z.rows + 31) / 32));
    else if (lanes == 32) PF_BWD(32, (unsigned)((z.rows + 7) / 8));
    else PF_BWD(256, dim3((unsigned)z.rows, (unsigned)slabs));
  });
#undef PF_BWD
  PF_CHECK_LAUNCH();
  return 0;
}
