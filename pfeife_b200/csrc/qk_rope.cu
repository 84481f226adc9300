// Rotary positions of every layout, alone or behind an RMS norm of each head, over queries and keys (and the
// values of a fused projection, which are copied), forward and backward.
//
// A head of D values has R of them in pairs: (i, i + R/2), or (2i, 2i + 1) when interleaved.  A pair turns by the
// angle of its position and of its frequency i: (a, b) -> (a c - b s, b c + a s); values R..D stay.  In front of
// that the norm multiplies by r w, r = (mean x^2 + eps)^-1/2.  With g the gradient turned back (the transposed
// rotation), xh = x r:  dx = r (g w - xh mean(g w xh)),  dw = sum over tokens and heads of g xh.
// r is computed again in the backward, which reads x anyway.
//
// A head lies across a group of lanes, a power of two of them.  A lane owns slots of two halves of VW values, VW i
// and VW i + R/2 on in the pairs, so that a rotation needs no other lane and the norm one sum over the group.
// Cosines and sines are loaded once per token and stay in registers, as does the gain.
#include "common.cuh"
#include "api.h"

namespace pf {

constexpr int MAX_HEAD_DIM = 256;
constexpr int BACK_CTAS = 2;         // of the backward behind a norm, that an SM holds
constexpr int RING_BYTES = 196608;   // of an SM's shared memory, through which heads come

struct HeadsView {                 // [B, S, heads, D] in any order of memory with D innermost
  char* at;
  long long b, s, h;               // strides in elements
};
struct HeadsPart {
  HeadsView x, y, g;               // forward: x -> y; backward: x and the gradient g -> y
  const float* w;                  // gain of the norm, or null
  float* dw;                       // backward: partial sums, one row [D] for each CTA of the call
  int heads, turn;                 // turn 0: the values of a projection, which are copied
  int cta0, ctas, per;             // the CTAs of this part, and the heads that a group of lanes takes
};
struct HeadsArgs {
  HeadsPart part[3];
  const float *cos_t, *sin_t;      // [rows, R/2]
  const long long* pos;            // row of the tables for each token, or null: the token's place
  long long pos_b, pos_s, rows;
  int S, D, R, lg;
  unsigned tokens;
  float eps, inv_D;
};

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = unsigned short; };

// two values of a pair of registers, rounded to 16 bits in one operation
template <typename T> __device__ __forceinline__ void narrow2(T* to, float a, float b) { to[0] = a; to[1] = b; }
template <> __device__ __forceinline__ void narrow2(__half* to, float a, float b) {
  *reinterpret_cast<__half2*>(to) = __floats2half2_rn(a, b);
}
template <> __device__ __forceinline__ void narrow2(__nv_bfloat16* to, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(a, b);
}

// Where a lane's slots lie in a head, and by how much they turn.  In registers the values of a slot are VW pairs
// (x, y) that turn together, x and y each packed two by two, whatever their order in memory.
// FIT: a head fills the lanes and turns as a whole, so that nothing has to be asked for.
template <typename T, int VW, int NS, bool INTER, bool FIT>
struct Slots {
  static constexpr int P = (VW + 1) / 2;             // packed registers of the x and of the y of a slot
  struct Values { uint64_t x[P], y[P]; };
  using raw = typename Raw<VW * sizeof(T)>::type;
  int a[NS], b[NS];                // first values of both halves, -1 where there is none
  int f[NS], g[NS];                // first frequencies of both halves of the cosines
  bool turns_[NS];
  __device__ __forceinline__ bool has_a(int n) const { return FIT || a[n] >= 0; }
  __device__ __forceinline__ bool has_b(int n) const { return FIT || b[n] >= 0; }
  __device__ __forceinline__ bool turns(int n) const { return FIT || turns_[n]; }

  // Both halves lie apart even where pairs lie side by side or do not turn, so that the lanes of a group read and
  // write whole sectors together (32 bytes a lane, 16 at a time: 41 us for 26, [1, 32768, 8, 128] interleaved).
  __device__ __forceinline__ Slots(const HeadsArgs& p, int lane) {
    const int pairs = p.R / (2 * VW), apart = ((p.D - p.R) / VW + 1) / 2;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int v = lane + (n << p.lg), w = v - pairs;
      turns_[n] = FIT || v < pairs;
      constexpr bool single = VW == 1 && INTER;       // a half is no pair
      a[n] = !turns_[n] ? p.R + VW * w : single ? 2 * v : VW * v;
      b[n] = !turns_[n] ? a[n] + VW * apart : single ? 2 * v + 1 : VW * v + p.R / 2;
      f[n] = INTER && !single ? VW / 2 * v : VW * v;
      g[n] = INTER ? p.R / 4 + VW / 2 * v : VW * v + VW / 2;
      if (!turns_[n]) {
        if (w >= apart) a[n] = b[n] = -1;
        if (b[n] >= p.D) b[n] = -1;
      }
    }
  }
  __device__ __forceinline__ void load(const T* x, raw (&r)[NS][2]) const {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      r[n][0] = r[n][1] = raw{};
      if (has_a(n)) r[n][0] = *reinterpret_cast<const raw*>(x + a[n]);
      if (has_b(n)) r[n][1] = *reinterpret_cast<const raw*>(x + b[n]);
    }
  }
  // the pairs of two halves: (a, b) of equal places, or neighbours
  template <typename E>
  static __device__ __forceinline__ Values pairs_of(const E* a, const E* b) {
    float x[2 * P] = {}, y[2 * P] = {};
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      const E* h = j < VW / 2 ? a : b;
      const int at = j < VW / 2 ? 2 * j : 2 * j - VW;
      x[j] = to_f32<E>(INTER && VW > 1 ? h[at] : a[j]);
      y[j] = to_f32<E>(INTER && VW > 1 ? h[at + 1] : b[j]);
    }
    Values v;
#pragma unroll
    for (int j = 0; j < P; ++j) { v.x[j] = f2_pack(x[2 * j], x[2 * j + 1]); v.y[j] = f2_pack(y[2 * j], y[2 * j + 1]); }
    return v;
  }
  static __device__ __forceinline__ Values widen(const raw (&r)[2]) {
    return pairs_of(reinterpret_cast<const T*>(&r[0]), reinterpret_cast<const T*>(&r[1]));
  }
  __device__ __forceinline__ void store(T* to, int n, const Values& v) const {
    float x[2 * P], y[2 * P];
#pragma unroll
    for (int j = 0; j < P; ++j) { f2_unpack(v.x[j], x[2 * j], x[2 * j + 1]); f2_unpack(v.y[j], y[2 * j], y[2 * j + 1]); }
    raw r[2];
    T* a = reinterpret_cast<T*>(&r[0]);
    T* b = reinterpret_cast<T*>(&r[1]);
    if constexpr (VW == 1) {
      *a = from_f32<T>(x[0]);
      *b = from_f32<T>(y[0]);
    } else {
#pragma unroll
      for (int j = 0; j < VW; j += 2) {
        if constexpr (INTER) {
          narrow2(a + j, x[j / 2], y[j / 2]);
          narrow2(b + j, x[VW / 2 + j / 2], y[VW / 2 + j / 2]);
        } else {
          narrow2(a + j, x[j], x[j + 1]);
          narrow2(b + j, y[j], y[j + 1]);
        }
      }
    }
    put(to, n, r);
  }
  __device__ __forceinline__ void put(T* y, int n, const raw (&r)[2]) const {
    if (has_a(n)) *reinterpret_cast<raw*>(y + a[n]) = r[0];
    if (has_b(n)) *reinterpret_cast<raw*>(y + b[n]) = r[1];
  }
  // gain of the norm at the slots' values
  __device__ __forceinline__ void gains(const float* w, Values (&v)[NS]) const {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      float first[VW], second[VW];
      take<VW>(w, a[n], first, 0.f);
      take<VW>(w, b[n], second, 0.f);
      v[n] = pairs_of(first, second);
    }
  }
  // K floats, or `none` where at is negative
  template <int K>
  static __device__ __forceinline__ void take(const float* t, long long at, float* v, float none) {
    if constexpr (K % 4 == 0) {
#pragma unroll
      for (int j = 0; j < K; j += 4) {
        const float4 q = at >= 0 ? __ldg(reinterpret_cast<const float4*>(t + at + j)) : make_float4(none, none, none, none);
        v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
      }
    } else if constexpr (VW >= 4) {
      const float2 q = at >= 0 ? __ldg(reinterpret_cast<const float2*>(t + at)) : make_float2(none, none);
      v[0] = q.x; v[1] = q.y;
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) v[j] = at >= 0 ? __ldg(t + at + j) : none;
    }
  }
  // Cosines and sines at a token's row of the tables; NaN for a row that they do not have, which no kernel can
  // refuse without the host waiting for it.
  struct Angles { float c[2 * P], s[2 * P]; };
  __device__ __forceinline__ void angles(const HeadsArgs& p, long long row, Angles (&to)[NS]) const {
    const bool there = row >= 0 && row < p.rows;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (!turns(n)) continue;
      const long long at = row * (p.R / 2), first = there ? at + f[n] : -1, second = there ? at + g[n] : -1;
      constexpr int K = VW > 1 ? VW / 2 : 1;
      take<K>(p.cos_t, first, to[n].c, NAN);
      take<K>(p.sin_t, first, to[n].s, NAN);
      if constexpr (VW > 1) {
        take<K>(p.cos_t, second, to[n].c + K, NAN);
        take<K>(p.sin_t, second, to[n].s + K, NAN);
      }
    }
  }
  // (x, y) -> (x c - y s, y c + x s), or with -s; the subtraction is not packed: packed operations do not negate
  template <bool INVERSE>
  static __device__ __forceinline__ void turn(const Angles& by, Values& v) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const uint64_t c = f2_pack(by.c[2 * j], by.c[2 * j + 1]), s = f2_pack(by.s[2 * j], by.s[2 * j + 1]);
      const uint64_t x = v.x[j], y = v.y[j], plus = fma2(INVERSE ? y : x, s, mul2(INVERSE ? x : y, c));
      float a0, a1, o0, o1;
      f2_unpack(mul2(INVERSE ? y : x, c), a0, a1);
      f2_unpack(INVERSE ? x : y, o0, o1);
      const uint64_t minus = f2_pack(fmaf(-o0, by.s[2 * j], a0), fmaf(-o1, by.s[2 * j + 1], a1));
      v.x[j] = INVERSE ? plus : minus;
      v.y[j] = INVERSE ? minus : plus;
    }
  }
};
__device__ __forceinline__ float halves(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// sums of U values over the lanes of a group, whose other groups of the warp may be done
template <int U>
__device__ __forceinline__ void group_sum(float (&v)[U], int lg, unsigned lanes) {
  for (int o = (1 << lg) >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(lanes, v[u], o);
}

// Where a group is in its walk over the heads of a part, token by token, and their places in one tensor or two.
struct Walk {
  unsigned b, s;
  int h;
  long long at, other;
  __device__ __forceinline__ Walk(const HeadsArgs& p, const HeadsPart& part, const HeadsView& v, const HeadsView& w,
                                  unsigned first) {
    const unsigned token = first / part.heads;
    h = first - token * part.heads;
    b = token / p.S;
    s = token - b * p.S;
    start(v, w);
    at += h * v.h;
    other += h * w.h;
  }
  __device__ __forceinline__ void start(const HeadsView& v, const HeadsView& w) {
    at = (long long)b * v.b + (long long)s * v.s;
    other = (long long)b * w.b + (long long)s * w.s;
  }
  // whether the next head is another token's
  __device__ __forceinline__ bool next(const HeadsArgs& p, const HeadsPart& part, const HeadsView& v,
                                       const HeadsView& w) {
    at += v.h;
    other += w.h;
    if (++h < part.heads) return false;
    h = 0;
    if (++s == (unsigned)p.S) { s = 0; ++b; }
    start(v, w);
    return true;
  }
};
// row of the tables for a token; that of one behind the last is never used
__device__ __forceinline__ long long table_row(const HeadsArgs& p, unsigned b, unsigned s) {
  if (b * p.S + s >= p.tokens) return -1;
  return p.pos ? __ldg(p.pos + b * p.pos_b + s * p.pos_s) : (long long)s;
}

template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from) {
  if constexpr (BYTES == 16) cp_async16(to, from);
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES) : "memory");
}

enum { ROTATE, UNROTATE, NORM, NORM_BACK };                    // what a call does

// What a thread has on its way through shared memory: its own vectors of the next STAGES heads, in which no other
// thread has a part, so that it waits for its own copies only.
template <typename T, int VW, int NS, int MODE>
struct HeadsRing {
  static constexpr bool BACK = MODE == NORM_BACK;
  // CTAs that an SM holds, by registers
  static constexpr int CTAS = BACK ? BACK_CTAS : (MODE == NORM ? 3 : 4) - (VW == 1);
  static constexpr int TENSORS = BACK ? 2 : 1, VEC = VW * (int)sizeof(T);
  static constexpr bool ASYNC = VEC >= 4;            // no copy moves 2 bytes
  static constexpr int STAGE = 256 * TENSORS * NS * 2 * VEC;
  static constexpr int ROOM = RING_BYTES / CTAS / STAGE, STAGES = ASYNC ? (ROOM > 12 ? 12 : ROOM) : 1;
  static constexpr int BYTES = STAGES * STAGE > 8 * MAX_HEAD_DIM * 4 ? STAGES * STAGE : 8 * MAX_HEAD_DIM * 4;
};

// ROTATE and NORM: x -> y; UNROTATE is the backward of a rotation alone.  NORM_BACK: x and the gradient g of the
// result -> y and the sums for dw, one row a CTA, which heads_fold_kernel adds in order.
// A CTA stays with one part.  Its groups take `per` heads each, one after the other, token by token: the parts of a
// call and the heads of a part need not divide anything.  `per` is rounded up, so the last groups of a part have what is
// left, or nothing.
// What bounds it is HBM behind some 200 (a rotation) to 350 instructions (a backward) a head and lane, half of them
// conversions and packed arithmetic: [1, 2048, 3, 32, 128] bf16 21 us forward (4.8 TB/s) and 30 backward with the fold
// (4.5), a rotation of [1, 32768, 8, 128] 25 (5.3), where an element-wise pass over as many bytes takes 17, 22 and 22.
// The backward's 122 registers leave two CTAs an SM, less than what hides its loads.  Heads loaded into registers by
// the four took 24 and 40 us; all groups going through memory together, 4 or 8 heads each at a time, 30 and 43 (angles
// are loaded more often); the next token's angles in registers 23 (fewer CTAs an SM).
template <typename T, int VW, int NS, int MODE, bool INTER, bool FIT>
__global__ void __launch_bounds__(256, HeadsRing<T, VW, NS, MODE>::CTAS)
heads_kernel(const __grid_constant__ HeadsArgs p) {
  using S = Slots<T, VW, NS, INTER, FIT>;
  using R = HeadsRing<T, VW, NS, MODE>;
  using raw = typename S::raw;
  constexpr int P = S::P, STEP = 256 * R::TENSORS * NS * 2;  // raws of a stage
  constexpr bool BACK = MODE == NORM_BACK;
  extern __shared__ __align__(16) char heads_smem[];
  raw* ring = reinterpret_cast<raw*>(heads_smem) + threadIdx.x;
  auto place = [&](int stage, int tensor, int n, int side) -> raw* {
    return ring + stage * STEP + ((tensor * NS + n) * 2 + side) * 256;
  };
  const int lane = threadIdx.x & ((1 << p.lg) - 1);
  int k = 0;
  while (blockIdx.x >= (unsigned)(p.part[k].cta0 + p.part[k].ctas)) ++k;
  const HeadsPart& part = p.part[k];
  const unsigned group = (blockIdx.x - part.cta0) * (256u >> p.lg) + (threadIdx.x >> p.lg);
  const unsigned all = p.tokens * (unsigned)part.heads;
  const unsigned first = (unsigned)min((unsigned long long)group * part.per, (unsigned long long)all);
  const int mine = min(all - first, (unsigned)part.per);
  // Groups make as many steps as they have heads, and add up among their own lanes; where lanes are left over, all
  // make as many as any, which keeps the warp together ([2, 4096] tokens of 32 and 8 heads: 34 us for 41).
  const int steps = FIT ? mine : part.per;
  const unsigned lanes = !FIT || p.lg == 5 ? 0xffffffffu : ((1u << (1 << p.lg)) - 1) << (threadIdx.x & 31 & ~((1 << p.lg) - 1));
  const S slot(p, lane);
  after_previous();

  const HeadsView &first_in = BACK ? part.g : part.x;
  Walk in(p, part, first_in, part.x, first), out(p, part, part.y, part.y, first);
  int filled = 0;                                    // the stage that the next fetch fills
  raw now[R::TENSORS][NS][2] = {}, then[R::TENSORS][NS][2] = {};
  auto fetch = [&](int step) {                       // one head of the walk, if the group still has it
    if (step < mine) {
      const T* from[2] = {reinterpret_cast<const T*>(first_in.at) + in.at,
                          BACK ? reinterpret_cast<const T*>(part.x.at) + in.other : nullptr};
#pragma unroll
      for (int q = 0; q < R::TENSORS; ++q) {
        if (BACK && q == 1 && !part.turn) continue;  // the values of a projection: only their gradient is read
        if constexpr (R::ASYNC) {
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            if (slot.has_a(n)) copy_async<R::VEC>(place(filled, q, n, 0), from[q] + slot.a[n]);
            if (slot.has_b(n)) copy_async<R::VEC>(place(filled, q, n, 1), from[q] + slot.b[n]);
          }
        } else {
          slot.load(from[q], then[q]);
        }
      }
      in.next(p, part, first_in, part.x);
    }
    if constexpr (R::ASYNC) {
      cp_async_commit();
      filled = filled + 1 < R::STAGES ? filled + 1 : 0;
    }
  };
  if constexpr (R::ASYNC) {
    for (int i = 0; i < R::STAGES - 1; ++i) fetch(i);
  } else {
    fetch(0);
  }

  typename S::Angles by[NS] = {};
  typename S::Values w[NS] = {}, dw[NS] = {};
  unsigned nb = out.b, ns = out.s;                   // the token whose row of the tables is on its way
  long long row = -1;
  auto next_angles = [&] {
    slot.angles(p, row, by);
    if (++ns == (unsigned)p.S) { ns = 0; ++nb; }
    row = table_row(p, nb, ns);
  };
  if (part.turn && mine > 0) {
    row = table_row(p, nb, ns);
    next_angles();
    if constexpr (MODE == NORM || BACK) slot.gains(part.w, w);
  }

  int stage = 0;
  for (int step = 0; step < steps; ++step) {
    const bool live = FIT || step < mine;
    if constexpr (R::ASYNC) {
      cp_async_wait<R::STAGES - 2>();
#pragma unroll
      for (int q = 0; q < R::TENSORS; ++q)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (!FIT) now[q][n][0] = now[q][n][1] = raw{};
          if (live && slot.has_a(n)) now[q][n][0] = *place(stage, q, n, 0);
          if (live && slot.has_b(n)) now[q][n][1] = *place(stage, q, n, 1);
        }
      stage = stage + 1 < R::STAGES ? stage + 1 : 0;
      fetch(step + R::STAGES - 1);                   // into the place that the step before this one has read
    } else {
#pragma unroll
      for (int q = 0; q < R::TENSORS; ++q)
#pragma unroll
        for (int n = 0; n < NS; ++n) { now[q][n][0] = then[q][n][0]; now[q][n][1] = then[q][n][1]; }
      fetch(step + 1);
    }
    T* y = reinterpret_cast<T*>(part.y.at) + out.at;
    if (!part.turn) {                                // the values of a projection
      if (live) {
#pragma unroll
        for (int n = 0; n < NS; ++n) slot.put(y, n, now[0][n]);
        out.next(p, part, part.y, part.y);
      }
      continue;
    }
    typename S::Values v[NS];                        // BACK: the gradient, turned back
    if constexpr (!BACK) {
      uint64_t squares = 0;                          // two zeros
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        v[n] = S::widen(now[0][n]);
        if constexpr (MODE == NORM)
#pragma unroll
          for (int j = 0; j < P; ++j) {
            squares = fma2(v[n].x[j], v[n].x[j], squares);
            squares = fma2(v[n].y[j], v[n].y[j], squares);
            v[n].x[j] = mul2(v[n].x[j], w[n].x[j]);
            v[n].y[j] = mul2(v[n].y[j], w[n].y[j]);
          }
        if (slot.turns(n)) S::template turn<MODE == UNROTATE>(by[n], v[n]);
      }
      if constexpr (MODE == NORM) {                  // what hangs on the sum comes last
        float sum[1] = {halves(squares)};
        group_sum(sum, p.lg, lanes);
        const float r = rsqrtf(sum[0] * p.inv_D + p.eps);
        const uint64_t r2 = f2_pack(r, r);
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int j = 0; j < P; ++j) { v[n].x[j] = mul2(v[n].x[j], r2); v[n].y[j] = mul2(v[n].y[j], r2); }
      }
    } else {
      uint64_t squares = 0, dots = 0;
      typename S::Values x[NS];
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        v[n] = S::widen(now[0][n]);
        if (slot.turns(n)) S::template turn<true>(by[n], v[n]);
        x[n] = S::widen(now[1][n]);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          squares = fma2(x[n].x[j], x[n].x[j], squares);
          squares = fma2(x[n].y[j], x[n].y[j], squares);
          dots = fma2(mul2(v[n].x[j], w[n].x[j]), x[n].x[j], dots);
          dots = fma2(mul2(v[n].y[j], w[n].y[j]), x[n].y[j], dots);
        }
      }
      float sum[2] = {halves(squares), halves(dots)};
      group_sum(sum, p.lg, lanes);
      // r (g w - xh m) with xh = x r and m = mean(g w xh) is (g w) r + x (-r^3 mean(g w x))
      const float r = rsqrtf(sum[0] * p.inv_D + p.eps), m = -(r * (r * (r * (sum[1] * p.inv_D))));
      const uint64_t r2 = f2_pack(r, r), m2 = f2_pack(m, m);
      if (live)
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const uint64_t gx = mul2(v[n].x[j], r2), gy = mul2(v[n].y[j], r2);
            dw[n].x[j] = fma2(gx, x[n].x[j], dw[n].x[j]);
            dw[n].y[j] = fma2(gy, x[n].y[j], dw[n].y[j]);
            v[n].x[j] = fma2(x[n].x[j], m2, mul2(gx, w[n].x[j]));
            v[n].y[j] = fma2(x[n].y[j], m2, mul2(gy, w[n].y[j]));
          }
    }
    if (live) {
#pragma unroll
      for (int n = 0; n < NS; ++n) slot.store(y, n, v[n]);
      if (out.next(p, part, part.y, part.y)) next_angles();
    }
  }

  if constexpr (BACK) {
    if (!part.turn) return;                          // the same for the whole CTA
    float(*sums)[MAX_HEAD_DIM] = reinterpret_cast<float(*)[MAX_HEAD_DIM]>(heads_smem);
    __syncwarp();
    if constexpr (R::ASYNC) cp_async_wait<0>();
    __syncthreads();                                 // nobody's copies are still on their way into the ring
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      float x[2 * P], y[2 * P];
#pragma unroll
      for (int j = 0; j < P; ++j) {
        f2_unpack(dw[n].x[j], x[2 * j], x[2 * j + 1]);
        f2_unpack(dw[n].y[j], y[2 * j], y[2 * j + 1]);
      }
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        for (int o = 1 << p.lg; o < 32; o <<= 1) {
          x[j] += __shfl_xor_sync(0xffffffffu, x[j], o);
          y[j] += __shfl_xor_sync(0xffffffffu, y[j], o);
        }
        constexpr bool beside = INTER && VW > 1;     // as in pairs_of
        const int half = j < VW / 2 ? slot.a[n] : slot.b[n], at = j < VW / 2 ? 2 * j : 2 * j - VW;
        const int x_at = beside ? half + at : slot.a[n] + j, y_at = beside ? half + at + 1 : slot.b[n] + j;
        if ((threadIdx.x & 31) < (1 << p.lg)) {
          if (FIT || (beside ? half : slot.a[n]) >= 0) sums[threadIdx.x >> 5][x_at] = x[j];
          if (FIT || (beside ? half : slot.b[n]) >= 0) sums[threadIdx.x >> 5][y_at] = y[j];
        }
      }
    }
    __syncthreads();
    if (threadIdx.x < p.D) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) t += sums[i][threadIdx.x];
      part.dw[(long long)blockIdx.x * p.D + threadIdx.x] = t;
    }
  }
}

// dw of each part (+)= its CTAs' sums, in their order.  blockIdx.y: the part; 32 columns and 32 shares of the rows a CTA.
__global__ void __launch_bounds__(1024)
heads_fold_kernel(const float* __restrict__ part0, const float* __restrict__ part1, float* __restrict__ dw0,
                  float* __restrict__ dw1, int ctas0, int ctas1, int D, int accumulate) {
  after_previous();
  __shared__ float sums[32][33];
  const float* in = blockIdx.y ? part1 : part0;
  float* out = blockIdx.y ? dw1 : dw0;
  const int n = blockIdx.y ? ctas1 : ctas0, lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  int col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < D)
#pragma unroll 4
    for (int i = share; i < n; i += 32) t += in[(long long)i * D + col];
  sums[share][lane] = t;
  __syncthreads();
  t = warp_sum(sums[lane][share]);                   // a warp a column
  col = blockIdx.x * 32 + share;
  if (lane == 0 && col < D) out[col] = accumulate ? out[col] + t : t;
}

}  // namespace pf

using namespace pf;

namespace {

// Values of a slot's halves: the widest that divides all it is given, which 16 bytes bound.
struct Width {
  int bytes, size;
  void all(const void* at) { fit(reinterpret_cast<uintptr_t>(at)); }
  void elements(long long n) { fit((unsigned long long)(n < 0 ? -n : n) * size); }
  void fit(unsigned long long n) { while (n % bytes) bytes /= 2; }
};

int pow2_log(int n) { int l = 0; while ((1 << l) < n) ++l; return l; }

// Fills in what a call's parts have in common and returns the values VW of a slot's halves, or a refusal.
int prepare(HeadsArgs& p, int parts, const void* cos_t, const void* sin_t, const void* pos,
            const long long* pos_strides, long long B, int S, int D, int R, long long rows, float eps,
            int dtype) {
  if (dtype != PF_F32 && dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (D < 1 || D > MAX_HEAD_DIM || R < 2 || R > D || R % 2) return -3;
  if (B * S > 0x7fffffffll) return -3;
  Width w{16, dtype == PF_F32 ? 4 : 2};
  for (int k = 0; k < parts; ++k)
    for (const HeadsView* v : {&p.part[k].x, &p.part[k].y, &p.part[k].g})
      if (v->at) {
        if (reinterpret_cast<uintptr_t>(v->at) % w.size) return -2;
        w.all(v->at);
        w.elements(v->b); w.elements(v->s); w.elements(v->h);
      }
  w.elements(D);
  w.elements(R / 2);
  int vw = w.bytes / w.size;
  if (reinterpret_cast<uintptr_t>(cos_t) % 4 || reinterpret_cast<uintptr_t>(sin_t) % 4 ||
      reinterpret_cast<uintptr_t>(pos) % 8)
    return -2;
  if (vw >= 4 && !on_vectors(p.part[0].w, p.part[parts > 1].w, (const float*)cos_t, (const float*)sin_t)) vw = 2;
  p.cos_t = (const float*)cos_t;
  p.sin_t = (const float*)sin_t;
  p.pos = (const long long*)pos;
  p.pos_b = pos ? pos_strides[0] : 0;
  p.pos_s = pos ? pos_strides[1] : 0;
  p.rows = rows;
  p.S = S; p.D = D; p.R = R;
  p.eps = eps;
  p.inv_D = 1.f / D;
  p.tokens = (unsigned)(B * S);
  const int slots = R / (2 * vw) + (D - R + 2 * vw - 1) / (2 * vw), each = vw >= 4 ? 1 : vw == 2 ? 2 : 4;
  p.lg = pow2_log((slots + each - 1) / each);
  return vw;
}

// CTAs and heads of their groups for each part: `most` CTAs altogether, shared by the bytes that the parts move,
// and no more than a part has heads for.  Returns the number of CTAs.
int deal(HeadsArgs& p, int parts, int most, const int* weight) {
  const int groups = 256 >> p.lg;
  long long total = 0;
  for (int k = 0; k < parts; ++k) total += (long long)weight[k] * p.part[k].heads;
  int ctas = 0;
  for (int k = 0; k < parts; ++k) {
    HeadsPart& part = p.part[k];
    const long long all = (long long)p.tokens * part.heads;
    long long share = total ? (long long)most * weight[k] * part.heads / total : 0;
    if (share < 1) share = 1;
    part.per = (int)((all + share * groups - 1) / (share * groups));
    part.ctas = part.per ? (int)((all + (long long)part.per * groups - 1) / ((long long)part.per * groups)) : 0;
    part.cta0 = ctas;
    ctas += part.ctas;
  }
  return ctas;
}

HeadsView view(const void* at, const long long* strides) {
  return {(char*)const_cast<void*>(at), strides[0], strides[1], strides[2]};
}

// calls f<T, VW, NS>()
template <typename F>
int by_width(int dtype, int vw, F& f) {
#define PF_W(T, W, NSLOTS) \
  if (vw == W) { f.template operator()<T, W, NSLOTS>(); return 0; }
  if (dtype == PF_F32) { PF_W(float, 4, 1) PF_W(float, 2, 2) PF_W(float, 1, 4) }
  if (dtype == PF_F16) { PF_W(__half, 8, 1) PF_W(__half, 4, 1) PF_W(__half, 2, 2) PF_W(__half, 1, 4) }
  if (dtype == PF_BF16) {
    PF_W(__nv_bfloat16, 8, 1) PF_W(__nv_bfloat16, 4, 1) PF_W(__nv_bfloat16, 2, 2) PF_W(__nv_bfloat16, 1, 4)
  }
#undef PF_W
  return -1;
}

template <int MODE>
struct Launch {
  HeadsArgs& p;
  int parts, interleaved, sms;
  const int* weight;
  cudaStream_t st;
  int code = 0;
  template <typename T, int VW, int NS> void operator()() {
    if (interleaved) fit<T, VW, NS, true>();
    else fit<T, VW, NS, false>();
  }
  // of the widest vectors alone: other heads seldom fill the lanes (a rotation of [1, 32768, 8, 128] 27 -> 25 us)
  template <typename T, int VW, int NS, bool INTER> void fit() {
    if constexpr (VW * sizeof(T) == 16)
      if (p.R == p.D && p.D == 2 * VW * NS << p.lg) return go<T, VW, NS, INTER, true>();
    go<T, VW, NS, INTER, false>();
  }
  template <typename T, int VW, int NS, bool INTER, bool FIT> void go() {
    using R = HeadsRing<T, VW, NS, MODE>;
    const int ctas = deal(p, parts, R::CTAS * sms, weight);
    if (ctas == 0) return;
    static bool done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (R::BYTES > 48 * 1024 && (dev < 0 || dev >= 64 || !done[dev])) {
      const cudaError_t e = cudaFuncSetAttribute(heads_kernel<T, VW, NS, MODE, INTER, FIT>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, R::BYTES);
      if (e != cudaSuccess) { code = (int)e; return; }
      if (dev >= 0 && dev < 64) done[dev] = true;
    }
    after(heads_kernel<T, VW, NS, MODE, INTER, FIT>, ctas, 256, R::BYTES, st)(p);
  }
};
template <int MODE>
int launch(HeadsArgs& p, int parts, const int* weight, int interleaved, int dtype, int vw, int sms, void* stream) {
  Launch<MODE> f{p, parts, interleaved, sms, weight, reinterpret_cast<cudaStream_t>(stream)};
  const int code = by_width(dtype, vw, f);
  return code ? code : f.code;
}
}  // namespace

// x: q [B, S, Hq, D], k [B, S, Hk, D] (null: none), v (null: none; strides of k, copied) -> yq, yk, yv.  wq / wk fp32
// [D] or null: a rotation alone.  cos / sin fp32 [rows, R/2]; pos int64 with strides (batch, seq), or null.
PF_API int pf_heads_fwd(const void* q, const void* k, const void* v, void* yq, void* yk, void* yv, const void* wq,
                        const void* wk, const void* cos_t, const void* sin_t, const void* pos, long long B, int S,
                        int Hq, int Hk, int D, int R, const long long* sq, const long long* sk,
                        const long long* syq, const long long* syk, const long long* spos, long long rows,
                        int interleaved, int inverse, float eps, int dtype, int sm_count, void* stream) {
  HeadsArgs p = {};
  int parts = 0;
  p.part[parts++] = {view(q, sq), view(yq, syq), {}, (const float*)wq, nullptr, Hq, 1, 0, 0, 0};
  if (k) p.part[parts++] = {view(k, sk), view(yk, syk), {}, (const float*)wk, nullptr, Hk, 1, 0, 0, 0};
  if (v) p.part[parts++] = {view(v, sk), view(yv, syk), {}, nullptr, nullptr, Hk, 0, 0, 0, 0};
  const int vw = prepare(p, parts, cos_t, sin_t, pos, spos, B, S, D, R, rows, eps, dtype);
  if (vw < 0) return vw;
  if ((long long)B * S * (Hq + 2ll * Hk) > 0x7fffffffll || (k && !wq != !wk)) return -3;
  if (p.tokens == 0 || (Hq == 0 && Hk == 0)) return 0;
  const int even[3] = {1, 1, 1};
  const int code = wq ? launch<NORM>(p, parts, even, interleaved, dtype, vw, sm_count, stream)
                   : inverse ? launch<UNROTATE>(p, parts, even, interleaved, dtype, vw, sm_count, stream)
                             : launch<ROTATE>(p, parts, even, interleaved, dtype, vw, sm_count, stream);
  if (code) return code;
  PF_CHECK_LAUNCH();
  return 0;
}

// Rows of partial sums that pf_heads_bwd needs: floats [that many][D].  A part that has heads gets a CTA though its
// share of them be less.
PF_API int pf_heads_bwd_rows(int Hq, int Hk, int sm_count) { return BACK_CTAS * sm_count + (Hq > 0) + (Hk > 0); }

// Gradients of pf_heads_fwd with a norm: gq, gk, gv (the outputs') -> dq, dk, dv and dwq, dwk fp32 [D]
// (accumulate: added to what is there).  gv null: there are no values.
PF_API int pf_heads_bwd(const void* gq, const void* gk, const void* gv, const void* q, const void* k, void* dq,
                        void* dk, void* dv, const void* wq, const void* wk, void* dwq, void* dwk, void* scratch,
                        const void* cos_t, const void* sin_t, const void* pos, long long B, int S, int Hq, int Hk,
                        int D, int R, const long long* sgq, const long long* sgk, const long long* sq,
                        const long long* sk, const long long* sdq, const long long* sdk, const long long* spos,
                        long long rows, int interleaved, float eps, int accumulate, int dtype, int sm_count,
                        void* stream) {
  HeadsArgs p = {};
  int parts = 0;
  p.part[parts++] = {view(q, sq), view(dq, sdq), view(gq, sgq), (const float*)wq, nullptr, Hq, 1, 0, 0, 0};
  p.part[parts++] = {view(k, sk), view(dk, sdk), view(gk, sgk), (const float*)wk, nullptr, Hk, 1, 0, 0, 0};
  if (gv) p.part[parts++] = {{}, view(dv, sdk), view(gv, sgk), nullptr, nullptr, Hk, 0, 0, 0, 0};
  const int vw = prepare(p, parts, cos_t, sin_t, pos, spos, B, S, D, R, rows, eps, dtype);
  if (vw < 0) return vw;
  if ((long long)B * S * (Hq + 2ll * Hk) > 0x7fffffffll || !wq || !wk || !dwq || !dwk || !scratch) return -3;
  // the sums' rows lie where the parts' CTAs do, at most BACK_CTAS an SM and one more for each of two parts
  const int weight[3] = {3, 3, 2};
  p.part[0].dw = p.part[1].dw = (float*)scratch;
  const int code = launch<NORM_BACK>(p, parts, weight, interleaved, dtype, vw, sm_count, stream);
  if (code) return code;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  after(heads_fold_kernel, dim3((D + 31) / 32, 2), 1024, 0, st)(
      (const float*)scratch, (const float*)scratch + (long long)p.part[1].cta0 * D, (float*)dwq, (float*)dwk,
      p.part[0].ctas, p.part[1].ctas, D, accumulate);
  PF_CHECK_LAUNCH();
  return 0;
}
