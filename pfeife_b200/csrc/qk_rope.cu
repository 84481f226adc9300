// Rotary positions of every layout, alone or behind an RMS norm of each head, over queries and keys (and the
// values of a fused projection, which are copied), forward and backward.
//
// A head of D values has R of them in pairs: (i, i + R/2), or (2i, 2i + 1) when interleaved.  A pair turns by the
// angle of its position and of its frequency i: (a, b) -> (a c - b s, b c + a s); values R..D stay.  In front of
// that the norm multiplies by r w, r = (mean x^2 + eps)^-1/2.  With g the gradient turned back (the transposed
// rotation), xh = x r:  dx = r (g w - xh mean(g w xh)),  dw = sum over tokens and heads of g xh.
// r is computed again in the backward, which reads x anyway.
//
// A head lies across a group of lanes, a power of two of them.  A lane owns slots of 2 VW values: in the pairs the
// VW values from i and those they turn with, behind them 2 VW in a row, so that a rotation needs no other lane
// and the norm one sum over the group.  Slot v turns by the frequencies VW v .. VW v + VW in both layouts: cosines
// and sines are loaded once per item, which is some heads of one token, and stay in registers.
#include "common.cuh"
#include "api.h"

namespace pf {

constexpr int MAX_HEAD_DIM = 256;

struct HeadsView {                 // [B, S, heads, D] in any order of memory with D innermost
  char* at;
  long long b, s, h;               // strides in elements
};
struct HeadsPart {
  HeadsView x, y, g;               // forward: x -> y; backward: x and the gradient g -> y
  const float* w;                  // gain of the norm, or null
  float* dw;                       // backward: [ctas][D] partial sums
  int heads, chunks;               // chunks: items of a token
  int turn;                        // 0: the values of a projection, which are copied
  int cta0, ctas;                  // backward: the CTAs of this part
};
struct HeadsArgs {
  HeadsPart part[3];
  const float *cos_t, *sin_t;      // [rows, R/2]
  const long long* pos;            // row of the tables for each token, or null: the token's place
  long long pos_b, pos_s, rows;
  int S, D, R, lg, chunks, per_item, interleaved, inverse;
  unsigned tokens, items;
  float eps, inv_D;
};

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = unsigned short; };

// Where a lane's slots lie in a head, and by how much they turn.
template <typename T, int VW, int NS>
struct Slots {
  static constexpr int N = 2 * VW;
  using raw = typename Raw<VW * sizeof(T)>::type;
  int a[NS], b[NS];                // first values of both halves, -1 where there is none
  bool turns[NS];

  __device__ __forceinline__ Slots(const HeadsArgs& p, int lane) {
    const int pairs = p.R / N;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int v = lane + (n << p.lg);
      turns[n] = v < pairs;
      a[n] = turns[n] ? (p.interleaved ? N * v : VW * v) : p.R + N * (v - pairs);
      b[n] = turns[n] && !p.interleaved ? a[n] + p.R / 2 : a[n] + VW;
      if (a[n] >= p.D) a[n] = -1;
      if (b[n] >= p.D || a[n] < 0) b[n] = -1;
    }
  }
  __device__ __forceinline__ void load(const T* x, raw (&r)[NS][2]) const {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      r[n][0] = r[n][1] = raw{};
      if (a[n] >= 0) r[n][0] = *reinterpret_cast<const raw*>(x + a[n]);
      if (b[n] >= 0) r[n][1] = *reinterpret_cast<const raw*>(x + b[n]);
    }
  }
  static __device__ __forceinline__ void widen(const raw (&r)[2], float (&v)[N]) {
    const T* e0 = reinterpret_cast<const T*>(&r[0]);
    const T* e1 = reinterpret_cast<const T*>(&r[1]);
#pragma unroll
    for (int j = 0; j < VW; ++j) { v[j] = to_f32<T>(e0[j]); v[VW + j] = to_f32<T>(e1[j]); }
  }
  __device__ __forceinline__ void store(T* y, int n, const float (&v)[N]) const {
    raw r[2];
    T* e0 = reinterpret_cast<T*>(&r[0]);
    T* e1 = reinterpret_cast<T*>(&r[1]);
#pragma unroll
    for (int j = 0; j < VW; ++j) { e0[j] = from_f32<T>(v[j]); e1[j] = from_f32<T>(v[VW + j]); }
    put(y, n, r);
  }
  __device__ __forceinline__ void put(T* y, int n, const raw (&r)[2]) const {
    if (a[n] >= 0) *reinterpret_cast<raw*>(y + a[n]) = r[0];
    if (b[n] >= 0) *reinterpret_cast<raw*>(y + b[n]) = r[1];
  }
  // gain of the norm at the slots' values
  __device__ __forceinline__ void gains(const float* w, float (&v)[NS][N]) const {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      take(w, a[n], v[n], 0.f);
      take(w, b[n], v[n] + VW, 0.f);
    }
  }
  // VW floats, or `none` where at is negative
  static __device__ __forceinline__ void take(const float* t, long long at, float* v, float none) {
#pragma unroll
    for (int j = 0; j < VW; j += (VW < 4 ? 1 : 4)) {
      if constexpr (VW >= 4) {
        const float4 q = at >= 0 ? __ldg(reinterpret_cast<const float4*>(t + at + j)) : make_float4(none, none, none, none);
        v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
      } else {
        v[j] = at >= 0 ? __ldg(t + at + j) : none;
      }
    }
  }
  // Cosines and sines at a token's row of the tables; NaN for a row that they do not have, which no kernel can
  // refuse without the host waiting for it.
  __device__ __forceinline__ void angles(const HeadsArgs& p, long long row, int lane, float (&c)[NS][VW],
                                         float (&s)[NS][VW]) const {
    const bool there = row >= 0 && row < p.rows;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (!turns[n]) continue;
      const long long at = there ? row * (p.R / 2) + VW * (lane + (n << p.lg)) : -1;
      take(p.cos_t, at, c[n], NAN);
      take(p.sin_t, at, s[n], NAN);
    }
  }
  // v turned by (c, s)
  static __device__ __forceinline__ void turn(bool interleaved, const float (&c)[VW], const float (&s)[VW],
                                              float (&v)[N]) {
    float t[N];
    if (interleaved) {
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        t[2 * j] = v[2 * j] * c[j] - v[2 * j + 1] * s[j];
        t[2 * j + 1] = v[2 * j + 1] * c[j] + v[2 * j] * s[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        t[j] = v[j] * c[j] - v[VW + j] * s[j];
        t[VW + j] = v[VW + j] * c[j] + v[j] * s[j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = t[j];
  }
};

// sums of U values over the group of a lane; every lane of the warp calls it
template <int U>
__device__ __forceinline__ void group_sum(float (&v)[U], int lg) {
  for (int o = (1 << lg) >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
}

__device__ __forceinline__ long long table_row(const HeadsArgs& p, unsigned b, unsigned s) {
  return p.pos ? __ldg(p.pos + b * p.pos_b + s * p.pos_s) : (long long)s;
}
template <typename T>
__device__ __forceinline__ T* head_at(const HeadsView& v, unsigned b, unsigned s, int h) {
  return reinterpret_cast<T*>(v.at) + (long long)b * v.b + (long long)s * v.s + (long long)h * v.h;
}

// x -> y.  The backward of a rotation without a norm is the same kernel with `inverse`.
constexpr int FWD = 128;
#ifndef XL
#define XL 1536
#endif
constexpr long long FWD_LANES = XL;
template <typename T, int VW, int NS, bool NORM>
__global__ void __launch_bounds__(FWD, NORM ? 5 : 6) heads_fwd_kernel(const __grid_constant__ HeadsArgs p) {
  constexpr int HEADS = NORM ? 4 : 2;                // heads that a group has in flight
  after_previous();
  using S = Slots<T, VW, NS>;
  const int lane = threadIdx.x & ((1 << p.lg) - 1);
  const unsigned item = blockIdx.x * ((unsigned)FWD >> p.lg) + (threadIdx.x >> p.lg);
  const bool live = item < p.items;
  const unsigned token = live ? item / p.chunks : 0;
  int chunk = live ? item - token * p.chunks : 0, k = 0;
  while (chunk >= p.part[k].chunks) chunk -= p.part[k++].chunks;
  const HeadsPart& part = p.part[k];
  const unsigned b = token / p.S, s = token - b * p.S;
  const int h0 = chunk * p.per_item, heads = live ? min(p.per_item, part.heads - h0) : 0;
  const S slot(p, lane);
  const T* x = head_at<const T>(part.x, b, s, h0);
  T* y = head_at<T>(part.y, b, s, h0);

  // the row's number, the heads and then what hangs on the number: two latencies in a row, not three
  const long long row = part.turn ? table_row(p, b, s) : 0;
  typename S::raw raw[HEADS][NS][2];
#pragma unroll
  for (int u = 0; u < HEADS; ++u)
    if (u < heads) slot.load(x + u * part.x.h, raw[u]);
  float c[NS][VW], sn[NS][VW], w[NS][S::N];
  if (part.turn) {
    slot.angles(p, row, lane, c, sn);
    if (p.inverse)
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int j = 0; j < VW; ++j) sn[n][j] = -sn[n][j];
    if constexpr (NORM) slot.gains(part.w, w);
  }
  for (int u0 = 0;;) {
    float r[HEADS];
    if constexpr (NORM) {
#pragma unroll
      for (int u = 0; u < HEADS; ++u) {
        r[u] = 0.f;
        if (u0 + u < heads)
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            float v[S::N];
            S::widen(raw[u][n], v);
#pragma unroll
            for (int j = 0; j < S::N; ++j) r[u] += v[j] * v[j];
          }
      }
      group_sum(r, p.lg);
#pragma unroll
      for (int u = 0; u < HEADS; ++u) r[u] = rsqrtf(r[u] * p.inv_D + p.eps);
    }
#pragma unroll
    for (int u = 0; u < HEADS; ++u)
      if (u0 + u < heads)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          if (!part.turn) {                          // the values of a projection
            slot.put(y + u * part.y.h, n, raw[u][n]);
            continue;
          }
          float v[S::N];
          S::widen(raw[u][n], v);
          if constexpr (NORM)
#pragma unroll
            for (int j = 0; j < S::N; ++j) v[j] *= r[u] * w[n][j];
          if (slot.turns[n]) S::turn(p.interleaved, c[n], sn[n], v);
          slot.store(y + u * part.y.h, n, v);
        }
    u0 += HEADS;
    if (u0 >= p.per_item) return;                    // the same for all items
    x += HEADS * part.x.h;
    y += HEADS * part.y.h;
#pragma unroll
    for (int u = 0; u < HEADS; ++u)
      if (u0 + u < heads) slot.load(x + u * part.x.h, raw[u]);
  }
}

// Gradients behind a norm.  A CTA stays with one part, its groups walk over that part's items, and a lane adds up
// dw of its values in registers; the CTA leaves one row of sums, which heads_fold_kernel adds in order.
template <typename T, int VW, int NS>
__global__ void __launch_bounds__(256, 2) heads_bwd_kernel(const __grid_constant__ HeadsArgs p) {
  after_previous();
  using S = Slots<T, VW, NS>;
  constexpr int N = S::N, U = 2;                     // heads that a group has in flight
  __shared__ float sums[8][MAX_HEAD_DIM];
  const int lane = threadIdx.x & ((1 << p.lg) - 1), groups = 256 >> p.lg;
  int k = 0;
  while (blockIdx.x >= (unsigned)(p.part[k].cta0 + p.part[k].ctas)) ++k;
  const HeadsPart& part = p.part[k];
  const unsigned cta = blockIdx.x - part.cta0, items = p.tokens * part.chunks, step = part.ctas * groups;
  const S slot(p, lane);
  float w[NS][N], dw[NS][N] = {};
  if (part.w) slot.gains(part.w, w);
  // whole warps stay in the loop together: the sums over a group are made by all lanes
  for (unsigned first = cta * groups; first < items; first += step) {
    const unsigned item = first + (threadIdx.x >> p.lg);
    const bool live = item < items;
    const unsigned token = live ? item / part.chunks : 0, chunk = live ? item - token * part.chunks : 0;
    const unsigned b = token / p.S, s = token - b * p.S;
    const int h0 = chunk * p.per_item, heads = live ? min(p.per_item, part.heads - h0) : 0;
    float c[NS][VW], sn[NS][VW];
    if (part.turn) slot.angles(p, table_row(p, b, s), lane, c, sn);
    for (int u0 = 0; u0 < p.per_item; u0 += U) {
      typename S::raw xr[U][NS][2], gr[U][NS][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u0 + u < heads) {
          slot.load(head_at<const T>(part.g, b, s, h0 + u0 + u), gr[u]);
          if (part.w) slot.load(head_at<const T>(part.x, b, s, h0 + u0 + u), xr[u]);
        }
      if (!part.w) {                                 // the values of a projection
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u0 + u < heads) {
            T* y = head_at<T>(part.y, b, s, h0 + u0 + u);
#pragma unroll
            for (int n = 0; n < NS; ++n) slot.put(y, n, gr[u][n]);
          }
        continue;
      }
      float sum[2 * U];                              // of x^2, then of g w x
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sum[u] = sum[U + u] = 0.f;
        if (u0 + u < heads)
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            float x[N], g[N];
            S::widen(xr[u][n], x);
            S::widen(gr[u][n], g);
            if (slot.turns[n]) {
              float back[VW];
#pragma unroll
              for (int j = 0; j < VW; ++j) back[j] = -sn[n][j];
              S::turn(p.interleaved, c[n], back, g);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
              sum[u] += x[j] * x[j];
              sum[U + u] += g[j] * w[n][j] * x[j];
            }
          }
      }
      group_sum(sum, p.lg);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u0 + u < heads) {
          T* y = head_at<T>(part.y, b, s, h0 + u0 + u);
          const float r = rsqrtf(sum[u] * p.inv_D + p.eps), m = r * sum[U + u] * p.inv_D;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            float x[N], g[N];
            S::widen(xr[u][n], x);
            S::widen(gr[u][n], g);
            if (slot.turns[n]) {
              float back[VW];
#pragma unroll
              for (int j = 0; j < VW; ++j) back[j] = -sn[n][j];
              S::turn(p.interleaved, c[n], back, g);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float xh = x[j] * r;
              dw[n][j] += g[j] * xh;
              x[j] = r * (g[j] * w[n][j] - xh * m);
            }
            slot.store(y, n, x);
          }
        }
    }
  }
  if (!part.dw) return;                              // the same for the whole CTA
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int j = 0; j < N; ++j)
      for (int o = 1 << p.lg; o < 32; o <<= 1) dw[n][j] += __shfl_xor_sync(0xffffffffu, dw[n][j], o);
  if ((threadIdx.x & 31) < (1 << p.lg))
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int at = j < VW ? slot.a[n] : slot.b[n];
        if (at >= 0) sums[threadIdx.x >> 5][at + (j < VW ? j : j - VW)] = dw[n][j];
      }
  __syncthreads();
  if (threadIdx.x < p.D) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sums[i][threadIdx.x];
    part.dw[(long long)cta * p.D + threadIdx.x] = t;
  }
}

// dw[part] (+)= the CTAs' sums, in their order.  blockIdx.y: the part; 32 columns and 8 shares of the rows a CTA.
__global__ void __launch_bounds__(256)
heads_fold_kernel(const float* __restrict__ part0, const float* __restrict__ part1, float* __restrict__ dw0,
                  float* __restrict__ dw1, int ctas0, int ctas1, int D, int accumulate) {
  after_previous();
  __shared__ float sums[8][33];
  const float* in = blockIdx.y ? part1 : part0;
  float* out = blockIdx.y ? dw1 : dw0;
  const int n = blockIdx.y ? ctas1 : ctas0, col = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  float t = 0.f;
  if (out && col < D)
#pragma unroll 4
    for (int i = share; i < n; i += 8) t += in[(long long)i * D + col];
  sums[share][threadIdx.x & 31] = t;
  __syncthreads();
  if (out && share == 0 && col < D) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sums[i][threadIdx.x & 31];
    out[col] = accumulate ? out[col] + t : t;
  }
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
            const long long* pos_strides, long long B, int S, int D, int R, long long rows, int interleaved,
            float eps, int dtype) {
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
  p.interleaved = interleaved;
  p.eps = eps;
  p.inv_D = 1.f / D;
  p.tokens = (unsigned)(B * S);
  const int slots = R / (2 * vw) + (D - R + 2 * vw - 1) / (2 * vw), each = vw >= 4 ? 1 : vw == 2 ? 2 : 4;
  p.lg = pow2_log((slots + each - 1) / each);
  return vw;
}

// Heads of an item: as many as leave every SM `lanes` lanes with an item of their own.
void deal(HeadsArgs& p, int parts, long long lanes) {
  for (p.per_item = 16;; p.per_item /= 2) {
    p.chunks = 0;
    for (int k = 0; k < parts; ++k) {
      p.part[k].chunks = (p.part[k].heads + p.per_item - 1) / p.per_item;
      p.chunks += p.part[k].chunks;
    }
    p.items = p.tokens * (unsigned)p.chunks;
    if (p.per_item == 1 || ((long long)p.items << p.lg) >= lanes) return;
  }
}

HeadsView view(const void* at, const long long* strides) {
  return {(char*)const_cast<void*>(at), strides[0], strides[1], strides[2]};
}

// calls f<T, VW, NS>()
template <typename F>
int by_width(int dtype, int vw, F&& f) {
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

struct Forward {
  const HeadsArgs& p;
  bool norm;
  cudaStream_t st;
  template <typename T, int VW, int NS> void operator()() {
    const unsigned per = (unsigned)FWD >> p.lg, grid = (p.items + per - 1) / per;
    if (norm) after(heads_fwd_kernel<T, VW, NS, true>, grid, FWD, 0, st)(p);
    else after(heads_fwd_kernel<T, VW, NS, false>, grid, FWD, 0, st)(p);
  }
};
struct Backward {
  const HeadsArgs& p;
  int ctas;
  cudaStream_t st;
  template <typename T, int VW, int NS> void operator()() {
    after(heads_bwd_kernel<T, VW, NS>, ctas, 256, 0, st)(p);
  }
};

// CTAs of the backward's parts, by their heads: together two per SM of the caller's count, no more than a part
// has items for.
int bwd_ctas(int heads, int all_heads, int sms) {
  const long long n = all_heads > 0 ? 2ll * sms * heads / all_heads : 0;
  return n < 1 ? 1 : (int)n;
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
  p.part[parts++] = {view(q, sq), view(yq, syq), {}, (const float*)wq, nullptr, Hq, 0, 1, 0, 0};
  if (k) p.part[parts++] = {view(k, sk), view(yk, syk), {}, (const float*)wk, nullptr, Hk, 0, 1, 0, 0};
  if (v) p.part[parts++] = {view(v, sk), view(yv, syk), {}, nullptr, nullptr, Hk, 0, 0, 0, 0};
  const int vw = prepare(p, parts, cos_t, sin_t, pos, spos, B, S, D, R, rows, interleaved, eps, dtype);
  if (vw < 0) return vw;
  p.inverse = inverse;
  if ((long long)B * S * (Hq + 2ll * Hk) > 0x7fffffffll) return -3;
  deal(p, parts, FWD_LANES * sm_count);
  if (p.items == 0) return 0;
  const int code = by_width(dtype, vw, Forward{p, wq != nullptr, reinterpret_cast<cudaStream_t>(stream)});
  if (code) return code;
  PF_CHECK_LAUNCH();
  return 0;
}

// Rows of partial sums that pf_heads_bwd needs: floats [that many][D].
PF_API int pf_heads_bwd_rows(int Hq, int Hk, int sm_count) {
  return bwd_ctas(Hq, Hq + Hk, sm_count) + bwd_ctas(Hk, Hq + Hk, sm_count);
}

// Gradients of pf_heads_fwd with a norm: gq, gk, gv (the outputs') -> dq, dk, dv and dwq, dwk fp32 [D] (null: not
// needed; accumulate: added to what is there).  gv null: there are no values.
PF_API int pf_heads_bwd(const void* gq, const void* gk, const void* gv, const void* q, const void* k, void* dq,
                        void* dk, void* dv, const void* wq, const void* wk, void* dwq, void* dwk, void* scratch,
                        const void* cos_t, const void* sin_t, const void* pos, long long B, int S, int Hq, int Hk,
                        int D, int R, const long long* sgq, const long long* sgk, const long long* sq,
                        const long long* sk, const long long* sdq, const long long* sdk, const long long* spos,
                        long long rows, int interleaved, float eps, int accumulate, int dtype, int sm_count,
                        void* stream) {
  HeadsArgs p = {};
  int parts = 0;
  p.part[parts++] = {view(q, sq), view(dq, sdq), view(gq, sgq), (const float*)wq, nullptr, Hq, 0, 1, 0, 0};
  p.part[parts++] = {view(k, sk), view(dk, sdk), view(gk, sgk), (const float*)wk, nullptr, Hk, 0, 1, 0, 0};
  if (gv) p.part[parts++] = {{}, view(dv, sdk), view(gv, sgk), nullptr, nullptr, Hk, 0, 0, 0, 0};
  const int vw = prepare(p, parts, cos_t, sin_t, pos, spos, B, S, D, R, rows, interleaved, eps, dtype);
  if (vw < 0) return vw;
  if ((long long)B * S * (Hq + 2ll * Hk) > 0x7fffffffll) return -3;
  deal(p, parts, 1024ll * sm_count);
  const int groups = 256 >> p.lg;
  int ctas = 0;
  float* left = (float*)scratch;
  for (int i = 0; i < parts; ++i) {
    HeadsPart& part = p.part[i];
    const long long items = (long long)p.tokens * part.chunks, most = (items + groups - 1) / groups;
    part.ctas = i < 2 ? bwd_ctas(part.heads, Hq + Hk, sm_count) : sm_count;
    if (part.ctas > most) part.ctas = (int)most;
    part.cta0 = ctas;
    ctas += part.ctas;
    if (i < 2 && (i ? dwk : dwq)) part.dw = left;
    if (i < 2) left += (long long)part.ctas * D;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (ctas) {
    const int code = by_width(dtype, vw, Backward{p, ctas, st});
    if (code) return code;
  }
  if (dwq || dwk)
    after(heads_fold_kernel, dim3((D + 31) / 32, 2), 256, 0, st)(
        (const float*)p.part[0].dw, (const float*)p.part[1].dw, (float*)dwq, (float*)dwk, p.part[0].ctas,
        p.part[1].ctas, D, accumulate);
  PF_CHECK_LAUNCH();
  return 0;
}
