// The gated feed-forward block, y = (act(x Wg^T + bg) * (x Wu^T + bu)) W2^T + b2 + residual, and its gradients, as the
// products of fused_gemm_sm100.cu and gemm_sm100.cu.
//
// Forward 6 M D H operations in two products (the first with both projections, the activation and their product in its
// epilogue), backward 12 M D H in five: dh with everything that follows from it in the epilogue, dx and the weights'
// gradients.  Gate, up, their gradients and h are operands of 16-bit products, or kept for them, and rounded to that (gate and
// up within the type's range); activations and their derivatives are of fp32 sums forward, and of what was kept backward.
// For few rows the weights are what moves, and products have few tiles: one is then split over its reduction
// into as many parts as keep all SMs reading (plan_parts), and what its epilogue does is done by the kernels here, which
// add the parts up in their order.
//
// On a B200, bf16, forward and backward: 2048 rows of 4096 over 11008 hidden values (1.66 TFLOP) 1.17 ms in a short run,
// 1.42 PFLOP/s; 16384 of 640 over 2560 with GELU and biases 568 us, 0.85 PFLOP/s, where gate, up, their gradients and h are
// 26 MB a thousand rows; 13 of 4096 over 11008 190 us, of which 124 are what memory takes for the weights twice and their
// gradients once.
#include "common.cuh"
#include "api.h"
#include "fused_gemm.h"

namespace pf {

struct Parts {
  const float* at;
  int parts;
  long long size;               // floats of a part
};
__device__ __forceinline__ void sum_parts(const Parts& p, long long i, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 4
  for (int k = 0; k < p.parts; ++k) {
    const float4* q = reinterpret_cast<const float4*>(p.at + k * p.size + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(e[j]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  uint4 q;
  T* e = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
  *reinterpret_cast<uint4*>(p) = q;
}
template <typename T> __device__ __forceinline__ void store8_saturated(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(saturated2<T>(v[0], v[1]), saturated2<T>(v[2], v[3]),
                                            saturated2<T>(v[4], v[5]), saturated2<T>(v[6], v[7]));
}
__device__ __forceinline__ void add_bias8(const void* b, int dtype, int i, float (&v)[8]) {
  if (!b) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] += dtype == PF_F32 ? static_cast<const float*>(b)[i + j]
            : dtype == PF_F16 ? __half2float(static_cast<const __half*>(b)[i + j])
                              : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i + j]);
}
__device__ __forceinline__ void act_of(int act, float z, float& a, float& slope) {
  if (act == 1) {
    a = gelu_erf(z);
    slope = dgelu_erf(z);
  } else {
    // z s(q), see fused_gemm_sm100.cu
    const float z2 = z * z, c = 2.f * 0.7978845608028654f;
    const float q = act == 2 ? c * z * fmaf(z2, 0.044715f, 1.f) : z;
    const float dq = act == 2 ? fmaf(fminf(z2, 1e6f), 3.f * 0.044715f * c, c) : 1.f;
    const float s = 1.f / (1.f + __expf(-q));
    a = z * s;
    slope = fmaf(a - a * s, dq, s);
  }
}

// Gate and up of 8 hidden values a thread -> h, and both kept.
template <typename T>
__global__ void __launch_bounds__(128)
glu_join_kernel(const Parts p, const void* __restrict__ bias, int bias_dtype, T* __restrict__ gu, T* __restrict__ h,
                int M, int H, int act) {
  after_previous();
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  const int nv = H / 8, m = (int)(i / nv), c = (int)(i - (long long)m * nv) * 8;
  if (m >= M) return;
  float g[8], u[8];
  sum_parts(p, (long long)m * 2 * H + c, g);
  sum_parts(p, (long long)m * 2 * H + H + c, u);
  add_bias8(bias, bias_dtype, c, g);
  add_bias8(bias, bias_dtype, H + c, u);
  if (gu) {                                             // within the type, see fused_gemm_sm100.cu
    store8_saturated(gu + (long long)m * 2 * H + c, g);
    store8_saturated(gu + (long long)m * 2 * H + H + c, u);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float a, slope;
    act_of(act, g[j], a, slope);
    g[j] = a * u[j];
  }
  store8(h + (long long)m * H + c, g);
}

// dh of 8 hidden values a thread -> the gradients of gate and up, and h.
template <typename T>
__global__ void __launch_bounds__(128)
glu_join_bwd_kernel(const Parts p, const T* __restrict__ gu, T* __restrict__ dgu, T* __restrict__ h, int M, int H,
                    int act) {
  after_previous();
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  const int nv = H / 8, m = (int)(i / nv), c = (int)(i - (long long)m * nv) * 8;
  if (m >= M) return;
  float d[8], g[8], u[8];
  const long long at = (long long)m * 2 * H + c;
  load8(gu + at, g);
  load8(gu + at + H, u);
  sum_parts(p, (long long)m * H + c, d);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float a, slope;
    act_of(act, g[j], a, slope);
    g[j] = d[j] * u[j] * slope;
    d[j] *= a;
    u[j] *= a;
  }
  store8(dgu + at, g);
  store8(dgu + at + H, d);
  store8(h + (long long)m * H + c, u);
}

// The sum of the parts, with a bias and a residual
template <typename T>
__global__ void __launch_bounds__(128)
row_join_kernel(const Parts p, const void* __restrict__ bias, int bias_dtype, const T* __restrict__ residual,
                long long ldr, T* __restrict__ out, int M, int N) {
  after_previous();
  const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
  const int nv = N / 8, m = (int)(i / nv), c = (int)(i - (long long)m * nv) * 8;
  if (m >= M) return;
  float v[8];
  sum_parts(p, (long long)m * N + c, v);
  add_bias8(bias, bias_dtype, c, v);
  if (residual) {
    float r[8];
    load8(residual + m * ldr + c, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store8(out + (long long)m * N + c, v);
}

// Gradients of both biases: sums over the rows of up to two matrices, 256 columns a CTA, a row a warp and step.  Where
// columns alone leave SMs idle the rows are dealt to `parts` CTAs, whose sums a second launch adds up in their order.
struct BiasGrad {
  const void* x;                // [M, cols], rows ld apart; null: none
  long long ld;
  int cols, dtype, add;         // of the output; add: to fp32
  void* out;
};
__device__ __forceinline__ void put_bias_grad(const BiasGrad& b, int c, float v) {
  if (b.dtype == PF_F32) {
    float* o = static_cast<float*>(b.out) + c;
    *o = b.add ? *o + v : v;
  } else if (b.dtype == PF_F16) {
    static_cast<__half*>(b.out)[c] = from_f32<__half>(v);
  } else {
    static_cast<__nv_bfloat16*>(b.out)[c] = from_f32<__nv_bfloat16>(v);
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
bias_grad_kernel(const BiasGrad b1, const BiasGrad b2, int blocks1, int M, int parts, float* __restrict__ ws) {
  after_previous();
  __shared__ float sums[8][256];
  const bool second = (int)blockIdx.x >= blocks1;
  const BiasGrad& b = second ? b2 : b1;
  const int c0 = ((int)blockIdx.x - (second ? blocks1 : 0)) * 256, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = c0 + lane * 8, part = blockIdx.y;
  const int begin = (int)((long long)M * part / parts), end = (int)((long long)M * (part + 1) / parts);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < b.cols) {
    const T* x = static_cast<const T*>(b.x) + c;
    for (int r = begin + warp; r < end; r += 32) {
      uint4 q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r + 8 * u < end) q[u] = __ldg(reinterpret_cast<const uint4*>(x + (long long)(r + 8 * u) * b.ld));
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r + 8 * u < end) {
          const T* e = reinterpret_cast<const T*>(&q[u]);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[j] += to_f32<T>(e[j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[warp][lane * 8 + j] = s[j];
  __syncthreads();
  const int col = c0 + threadIdx.x;
  if (col >= b.cols) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += sums[k][threadIdx.x];
  if (parts == 1) put_bias_grad(b, col, v);
  else ws[(long long)part * (b1.cols + b2.cols) + (second ? b1.cols : 0) + col] = v;
}
__global__ void __launch_bounds__(256)
bias_join_kernel(const BiasGrad b1, const BiasGrad b2, int parts, const float* __restrict__ ws) {
  after_previous();
  const int all = b1.cols + b2.cols, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  float v = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; ++k) v += ws[(long long)k * all + i];
  if (i < b1.cols) put_bias_grad(b1, i, v);
  else put_bias_grad(b2, i - b1.cols, v);
}
static int bias_parts(long long M, long long cols, int sm_count) {
  const long long blocks = (cols + 255) / 256 + 1, most = (M + 63) / 64, parts = (4ll * sm_count + blocks - 1) / blocks;
  return (int)(parts < most ? parts : most);
}

}  // namespace pf

using namespace pf;

// KiB of workspace of both directions for M rows; 0 where nothing is split
PF_API int pf_gated_mlp_scratch(int M, int D, int H, int N, int sm_count) {
  if (M <= 0) return 0;
  if (sm_count <= 0) sm_count = 148;
  long long most = 0;
  auto need = [&](long long n, long long k) {
    const int p = plan_parts(M, n, k, sm_count, false).parts;
    if (p > 1 && p * n > most) most = p * n;
  };
  need(2ll * H, D);
  need(N, H);
  need(H, N);
  need(D, 2ll * H);
  most *= M;
  const int p = bias_parts(M, 2ll * H + N, sm_count);
  if (p > 1 && p * (2ll * H + N) > most) most = p * (2ll * H + N);
  return (int)((most * 4 + 1023) / 1024);
}

namespace pf {
struct Block {
  int M, D, H, N, act, dtype, sms;
  int* status;
  float* ws;
  cudaStream_t st;
  FusedCall call(int n, int k, const void* a, long long lda, const void* b, long long ldb) const {
    FusedCall c;
    c.M = M; c.N = n; c.K = k; c.A = a; c.lda = lda; c.B = b; c.ldb = ldb;
    c.dtype = dtype; c.status = status; c.sm_count = sms; c.stream = st;
    return c;
  }
  PartPlan plan(long long n, long long k) const { return ws ? plan_parts(M, n, k, sms, false) : PartPlan(); }
  // A B^T in parts, more than one
  int in_parts(Job job, FusedCall c, PartPlan g, Parts& p) const {
    c.C = ws; c.ldc = c.N; c.out_dtype = PF_F32; c.split = g.parts; c.part_rows = M; c.tile = g.pair;
    p = {ws, g.parts, (long long)M * c.N};
    return fused_gemm(job, c);
  }
  unsigned grid(int width) const { return (unsigned)(((long long)M * (width / 8) + 127) / 128); }
  template <typename T> int bias_grads(BiasGrad b1, BiasGrad b2) const {
    for (BiasGrad* b : {&b1, &b2})
      if (!b->out) b->cols = 0;
    const int all = b1.cols + b2.cols;
    if (!all) return 0;
    const int blocks1 = (b1.cols + 255) / 256, blocks = blocks1 + (b2.cols + 255) / 256;
    const int parts = ws ? bias_parts(M, 2ll * H + N, sms) : 1;
    after(bias_grad_kernel<T>, dim3(blocks, parts), 256, 0, st)(b1, b2, blocks1, M, parts, ws);
    PF_CHECK_LAUNCH();
    if (parts > 1) {
      after(bias_join_kernel, (unsigned)((all + 255) / 256), 256, 0, st)(b1, b2, parts, (const float*)ws);
      PF_CHECK_LAUNCH();
    }
    return 0;
  }
  // dst [rows, cols] (+)= a^T b over the M rows
  int weight_grad(const void* a, long long lda, const void* b, long long ldb, void* dst, int rows, int cols,
                  int dst_dtype, int add) const {
    FusedCall c = call(cols, M, a, lda, b, ldb);
    c.M = rows; c.C = dst; c.ldc = cols; c.out_dtype = dst_dtype; c.accumulate = add;
    return fused_gemm(HEAD_DW, c);
  }
};

template <typename T>
static int mlp_forward(const Block& b, const void* x, const void* w1, const void* b1, int b1_dtype, const void* w2,
                       const void* b2, int b2_dtype, const void* residual, void* h, void* gu, void* y, long long ldx,
                       long long ldw1, long long ldw2, long long ldr) {
  int r;
  const PartPlan p1 = b.plan(2ll * b.H, b.D), p2 = b.plan(b.N, b.H);
  Parts p;
  if (p1.parts > 1) {
    if ((r = b.in_parts(PARTS_K, b.call(2 * b.H, b.D, x, ldx, w1, ldw1), p1, p))) return r;
    after(glu_join_kernel<T>, b.grid(b.H), 128, 0, b.st)(p, b1, b1_dtype, (T*)gu, (T*)h, b.M, b.H, b.act);
    PF_CHECK_LAUNCH();
  } else {
    FusedCall c = b.call(b.H, b.D, x, ldx, w1, ldw1);
    c.C = h; c.ldc = b.H; c.gu = gu; c.bias = b1; c.bias_dtype = b1_dtype; c.act = b.act;
    if ((r = fused_gemm(GLU_FWD, c))) return r;
  }
  if (p2.parts > 1) {
    if ((r = b.in_parts(PARTS_K, b.call(b.N, b.H, h, b.H, w2, ldw2), p2, p))) return r;
    after(row_join_kernel<T>, b.grid(b.N), 128, 0, b.st)(p, b2, b2_dtype, (const T*)residual, ldr, (T*)y, b.M, b.N);
    PF_CHECK_LAUNCH();
    return 0;
  }
  return pf_gemm(h, w2, y, b.M, b.N, b.H, b.H, ldw2, b.N, 0, 0, b.dtype, b.dtype, b2, b2_dtype, residual, ldr, nullptr,
                 0, 0, 0, 1.0f, b.status, b.sms, 0, nullptr, 0, b.st);
}

// what a backward writes; `add`: bits 1 dw1, 2 dw2, 4 db1, 8 db2
struct Grads {
  void *dx, *dw1, *dw2, *db1, *db2;
  int dw1_dtype, dw2_dtype, db1_dtype, db2_dtype, add;
};
template <typename T>
static int mlp_backward(const Block& b, const void* dy, const void* x, const void* w1, const void* w2, const void* gu,
                        void* dgu, void* h, const Grads& g, long long lddy, long long ldx, long long ldw1,
                        long long ldw2) {
  int r;
  const PartPlan p1 = b.plan(b.H, b.N), p2 = b.plan(b.D, 2ll * b.H);
  Parts p;
  if (p1.parts > 1) {
    if ((r = b.in_parts(PARTS_N, b.call(b.H, b.N, dy, lddy, w2, ldw2), p1, p))) return r;
    after(glu_join_bwd_kernel<T>, b.grid(b.H), 128, 0, b.st)(p, (const T*)gu, (T*)dgu, (T*)h, b.M, b.H, b.act);
    PF_CHECK_LAUNCH();
  } else {
    FusedCall c = b.call(b.H, b.N, dy, lddy, w2, ldw2);
    c.C = h; c.ldc = b.H; c.gu = const_cast<void*>(gu); c.dgu = dgu; c.act = b.act;
    if ((r = fused_gemm(GLU_BWD, c))) return r;
  }
  const long long ldgu = 2ll * b.H;
  if (g.dw2 && (r = b.weight_grad(dy, lddy, h, b.H, g.dw2, b.N, b.H, g.dw2_dtype, g.add & 2))) return r;
  if (g.dx) {
    if (p2.parts > 1) {
      if ((r = b.in_parts(PARTS_N, b.call(b.D, 2 * b.H, dgu, ldgu, w1, ldw1), p2, p))) return r;
      after(row_join_kernel<T>, b.grid(b.D), 128, 0, b.st)(p, (const void*)nullptr, 0, (const T*)nullptr, 0ll, (T*)g.dx,
                                                           b.M, b.D);
      PF_CHECK_LAUNCH();
    } else if ((r = pf_gemm(dgu, w1, g.dx, b.M, b.D, 2 * b.H, ldgu, ldw1, b.D, 0, 1, b.dtype, b.dtype, nullptr, 0,
                            nullptr, 0, nullptr, 0, 0, 0, 1.0f, b.status, b.sms, 0, nullptr, 0, b.st))) {
      return r;
    }
  }
  if (g.dw1 && (r = b.weight_grad(dgu, ldgu, x, ldx, g.dw1, 2 * b.H, b.D, g.dw1_dtype, g.add & 1))) return r;
  return b.bias_grads<T>({dgu, ldgu, 2 * b.H, g.db1_dtype, g.add & 4, g.db1},
                         {dy, lddy, b.N, g.db2_dtype, g.add & 8, g.db2});
}

static int mlp_block(Block& b, int M, int D, int H, int N, int act, int dtype, void* ws, int ws_kib, int* status,
                     int sm_count, void* stream) {
  if (dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (act < 1 || act > 3) return -1;
  if (M < 0 || D <= 0 || H <= 0 || N <= 0 || H > (1 << 29)) return -3;
  if (D % 8 || H % 8 || N % 8 || !on_vectors(ws)) return -2;
  b = {M, D, H, N, act, dtype, sm_count > 0 ? sm_count : 148, status, static_cast<float*>(ws),
       reinterpret_cast<cudaStream_t>(stream)};
  if (!ws || ws_kib < pf_gated_mlp_scratch(M, D, H, N, b.sms)) b.ws = nullptr;       // every product stays whole
  return 0;
}
}  // namespace pf

// x [M, D], w1 [2H, D], w2 [N, H], all with rows on 16 bytes, b1 [2H], b2 [N] and residual [M, N] may be null; D, H and N
// are multiples of 8.  h [M, H], gu [M, 2H] (null: gate and up are not kept) and y [M, N] are packed.
// act: 1 GELU (erf), 2 GELU (tanh), 3 SiLU.  ws: pf_gated_mlp_scratch.
PF_API int pf_gated_mlp_fwd(const void* x, const void* w1, const void* b1, int b1_dtype, const void* w2, const void* b2,
                            int b2_dtype, const void* residual, void* h, void* gu, void* y, void* ws, int ws_kib, int M,
                            int D, int H, int N, long long ldx, long long ldw1, long long ldw2, long long ldr, int act,
                            int dtype, int* status, int sm_count, void* stream) {
  Block b;
  const int r = mlp_block(b, M, D, H, N, act, dtype, ws, ws_kib, status, sm_count, stream);
  if (r || M == 0) return r;
  if (ldx % 8 || ldw1 % 8 || ldw2 % 8 || (residual && ldr % 8) || !on_vectors(x, w1, w2, residual, h, gu, y)) return -2;
  return dtype == PF_F16 ? mlp_forward<__half>(b, x, w1, b1, b1_dtype, w2, b2, b2_dtype, residual, h, gu, y, ldx, ldw1,
                                               ldw2, ldr)
                         : mlp_forward<__nv_bfloat16>(b, x, w1, b1, b1_dtype, w2, b2, b2_dtype, residual, h, gu, y, ldx,
                                                      ldw1, ldw2, ldr);
}

// From dy [M, N] and the kept gu: dx [M, D], dw1 [2H, D], dw2 [N, H], db1 [2H] and db2 [N], packed, each in 16 bits or fp32
// but dx; any of these may be null.  add: bits 1 dw1, 2 dw2, 4 db1, 8 db2 are added to, in fp32.  dgu [M, 2H] and h [M, H]
// are scratch.
PF_API int pf_gated_mlp_bwd(const void* dy, const void* x, const void* w1, const void* w2, const void* gu, void* dgu,
                            void* h, void* dx, void* dw1, void* dw2, void* db1, void* db2, void* ws, int ws_kib, int M,
                            int D, int H, int N, long long lddy, long long ldx, long long ldw1, long long ldw2, int act,
                            int dtype, int dw1_dtype, int dw2_dtype, int db1_dtype, int db2_dtype, int add, int* status,
                            int sm_count, void* stream) {
  Block b;
  const int r = mlp_block(b, M, D, H, N, act, dtype, ws, ws_kib, status, sm_count, stream);
  if (r) return r;
  const Grads g{dx, dw1, dw2, db1, db2, dw1_dtype, dw2_dtype, db1_dtype, db2_dtype, add};
  void* const out[4] = {dw1, dw2, db1, db2};
  const int types[4] = {dw1_dtype, dw2_dtype, db1_dtype, db2_dtype};
  const size_t sizes[4] = {2 * (size_t)H * D, (size_t)N * H, 2 * (size_t)H, (size_t)N};
  for (int i = 0; i < 4; ++i) {
    if (!out[i]) continue;
    const bool added = add >> i & 1;
    if (types[i] != PF_F32 && (added || types[i] < 0 || types[i] > 2 || (i < 2 && types[i] != dtype))) return -1;
    if (M == 0 && !added) {                             // nothing to add up
      cudaError_t e = cudaMemsetAsync(out[i], 0, sizes[i] * (types[i] == PF_F32 ? 4 : 2), b.st);
      if (e != cudaSuccess) return (int)e;
    }
  }
  if (M == 0) return 0;
  if (lddy % 8 || ldx % 8 || ldw1 % 8 || ldw2 % 8 || !on_vectors(dy, x, w1, w2, gu, dgu, h, dx, dw1, dw2)) return -2;
  return dtype == PF_F16 ? mlp_backward<__half>(b, dy, x, w1, w2, gu, dgu, h, g, lddy, ldx, ldw1, ldw2)
                         : mlp_backward<__nv_bfloat16>(b, dy, x, w1, w2, gu, dgu, h, g, lddy, ldx, ldw1, ldw2);
}
