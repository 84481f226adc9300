// Cross entropy of an output head, z = x W^T, without the logits.
//
// loss = log sum_v e^(z_v) - z_label over the rows that count, and with p = softmax(z), dz = g (p - onehot):
// dx = dz W, dW = dz^T x.
//
// Forward: the rows that count are gathered (prompts, padding and last tokens then cost nothing, and what they hold
// reaches nothing), one product whose epilogue keeps a reference and a sum of exponentials of each row and part of
// the words, and a fold over the parts.  Backward, piece by piece of the vocabulary: the product again, now with
// the sums at hand, leaves dz of a piece in 16 bits; from it come the piece's rows of dW, complete, and its share of
// dx, which adds up in fp32.  Four products of 2 rows D V operations where keeping the logits takes three.  Kept from
// forward to backward are the rows that count, 8 bytes of each and the index (sized for all rows).  Beside that, forward has
// 8 bytes for each row and 64 words, and backward dz of a piece, PIECE values or PIECE_WORDS of every row, and 4 bytes for
// each value of dx and part (2^26 values at most where there are several parts).  8192 rows of 4096 over 32000 words, half of
// which count: 67 MB kept, 100 at most in the forward and 795 in the backward, the gradients' 329 among them; with the logits
// kept it is 524, 524 and 1049.
//
// On a B200, bf16, forward and backward, 4096 values a row and 32000 words: 2048 rows 1.42 ms in a short run (four
// products 1384 us at 1.45 to 1.63 PFLOP/s, picking the rows 12, the fold 13, zeros for rows that do not count 6);
// 13 rows 0.23 ms, bound by what memory takes for W three times and dW once.  The fold reads 8 bytes of each row and 64
// words, 1/16 of what the logits in 16 bits would be.
//
// dz is rounded to 16 bits as p - onehot, times 2^15 for fp16: from 6e-5 / 2^15 on the probabilities keep all
// their bits, whatever the gradient of the loss is; that and the mean's factor come in 32 bits behind the products.
#include <algorithm>
#include "common.cuh"
#include "api.h"
#include "fused_gemm.h"

namespace pf {

// index: [0] rows that count, [1] CTAs of the fold that have finished, then the rows that count, their labels, and
// where each row is among them (or -1)
constexpr int HEAD_HEADER = 4;
struct HeadIndex {
  int *count, *list, *labels, *at;
};
static long long padded_rows(long long N) { return (N + 255) / 256 * 256; }
static HeadIndex head_index(int* index, long long N) {
  const long long Mp = padded_rows(N);
  return {index, index + HEAD_HEADER, index + HEAD_HEADER + Mp, index + HEAD_HEADER + 2 * Mp};
}

// One CTA: ranks of the rows that count, 4 rows a thread at a time.  8192 rows take two rounds.
__global__ void __launch_bounds__(1024)
head_rows_kernel(const long long* __restrict__ target, HeadIndex ix, float* __restrict__ loss_of_row, int N,
                 long long V, long long ignore_index) {
  after_previous();
  __shared__ int sums[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int base = 0;
  for (int n0 = 0; n0 < N; n0 += 4096) {
    const int n = n0 + threadIdx.x * 4;
    int label[4], mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long t = n + j < N ? target[n + j] : -1;
      label[j] = t >= 0 && t < V && t != ignore_index ? (int)t : -1;
      mine += label[j] >= 0;
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    const int other = sums[lane];
    const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0);
    const int all = __reduce_add_sync(0xffffffffu, other);
    int at = base + ahead + before - mine;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n + j >= N) break;
      const bool in = label[j] >= 0;
      ix.at[n + j] = in ? at : -1;
      if (in) {
        ix.list[at] = n + j;
        ix.labels[at] = label[j];
        ++at;
      } else if (loss_of_row) {
        loss_of_row[n + j] = 0.f;
      }
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    ix.count[0] = base;
    ix.count[1] = 0;
  }
}

// A row of x into the packed rows, or zeros; a warp.
template <typename T>
__device__ __forceinline__ void put_row(const T* src, T* dst, int D, int Dp, int vec) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    uint4* dv = reinterpret_cast<uint4*>(dst);
    const uint4* sv = reinterpret_cast<const uint4*>(src);
    const int nv = Dp / 8;
    for (int c = lane; c < nv; c += 128) {
      uint4 q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * 32 < nv) q[u] = src ? __ldg(sv + c + u * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c + u * 32 < nv) dv[c + u * 32] = q[u];
    }
  } else {
    for (int c = lane; c < Dp; c += 32) dst[c] = src && c < D ? src[c] : from_f32<T>(0.f);
  }
}
// A reduction over rows reads whole blocks of 64: zeros behind the last row
__device__ __forceinline__ int zeroed_rows(int count, int Mp) { return min(Mp, (count + 63) / 64 * 64); }

// xc[i] = x[list[i]], a warp per row
template <typename T>
__global__ void __launch_bounds__(256)
head_gather_kernel(const T* __restrict__ x, T* __restrict__ xc, HeadIndex ix, int Mp, int D, int Dp, long long ldx,
                   int vec) {
  after_previous();
  const int count = *ix.count, i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= zeroed_rows(count, Mp)) return;
  put_row(i < count ? x + ix.list[i] * ldx : nullptr, xc + (long long)i * Dp, D, Dp, vec);
}

// Both at once for calls of few rows, where a launch costs more than that every CTA, of 8 rows, looks at all labels.
constexpr int PICK_ROWS = 4096;
template <typename T>
__global__ void __launch_bounds__(256)
head_pick_kernel(const long long* __restrict__ target, const T* __restrict__ x, T* __restrict__ xc, HeadIndex ix,
                 float* __restrict__ loss_of_row, int N, int Mp, int D, int Dp, long long ldx, long long V,
                 long long ignore_index, int vec) {
  after_previous();
  __shared__ int sums[2][8];
  __shared__ int labels[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = blockIdx.x * 8;
  int before = 0, all = 0;
  for (int n = threadIdx.x; n < N; n += 256) {
    const long long t = target[n];
    const bool in = t >= 0 && t < V && t != ignore_index;
    all += in;
    before += in && n < row0;
    if (n >= row0 && n < row0 + 8) labels[n - row0] = in ? (int)t : -1;
  }
  all = __reduce_add_sync(0xffffffffu, all);
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) { sums[0][warp] = all; sums[1][warp] = before; }
  __syncthreads();
  all = before = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) { all += sums[0][k]; before += sums[1][k]; }
  const int row = row0 + warp;
  if (row < N) {
    const int label = labels[warp];
    int at = before;
    for (int k = 0; k < warp; ++k) at += labels[k] >= 0;
    if (lane == 0) {
      ix.at[row] = label >= 0 ? at : -1;
      if (label >= 0) {
        ix.list[at] = row;
        ix.labels[at] = label;
      } else if (loss_of_row) {
        loss_of_row[row] = 0.f;
      }
    }
    if (label >= 0) put_row(x + row * ldx, xc + (long long)at * Dp, D, Dp, vec);
  }
  if (row >= all && row < zeroed_rows(all, Mp)) put_row<T>(nullptr, xc + (long long)row * Dp, D, Dp, vec);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    ix.count[0] = all;
    ix.count[1] = 0;
  }
}

// Joins the parts of ROWS rows: 1024 / ROWS threads share the parts of a row, with lanes on neighbouring rows; then a warp
// has a row at a time.  Few parts would leave most of 128 threads with none (4 parts of 13965 rows: 40 us with 8 rows a CTA,
// 10 with 128).  References are integers: 2^(a - b) is exact.  The row's loss is formed in 64 bits; `sums` gets a CTA's sum
// of them, and the CTA that finishes last adds those up in their order.
constexpr int FOLD_ROWS = 8, FOLD_MOST_ROWS = 128, FOLD_FEW_PARTS = 32;
__device__ __forceinline__ void join(float& ref, float& sum, float ref2, float sum2) {
  const float m = fmaxf(ref, ref2), sub = m == -INFINITY ? 0.f : m;
  sum = sum * exp2f(ref - sub) + sum2 * exp2f(ref2 - sub);
  ref = m;
}
template <int ROWS>
__global__ void __launch_bounds__(1024)
head_fold_kernel(const RowStat* __restrict__ parts, long long pitch, int n_parts, const float* __restrict__ picked,
                 HeadIndex ix, RowStat* __restrict__ stats, float* __restrict__ loss, float* __restrict__ inv,
                 double* __restrict__ sums, int reduction) {
  after_previous();
  constexpr int LANES = 1024 / ROWS;
  __shared__ RowStat all[ROWS][LANES + 1];
  __shared__ double rows[ROWS > 32 ? ROWS : 32];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = *ix.count, row0 = blockIdx.x * ROWS;
  if (row0 < count) {
    const int r = threadIdx.x % ROWS, l = threadIdx.x / ROWS, row = row0 + r;
    float ref = -INFINITY, sum = 0.f;
    if (row < count) {
      const RowStat* src = parts + row;
      for (int k = l; k < n_parts; k += 8 * LANES) {
        RowStat q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (k + LANES * u < n_parts) q[u] = src[(k + LANES * u) * pitch];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (k + LANES * u < n_parts) join(ref, sum, q[u].ref, q[u].inv);
      }
    }
    all[r][l] = {ref, sum};
  }
  __syncthreads();
  for (int r = warp; r < ROWS; r += 32) {
    const int row = row0 + r;
    if (lane == 0) rows[r] = 0.0;
    if (row >= count) continue;
    float ref = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < (LANES + 31) / 32; ++k)
      if (LANES >= 32 || lane < LANES) join(ref, sum, all[r][lane + 32 * k].ref, all[r][lane + 32 * k].inv);
#pragma unroll
    for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1)
      join(ref, sum, __shfl_xor_sync(0xffffffffu, ref, o), __shfl_xor_sync(0xffffffffu, sum, o));
    if (lane == 0) {
      if (ref == -INFINITY) ref = 0.f;
      stats[row] = {ref, 1.f / sum};
      constexpr double ln2 = 0.69314718055994531;
      const double l = (log2((double)sum) + (double)ref - (double)picked[row] * (double)1.4426950408889634f) * ln2;
      rows[r] = l;
      if (reduction == 0) loss[ix.list[row]] = (float)l;
    }
  }
  if (reduction == 0) return;                           // of no rows the losses have no address
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < ROWS; ++i) s += rows[i];
    sums[blockIdx.x] = s;
    __threadfence();
    last = atomicAdd(ix.count + 1, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int i = threadIdx.x; i < (count + ROWS - 1) / ROWS; i += 1024)
    s += reinterpret_cast<volatile double*>(sums)[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) rows[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < 32; ++i) s += rows[i];
    const double n = reduction == 1 ? (double)max(count, 1) : 1.0;
    *loss = (float)(s / n);
    *inv = (float)(1.0 / n);
  }
}

// Gradients that arrive row by row, of the rows that count: divided by a power of two near the largest number among
// them, which goes into `scale`, so that 16 bits hold the products.
__global__ void __launch_bounds__(1024)
head_factor_kernel(const float* __restrict__ g, long long step, HeadIndex ix, float* __restrict__ factor,
                   float* __restrict__ scale) {
  after_previous();
  __shared__ float tops[32];
  const int count = *ix.count;
  float top = 0.f;
  for (int i = threadIdx.x; i < count; i += 1024) {
    const float v = g[ix.list[i] * step];
    factor[i] = v;
    if (fabsf(v) < INFINITY) top = fmaxf(top, fabsf(v));
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  top = warp_max(tops[threadIdx.x & 31]);
  int e = 0;
  if (top > 0.f) {
    frexpf(top, &e);
    e = max(-120, min(120, e));
  }
  const float down = ldexpf(1.f, -e);
  for (int i = threadIdx.x; i < count; i += 1024) factor[i] *= down;
  if (threadIdx.x == 0) *scale = ldexpf(1.f, e);
}

// dx[n] = the sum over parts of acc at the row's place, times the scale; zeros for rows that do not count.  A warp has
// DX_COLUMNS of a row.
constexpr int DX_COLUMNS = 512;
template <typename T>
__global__ void __launch_bounds__(256)
head_dx_kernel(const float* __restrict__ acc, T* __restrict__ dx, HeadIndex ix, long long N, int D, int Dp,
               const int* __restrict__ parts_word, const float* __restrict__ scale, const float* __restrict__ scale2,
               float scale3, int vec, int direct) {
  after_previous();
  const int parts = *parts_word;
  const long long part_size = (long long)rows_of_part(*ix.count) * Dp;
  const float s = *scale * (scale2 ? *scale2 : 1.f) * scale3;
  const int lane = threadIdx.x & 31;
  const long long n = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (n >= N) return;
  const int at = ix.at[n];
  if (at >= 0 && direct && parts == 1) return;          // the product has written it
  const float* src = acc + (long long)at * Dp;
  T* dst = dx + n * D;
  for (int begin = blockIdx.y * DX_COLUMNS; begin < D; begin += gridDim.y * DX_COLUMNS) {
    const int end = min(D, begin + DX_COLUMNS);
    if (vec) {
      float v[2][8] = {};
      if (at >= 0) {
#pragma unroll 2
        for (int k = 0; k < parts; ++k) {
          float4 q[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int c = begin + lane * 8 + 256 * u;
            const float4* from = reinterpret_cast<const float4*>(src + k * part_size + c);
            if (c < end) { q[u][0] = from[0]; q[u][1] = from[1]; }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float* e = reinterpret_cast<const float*>(q[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] += e[j];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = begin + lane * 8 + 256 * u;
        uint4 q;
        T* e = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(at >= 0 ? v[u][j] * s : 0.f);
        if (c < end) *reinterpret_cast<uint4*>(dst + c) = q;
      }
    } else {
      for (int c = begin + lane; c < end; c += 32) {
        float v = 0.f;
        if (at >= 0) {
          for (int k = 0; k < parts; ++k) v += src[k * part_size + c];
          v *= s;
        }
        dst[c] = from_f32<T>(v);
      }
    }
  }
}

// Values of dz that are alive at one time: 256 MB, which is all of dz where rows times words are no more.  Pieces of fewer
// than 4096 words would have dx added to too often (8 bytes of each of its values a piece, for 6 x 4096 operations), so that
// from 32768 rows on dz takes 8 KB a row: 1 GB at 131072.
constexpr long long PIECE = 128ll << 20;
constexpr int PIECE_WORDS = 4096;

}  // namespace pf

using namespace pf;

static bool head_sizes_ok(long long N, long long V, long long D) {
  return N >= 0 && V > 0 && D > 0 && N <= (1ll << 28) && V <= (1ll << 28) && D <= (1ll << 20);
}

// int32 values of `index`
PF_API int pf_head_index(long long N) {
  return N < 0 || N > (1ll << 28) ? -3 : (int)(HEAD_HEADER + 2 * padded_rows(N) + N);
}

// KiB of scratch of pf_head_fwd
PF_API int pf_head_scratch(long long N, long long V) {
  if (!head_sizes_ok(N, V, 1)) return -3;
  const long long Mp = padded_rows(N), parts = (V + HEAD_PART - 1) / HEAD_PART;
  const long long kib = (parts * Mp * 8 + Mp * 4 + (Mp / FOLD_ROWS + 1) * 8 + 1023) / 1024 + 1;
  return kib > 0x7fffffffll ? -3 : (int)kib;
}

// Words of a piece of the backward, all pieces as near in size as multiples of 256 allow
PF_API int pf_head_words(long long N, long long V) {
  if (!head_sizes_ok(N, V, 1)) return -3;
  const long long Mp = N > 0 ? padded_rows(N) : 256;
  long long most = PIECE / Mp / 256 * 256;
  if (most < PIECE_WORDS) most = PIECE_WORDS;
  const long long pieces = (V + most - 1) / most;
  return (int)(((V + pieces - 1) / pieces + 255) / 256 * 256);
}

static PartPlan head_plan(long long N, long long V, int D, int sm_count) {
  const long long words = pf_head_words(N, V);
  return N > 0 ? plan_parts(N, (D + 7) / 8 * 8, words < V ? words : V, sm_count > 0 ? sm_count : 148, true) : PartPlan();
}

// Parts in which the reduction of dx over the words of a piece is split if all rows count, where they leave SMs idle.  In
// the memory of these go more parts of fewer rows.
PF_API int pf_head_parts(long long N, long long V, int D, int sm_count) {
  return head_sizes_ok(N, V, D) ? head_plan(N, V, D, sm_count).parts : -3;
}

// Rows of the tiles of that product: 256 of a pair of CTAs, or 128
PF_API int pf_head_tile(long long N, long long V, int D, int sm_count) {
  return !head_sizes_ok(N, V, D) ? -3 : head_plan(N, V, D, sm_count).pair ? 256 : 128;
}

// x [N, D] (rows ldx apart), w [V, Dp] (Dp: D up to a multiple of 8, filled with zeros; rows ldw apart), target [N].
// xc [Mp, Dp] (Mp: N up to a multiple of 256), index: pf_head_index, stats [Mp, 2] are for the backward.
// reduction 0: loss [N], 0 where no label counts; 1: mean over the rows that count, 2: their sum, both with inv.
PF_API int pf_head_fwd(const void* x, const void* w, const void* target, void* xc, void* index, void* stats, void* loss,
                       void* inv, void* scratch, long long N, long long V, int D, int Dp, long long ldx, long long ldw,
                       long long ignore_index, int reduction, int dtype, int* status, int sm_count, void* stream) {
  if (dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (!head_sizes_ok(N, V, D)) return -3;
  if (Dp % 8 || Dp < D || !on_vectors(w, xc, scratch) || ldw % 8) return -2;
  if (sm_count <= 0) sm_count = 148;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long Mp = padded_rows(N);
  const HeadIndex ix = head_index(static_cast<int*>(index), N);
  const int n_parts = (int)((V + HEAD_PART - 1) / HEAD_PART);
  RowStat* parts = static_cast<RowStat*>(scratch);
  double* sums = reinterpret_cast<double*>(parts + n_parts * Mp);
  float* picked = reinterpret_cast<float*>(sums + Mp / FOLD_ROWS + 1);
  float* each = reduction == 0 ? static_cast<float*>(loss) : nullptr;
  const int vec = D == Dp && ldx % 8 == 0 && on_vectors(x);
  const unsigned eights = (unsigned)(Mp / 8);
  auto pick = [&](auto type) -> int {
    using T = decltype(type);
    after(head_pick_kernel<T>, eights, 256, 0, st)((const long long*)target, (const T*)x, (T*)xc, ix, each, (int)N,
                                                   (int)Mp, D, Dp, ldx, V, ignore_index, vec);
    PF_CHECK_LAUNCH();
    return 0;
  };
  auto gather = [&](auto type) -> int {
    using T = decltype(type);
    after(head_gather_kernel<T>, eights, 256, 0, st)((const T*)x, (T*)xc, ix, (int)Mp, D, Dp, ldx, vec);
    PF_CHECK_LAUNCH();
    return 0;
  };
  int r = 0;
  if (N > 0 && N <= PICK_ROWS) {
    r = dtype == PF_F16 ? pick(__half()) : pick(__nv_bfloat16());
  } else {
    after(head_rows_kernel, 1, 1024, 0, st)((const long long*)target, ix, each, (int)N, V, ignore_index);
    PF_CHECK_LAUNCH();
    if (N > 0) r = dtype == PF_F16 ? gather(__half()) : gather(__nv_bfloat16());
  }
  if (r) return r;
  if (N > 0) {
    FusedCall c;
    c.M = (int)N; c.N = (int)V; c.K = Dp; c.A = xc; c.B = w; c.lda = Dp; c.ldb = ldw; c.dtype = dtype;
    c.rows = ix.count; c.labels = ix.labels; c.parts = parts; c.part_pitch = Mp; c.picked = picked;
    c.status = status; c.sm_count = sm_count; c.stream = st;
    if ((r = fused_gemm(HEAD_STATS, c))) return r;
  }
  const auto fold = [&](auto* kernel, int rows) -> int {
    const unsigned grid = (unsigned)(N > 0 ? (N + rows - 1) / rows : 1);
    after(kernel, grid, 1024, 0, st)((const RowStat*)parts, Mp, n_parts, (const float*)picked, ix, (RowStat*)stats,
                                     (float*)loss, (float*)inv, sums, reduction);
    PF_CHECK_LAUNCH();
    return 0;
  };
  // 128 rows a CTA where each of its 8 threads has few parts and there are rows for all SMs
  if (n_parts <= FOLD_FEW_PARTS && N >= (long long)sm_count * FOLD_MOST_ROWS / 4)
    return fold(head_fold_kernel<FOLD_MOST_ROWS>, FOLD_MOST_ROWS);
  return fold(head_fold_kernel<FOLD_ROWS>, FOLD_ROWS);
}

// dloss: one value, or with by_row the rows' dloss[n * dloss_step]; inv as the forward left it.
// dx [N, D] packed, dw [V, Dp] (rows lddw apart, added to where accumulate); either may be null.
// dz [Mp, pf_head_words], acc [pf_head_parts * Mp * Dp + 1] (with dx), factor [Mp + 1] (with by_row) are scratch.
PF_API int pf_head_bwd(const void* dloss, const void* inv, const void* xc, const void* w, void* index, const void* stats,
                       void* dx, void* dw, void* dz, void* acc, void* factor, long long N, long long V, int D, int Dp,
                       long long dloss_step, long long ldw, long long lddw, int by_row, int accumulate, int dtype,
                       int dw_dtype, int* status, int sm_count, void* stream) {
  if (dtype != PF_F16 && dtype != PF_BF16) return -1;
  if (dw && dw_dtype != dtype && dw_dtype != PF_F32) return -1;
  if (!head_sizes_ok(N, V, D)) return -3;
  if (Dp % 8 || Dp < D || !on_vectors(w, xc, dw, dz, acc) || ldw % 8 || (dw && lddw % 8)) return -2;
  if (accumulate && dw && dw_dtype != PF_F32) return -1;
  if (sm_count <= 0) sm_count = 148;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long Mp = padded_rows(N);
  const HeadIndex ix = head_index(static_cast<int*>(index), N);
  const PartPlan plan = head_plan(N, V, D, sm_count);
  const int words = pf_head_words(N, V), parts = plan.parts, tile = plan.pair;
  const float unit = dtype == PF_F16 ? 32768.f : 1.f;
  const float* scale = static_cast<const float*>(dloss);
  const float* scale2 = static_cast<const float*>(inv);
  float* each = nullptr;
  if (by_row) {
    each = static_cast<float*>(factor);
    scale = each + Mp;
    scale2 = nullptr;
    after(head_factor_kernel, 1, 1024, 0, st)((const float*)dloss, dloss_step, ix, each, each + Mp);
    PF_CHECK_LAUNCH();
  }
  FusedCall base;
  base.dtype = dtype; base.rows = ix.count; base.status = status; base.sm_count = sm_count; base.stream = st;
  int* parts_word = reinterpret_cast<int*>(static_cast<float*>(acc) + parts * Mp * Dp);
  // One piece in one part is dx itself, by way of the rows' list: 13965 rows of 4096 over 256 words, both directions, 365 us
  // with 32 bits in between and 295 without.
  const int vec = D == Dp && on_vectors(dx), direct = vec && words >= V;
  PartRule rule;                                        // of the first piece; no other has more words
  rule.tile_rows = tile ? 256 : 128; rule.columns = (Dp + rule.tile_rows - 1) / rule.tile_rows;
  rule.slots = tile ? sm_count / 2 : sm_count;
  rule.kb = (int)(((words < V ? words : V) + 63) / 64); rule.planned = parts;
  rule.rows = (int)std::min<long long>(parts * Mp, 0x7fffffff);
  const size_t es = dw_dtype == PF_F32 ? 4 : 2;
  if (N == 0) {                                         // nothing to add up, and no rows for a tensor map
    return dw && !accumulate ? (int)cudaMemsetAsync(dw, 0, (size_t)V * lddw * es, st) : 0;
  }
  for (long long v0 = 0; v0 < V; v0 += words) {
    const int n = (int)(V - v0 < words ? V - v0 : words);
    const char* wp = static_cast<const char*>(w) + v0 * ldw * 2;
    int r;
    FusedCall z = base;
    z.M = (int)N; z.N = n; z.K = Dp; z.A = xc; z.B = wp; z.lda = Dp; z.ldb = ldw; z.C = dz; z.ldc = words;
    z.labels = ix.labels; z.first = (int)v0; z.stats = static_cast<const RowStat*>(stats); z.factor = each;
    z.unit = unit;
    if ((r = fused_gemm(HEAD_DZ, z))) return r;
    if (dx) {
      FusedCall c = base;
      c.M = (int)N; c.N = Dp; c.K = n; c.A = dz; c.B = wp; c.lda = words; c.ldb = ldw; c.C = acc; c.ldc = Dp;
      c.out_dtype = PF_F32; c.split = parts; c.tile = tile; c.rule = rule; c.accumulate = v0 > 0;
      c.parts_word = v0 ? nullptr : parts_word;
      if (direct) { c.direct = dx; c.list = ix.list; c.scale = scale; c.scale2 = scale2; c.scale3 = 1.f / unit; }
      if ((r = fused_gemm(PARTS_N, c))) return r;
    }
    if (dw) {
      FusedCall c = base;
      c.M = n; c.N = Dp; c.K = (int)N; c.A = dz; c.B = xc; c.lda = words; c.ldb = Dp;
      c.C = static_cast<char*>(dw) + v0 * lddw * es; c.ldc = lddw; c.out_dtype = dw_dtype; c.accumulate = accumulate;
      c.scale = scale; c.scale2 = scale2; c.scale3 = 1.f / unit;
      if ((r = fused_gemm(HEAD_DW, c))) return r;
    }
  }
  if (dx) {
    // columns side by side as far as rows leave SMs idle
    const long long rows = (N + 7) / 8, columns = (D + DX_COLUMNS - 1) / DX_COLUMNS;
    const long long most = (8ll * sm_count + rows - 1) / rows;
    const dim3 grid((unsigned)rows, (unsigned)std::min(columns, most));
    if (dtype == PF_F16)
      after(head_dx_kernel<__half>, grid, 256, 0, st)((const float*)acc, (__half*)dx, ix, N, D, Dp, (const int*)parts_word,
                                                      scale, scale2, 1.f / unit, vec, direct);
    else
      after(head_dx_kernel<__nv_bfloat16>, grid, 256, 0, st)((const float*)acc, (__nv_bfloat16*)dx, ix, N, D, Dp,
                                                             (const int*)parts_word, scale, scale2, 1.f / unit, vec, direct);
    PF_CHECK_LAUNCH();
  }
  return 0;
}
