// Embedded tokens with a scale, and the gradient of the table by sorted tokens.
//
// out[t] = scale table[id_t];  dtable[v] = scale sum over t with id_t = v of dout[t].
//
// Both are bound by memory: forward the rows that are named and the output, backward dout and the whole gradient
// table, most of whose rows are zeros.  Sums go over the tokens in their order (the sort is stable) in 32 bits, in
// windows of the sorted tokens: a run of one id is summed and written by the window in which it starts, unless it is
// longer than several windows; then every window leaves its part, and the parts are added in their order.  So the same
// tokens give the same bits, a row is written once and rounded once, and a padding token that a third of the batch
// shares is summed by as many CTAs as it has windows.  Ids outside the table have zeros and no gradient.
//
// On a B200, 8192 tokens of 32000 rows of 4096 in fp32, values in bf16: forward 21 us (9.4 TB/s of rows read, some from
// L2, and values written), backward 108: zeros for the 524 MB table 72 (7.3 TB/s), with the sort's 20 beside them, sums
// 32, joins 6.  65536 tokens of 128000 rows of 2048, a third of them one id: forward 50, backward 168: zeros 74 beside the
// sort's 52 to 74, sums 71, joins 21, each CTA of which adds up hundreds of parts.
#include <algorithm>
#include <type_traits>
#include "common.cuh"
#include "api.h"

namespace pf {

// V values of a row; 8 of fp32 move as one access of 32 bytes: two of 16 at a distance of 32 would write each sector twice.
template <typename T, int V> struct Vec {
  float v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 8 && sizeof(T) == 2) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(e[j]);
    } else if constexpr (V == 8) {
      asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                   : "l"(p) : "memory");
    } else {
      v[0] = to_f32<T>(p[0]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 8 && sizeof(T) == 2) {
      uint4 q;
      T* e = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
      *reinterpret_cast<uint4*>(p) = q;
    } else if constexpr (V == 8) {
      asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                   "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    } else {
      p[0] = from_f32<T>(v[0]);
    }
  }
};
// the same as it was loaded: 16-bit values stay packed until they are added
template <typename T, int V> struct Raw {
  static constexpr bool PACKED = V == 8 && sizeof(T) == 2;
  typename std::conditional<PACKED, uint4, Vec<T, V>>::type q;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (PACKED) q = __ldg(reinterpret_cast<const uint4*>(p));
    else q.load(p);
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (PACKED) return to_f32<T>(reinterpret_cast<const T*>(&q)[j]);
    else return q.v[j];
  }
};
// whether rows of D values start on the 8-value accesses of their type
static bool on_rows(const void* p, int D, int dtype) {
  return D % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & (dtype == PF_F32 ? 31 : 15)) == 0;
}

// 2^lanes_log threads a row, up to eight vectors of V values each requested before any is written.
template <typename TT, typename T, int V>
__global__ void __launch_bounds__(256)
scaled_embed_kernel(const TT* __restrict__ table, const long long* __restrict__ ids, T* __restrict__ out,
                    long long tokens, int lanes_log, int D, long long words, float scale) {
  after_previous();
  constexpr int U = V == 8 && sizeof(TT) == 4 ? 4 : 8;
  const long long t = ((long long)blockIdx.x * 256 + threadIdx.x) >> lanes_log;
  if (t >= tokens) return;
  const long long id = __ldg(ids + t);
  const bool there = id >= 0 && id < words;
  const int step = V << lanes_log;
  const TT* src = table + (there ? id : 0) * D;
  T* dst = out + t * D;
  for (int c0 = (threadIdx.x & ((1 << lanes_log) - 1)) * V; c0 < D; c0 += U * step) {
    Raw<TT, V> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * step;
      if (c < D && there) q[u].load(src + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * step;
      if (c < D) {
        Vec<T, V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = there ? q[u].at(j) * scale : 0.f;
        r.store(dst + c);
      }
    }
  }
}

// Stable sort of the tokens by id, least digit first, in one cluster: CTAs have neighbouring stretches of the order so
// far and warps neighbouring stretches of those; a warp ranks 32 tokens at a time by matching digits.  The CTAs read one
// another's counts through distributed shared memory; the order goes through global memory (L2).
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_BINS = 512;
constexpr int SORT_SMEM = (SORT_WARPS * SORT_BINS + 2 * SORT_BINS + 64) * 4;

template <int CTAS>
__global__ void __launch_bounds__(SORT_THREADS)
sort_tokens_kernel(const long long* __restrict__ ids, int N, int words, int bits, int passes, int* __restrict__ order,
                   int* __restrict__ other, int* __restrict__ keys, int2* __restrict__ runs) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;                              // [warp][bin]
  int* totals = counts + SORT_WARPS * SORT_BINS;        // [bin], read by the other CTAs
  int* starts = totals + SORT_BINS;
  int* sums = starts + SORT_BINS;
  after_previous();
  let_next_start();                                     // zeros for the table, which need nothing of this
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS > 1 ? (int)cluster_ctarank() : 0;
  const int bins = 1 << bits;
  // stretches of whole rounds of 32 tokens a warp
  const int per_warp = ((N + CTAS * SORT_WARPS - 1) / (CTAS * SORT_WARPS) + 31) / 32 * 32;
  const long long lo = (long long)(rank * SORT_WARPS + warp) * per_warp;
  const int begin = (int)(lo < N ? lo : N), end = (int)(lo + per_warp < N ? lo + per_warp : N);
  auto key_of = [&](int t) {
    const long long id = __ldg(ids + t);
    return id >= 0 && id < words ? (int)id : words;     // ids outside the table come last
  };
  auto all_sync = [&]() {
    __threadfence();
    if (CTAS > 1) cluster_sync();
    else __syncthreads();
  };
  all_sync();
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    // the order ends in `order`: an odd number of passes starts by writing there
    int* dst = ((passes - pass) & 1) ? order : other;
    const int* src = ((passes - pass) & 1) ? other : order;
    int* mine = counts + warp * SORT_BINS;
    for (int b = lane; b < bins; b += 32) mine[b] = 0;
    __syncwarp();
    // rounds of 32 tokens, 8 at a time so that their loads overlap; a stretch of no more keeps them for the second turn
    int tok[8], key[8];
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + 32 * u + lane;
        tok[u] = i < end ? (pass ? __ldcg(src + i) : i) : -1;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) key[u] = tok[u] >= 0 ? key_of(tok[u]) : -1;
    };
    for (int i0 = begin; i0 < end; i0 += 256) {
      load(i0);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (i0 + 32 * u >= end) break;                  // uniform across the warp
        const bool in = tok[u] >= 0;
        const int digit = in ? (key[u] >> shift) & (bins - 1) : bins;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (in && lane == __ffs(same) - 1) mine[digit] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) {
      int s = 0;
      for (int w = 0; w < SORT_WARPS; ++w) {
        const int n = counts[w * SORT_BINS + b];
        counts[w * SORT_BINS + b] = s;
        s += n;
      }
      totals[b] = s;
    }
    all_sync();
    // where each bin starts: all tokens of the bins before it, then those of the bin in the CTAs before this one
    int all = 0, before = 0;
    if ((int)threadIdx.x < bins) {
      for (int r = 0; r < CTAS; ++r) {
        int n;
        if (CTAS > 1) {
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(mapa_u32(totals + threadIdx.x, r)) : "memory");
        } else {
          n = totals[threadIdx.x];
        }
        all += n;
        if (r < rank) before += n;
      }
    }
    int up = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += n;
    }
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
    if ((int)threadIdx.x < bins) starts[threadIdx.x] = ahead + up - all + before;
    __syncthreads();
    for (int b = lane; b < bins; b += 32) mine[b] += starts[b];
    __syncwarp();
    for (int i0 = begin; i0 < end; i0 += 256) {
      if (end - begin > 256) load(i0);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (i0 + 32 * u >= end) break;
        const bool in = tok[u] >= 0;
        const int digit = in ? (key[u] >> shift) & (bins - 1) : bins;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (in) {
          const int to = mine[digit] + __popc(same & ((1u << lane) - 1));
          __stcg(dst + to, tok[u]);
          if (pass == passes - 1) __stcg(keys + to, key[u]);
        }
        __syncwarp();
        if (in && lane == __ffs(same) - 1) mine[digit] += __popc(same);
        __syncwarp();
      }
    }
    all_sync();
  }
  // where the run of each id starts and ends
#pragma unroll 4
  for (int i = rank * SORT_THREADS + threadIdx.x; i < N; i += CTAS * SORT_THREADS) {
    const int key = __ldcg(keys + i);
    const int left = i > 0 ? __ldcg(keys + i - 1) : -1, right = i < N - 1 ? __ldcg(keys + i + 1) : -1;
    if (key < words && left != key) runs[key].x = i;
    if (key < words && right != key) runs[key].y = i + 1;
  }
}

// Zeros for a table's gradient, 16 bytes a thread and store, beside the sort: rows that tokens name are written again
// behind both.
__global__ void __launch_bounds__(512)
table_zeros_kernel(uint4* __restrict__ dst, long long n, unsigned char* __restrict__ tail, int bytes) {
  const long long i0 = (long long)blockIdx.x * (512 * 8) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (i0 + u * 512 < n) dst[i0 + u * 512] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == 0 && (int)threadIdx.x < bytes) tail[threadIdx.x] = 0;
  if (blockIdx.x == gridDim.x - 1) after_previous();    // what comes next finds the sort completed, too
}

// Sums of windows of the sorted tokens.  `lanes` threads (a power of two) share a row of V-wide vectors, 128 / lanes
// windows a CTA.
struct TableGrad {
  const int* keys;
  const int* order;
  const int2* runs;
  int N, words, D, window, lanes_log, slices;
  float scale;
  int accumulate;
  float* parts;                 // [window][2][D]: of a long run that came in, of one that goes on
  int most;                     // tokens of a run that is not long
};

template <typename TT, int V>
__device__ __forceinline__ void put_row(TT* dtable, const TableGrad& p, int key, int c, Vec<TT, V> r) {
  TT* dst = dtable + (long long)key * p.D + c;
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] *= p.scale;
  if (p.accumulate) {
    Vec<TT, V> old;
    old.load(dst);
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] += old.v[j];
  }
  r.store(dst);
}

template <typename T, typename TT, int V>
__global__ void __launch_bounds__(128)
table_grad_kernel(const T* __restrict__ dout, TT* __restrict__ dtable, const TableGrad p) {
  after_previous();
  constexpr int U = V == 8 && sizeof(T) == 4 ? 4 : 8;
  const int lanes = 1 << p.lanes_log;
  const int slice = blockIdx.x % p.slices;
  const long long w = (long long)(blockIdx.x / p.slices) * (128 >> p.lanes_log) + (threadIdx.x >> p.lanes_log);
  const long long b = w * p.window;
  const int c = (slice * lanes + (threadIdx.x & (lanes - 1))) * V;
  if (b >= p.N || c >= p.D) return;
  int begin = (int)b, end = min(p.N, begin + p.window);
  int run = p.keys[begin];
  if (run >= p.words) return;                           // ids outside the table come last
  bool came_in = false, goes_on = false;                // a long run that another window starts, or ends
  const int2 first = p.runs[run];
  if (first.x < begin) {
    if (first.y - first.x > p.most) came_in = true;
    else begin = first.y;                               // summed where it starts
    if (begin >= end) return;
    run = p.keys[begin];
  }
  const int tail = p.keys[end - 1];
  if (tail < p.words) {
    const int2 last = p.runs[tail];
    if (last.y > end && (last.x >= begin || came_in)) {
      if (last.y - last.x > p.most) goes_on = true;
      else end = last.y;
    }
  }
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  float* part = p.parts + w * 2 * p.D + c;
  auto done = [&]() {                                   // the run has ended inside the window
    if (run >= p.words) return;
    if (came_in) {
      Vec<float, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = acc[j];
      r.store(part);
    } else {
      Vec<TT, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = acc[j];
      put_row<TT, V>(dtable, p, run, c, r);
    }
  };
  for (int e = begin; e < end; e += U) {
    int key[U];
    Raw<T, V> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = e + u < end ? p.keys[e + u] : p.words;
      if (key[u] < p.words) q[u].load(dout + (long long)p.order[e + u] * p.D + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e + u < end) {
        if (key[u] != run) {
          done();
          run = key[u];
          came_in = false;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = 0.f;
        }
        if (run < p.words) {
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += q[u].at(j);
        }
      }
    }
  }
  if (goes_on && !came_in) {
    Vec<float, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = acc[j];
    r.store(part + p.D);
  } else {
    done();                                             // a run through the whole window leaves its part as one that came in
  }
}

// Long runs: their parts are added up, JOIN_GROUPS neighbouring stretches of them side by side and then those.  A long
// run holds a multiple of `most`, and is found by the first that it holds.  A CTA has a slice of a row.
constexpr int JOIN_GROUPS = 8;
template <typename TT, int V>
__global__ void __launch_bounds__(128 * JOIN_GROUPS)
table_join_kernel(TT* __restrict__ dtable, const TableGrad p) {
  after_previous();
  __shared__ float sums[JOIN_GROUPS][128 * V];
  const int slice = blockIdx.x % p.slices, at = blockIdx.x / p.slices * p.most;         // at < N
  const int run = p.keys[at];
  if (run >= p.words) return;
  const int2 range = p.runs[run];
  if (range.y - range.x <= p.most || at - range.x >= p.most) return;
  const int w = range.x / p.window, last = (range.y - 1) / p.window;
  const int group = threadIdx.x >> 7, x = threadIdx.x & 127, c = (slice * 128 + x) * V;
  const int n = last - w, each = (n + JOIN_GROUPS - 1) / JOIN_GROUPS;
  const bool mine = c < p.D;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (mine) {
    const float* src = p.parts + c;
    const long long size = 2ll * p.D;
    Vec<float, V> q[4];
    if (group == 0) {
      q[0].load(src + w * size + p.D);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = q[0].v[j];
    }
    const int k1 = w + 1 + min(n, (group + 1) * each);
    for (int k = w + 1 + group * each; k < k1; k += 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < k1) q[u].load(src + (k + u) * size);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < k1) {
#pragma unroll
          for (int j = 0; j < V; ++j) s[j] += q[u].v[j];
        }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sums[group][j * 128 + x] = s[j];
  __syncthreads();
  if (group || !mine) return;
  Vec<TT, V> r;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    r.v[j] = sums[0][j * 128 + x];
    for (int k = 1; k < JOIN_GROUPS; ++k) r.v[j] += sums[k][j * 128 + x];
  }
  put_row<TT, V>(dtable, p, run, c, r);
}

template <int CTAS>
static int launch_sort(const long long* ids, int N, int words, int* order, int* other, int* keys, int2* runs,
                       cudaStream_t st) {
  auto kern = sort_tokens_kernel<CTAS>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  if (!known || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_SMEM);
    if (e != cudaSuccess) return (int)e;
    if (known) configured[dev] = true;
  }
  int bits = 1;
  while ((words >> bits) > 0) ++bits;                   // keys are 0 .. words
  const int passes = (bits + 8) / 9, per_pass = (bits + passes - 1) / passes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CTAS);
  cfg.blockDim = dim3(SORT_THREADS);
  cfg.dynamicSmemBytes = SORT_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)LaunchAfter<const long long*, int, int, int, int, int*, int*, int*, int2*>{kern, cfg}(
      ids, N, words, per_pass, passes, order, other, keys, runs);
}

}  // namespace pf

using namespace pf;

static bool embed_sizes_ok(long long N, long long words, int D) {
  return N >= 0 && N <= (1ll << 30) && words >= 0 && words < (1ll << 30) && D >= 0;
}

// tokens of a window: some 4000 CTAs' worth, at least 8 and at most 128
static int window_of(long long N, int per_cta_slices) {
  long long w = N * per_cta_slices / 4096;
  return (int)(w < 8 ? 8 : w > 128 ? 128 : w);
}

struct EmbedPlan {
  int V, lanes_log, slices, window;
  long long windows;
};
static EmbedPlan embed_plan(long long N, int D, bool vec) {
  EmbedPlan g;
  g.V = vec ? 8 : 1;
  const int per_row = (D + g.V - 1) / g.V;
  g.lanes_log = 0;
  while (g.lanes_log < 7 && (1 << g.lanes_log) < per_row) ++g.lanes_log;
  g.slices = (per_row + (1 << g.lanes_log) - 1) >> g.lanes_log;
  if (g.slices < 1) g.slices = 1;
  g.window = window_of(N, g.slices);
  g.windows = (N + g.window - 1) / g.window;
  return g;
}

// out [tokens, D] = scale table[ids], packed; zeros for ids outside the table
PF_API int pf_scaled_embed_fwd(const void* table, const void* ids, void* out, long long tokens, int D, long long words,
                               float scale, int table_dtype, int out_dtype, void* stream) {
  if (!embed_sizes_ok(tokens, words, D)) return -3;
  if (tokens == 0 || D == 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = on_rows(table, D, table_dtype) && on_rows(out, D, out_dtype);
  const int per_row = vec ? D / 8 : D;
  int lanes_log = 0;
  while (lanes_log < 5 && (1 << lanes_log) < per_row) ++lanes_log;
  const long long ctas = ((tokens << lanes_log) + 255) / 256;
  if (ctas > 0x7fffffffll) return -3;
  const long long* I = (const long long*)ids;
#define PF_FWD(TD, TT_, OD, OT_)                                                                                       \
  if (table_dtype == TD && out_dtype == OD) {                                                                          \
    if (vec)                                                                                                           \
      after(scaled_embed_kernel<TT_, OT_, 8>, (unsigned)ctas, 256, 0, st)((const TT_*)table, I, (OT_*)out, tokens,     \
                                                                          lanes_log, D, words, scale);                 \
    else                                                                                                               \
      after(scaled_embed_kernel<TT_, OT_, 1>, (unsigned)ctas, 256, 0, st)((const TT_*)table, I, (OT_*)out, tokens,     \
                                                                          lanes_log, D, words, scale);                 \
  } else
  PF_FWD(PF_F32, float, PF_F32, float)
  PF_FWD(PF_F32, float, PF_F16, __half)
  PF_FWD(PF_F32, float, PF_BF16, __nv_bfloat16)
  PF_FWD(PF_F16, __half, PF_F16, __half)
  PF_FWD(PF_BF16, __nv_bfloat16, PF_BF16, __nv_bfloat16)
  return -1;
#undef PF_FWD
  PF_CHECK_LAUNCH();
  return 0;
}

// KiB of scratch of pf_scaled_embed_bwd, for rows that lie on 16 bytes or not
PF_API int pf_scaled_embed_scratch(long long tokens, int D, long long words) {
  if (!embed_sizes_ok(tokens, words, D)) return -3;
  const EmbedPlan a = embed_plan(tokens, D, true), b = embed_plan(tokens, D, false);
  const long long windows = a.windows > b.windows ? a.windows : b.windows;
  const long long bytes = tokens * 12 + (words + 3) / 4 * 32 + windows * 2 * D * 4 + 64;
  const long long kib = (bytes + 1023) / 1024;
  return kib > 0x7fffffffll ? -3 : (int)kib;
}

// dtable [words, D] = (or, in fp32, +=) scale times the sums of dout [tokens, D] by ids, both packed
PF_API int pf_scaled_embed_bwd(const void* dout, const void* ids, void* dtable, void* scratch, long long tokens, int D,
                               long long words, float scale, int accumulate, int dtype, int table_dtype, void* stream) {
  if (!embed_sizes_ok(tokens, words, D)) return -3;
  if (accumulate && table_dtype != PF_F32) return -1;
  if (reinterpret_cast<uintptr_t>(scratch) & 31) return -2;
  if (D == 0 || words == 0 || (accumulate && tokens == 0)) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = on_rows(dout, D, dtype) && on_rows(dtable, D, table_dtype);
  const EmbedPlan g = embed_plan(tokens, D, vec);
  TableGrad p;
  const int N = (int)tokens;
  int2* runs = static_cast<int2*>(scratch);
  p.parts = reinterpret_cast<float*>(runs + (words + 3) / 4 * 4);       // 32 bytes for vectors of 8
  int* keys = reinterpret_cast<int*>(p.parts + g.windows * 2 * D);
  int* order = keys + N;
  int* other = order + N;
  // one CTA where a second or two of its rounds are all there is
  const int r = N <= 4096 ? launch_sort<1>((const long long*)ids, N, (int)words, order, other, keys, runs, st)
                          : launch_sort<8>((const long long*)ids, N, (int)words, order, other, keys, runs, st);
  if (r) return r;
  p.keys = keys; p.order = order; p.runs = runs; p.most = std::max(64, 4 * g.window);
  p.N = N; p.words = (int)words; p.D = D; p.window = g.window; p.lanes_log = g.lanes_log; p.slices = g.slices;
  p.scale = scale; p.accumulate = accumulate;
  const int per_cta = 128 >> g.lanes_log;
  const long long work = (g.windows + per_cta - 1) / per_cta * g.slices;
  if (work > 0x7fffffffll) return -3;
  if (!accumulate) {
    const size_t bytes = (size_t)words * D * (table_dtype == PF_F32 ? 4 : 2);
    // up to the first 16 bytes, and behind the last: a table that is a view may start anywhere
    char* at = static_cast<char*>(dtable);
    const size_t head = std::min(bytes, (16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15);
    if (head) {
      cudaError_t e = cudaMemsetAsync(at, 0, head, st);
      if (e != cudaSuccess) return (int)e;
    }
    const long long n = (long long)((bytes - head) / 16), zeros = std::max(1ll, (n + 4095) / 4096);
    if (zeros > 0x7fffffffll) return -3;
    after(table_zeros_kernel, (unsigned)zeros, 512, 0, st)(reinterpret_cast<uint4*>(at + head), n,
        reinterpret_cast<unsigned char*>(at + head + n * 16), (int)((bytes - head) & 15));
    PF_CHECK_LAUNCH();
  }
  if (N == 0) return 0;
  const unsigned grid = (unsigned)work;
  const int join_slices = (D + 128 * g.V - 1) / (128 * g.V);
  const long long joins = N > p.most ? (long long)((N + p.most - 1) / p.most) * join_slices : 0;
  if (joins > 0x7fffffffll) return -3;
  TableGrad pj = p;
  pj.slices = join_slices;
#define PF_BWD(ID, T_, TD, TT_)                                                                                        \
  if (dtype == ID && table_dtype == TD) {                                                                              \
    if (vec) {                                                                                                         \
      after(table_grad_kernel<T_, TT_, 8>, grid, 128, 0, st)((const T_*)dout, (TT_*)dtable, p);                        \
      if (joins > 0)                                                                                                   \
        after(table_join_kernel<TT_, 8>, (unsigned)joins, 128 * JOIN_GROUPS, 0, st)((TT_*)dtable, pj);                 \
    } else {                                                                                                           \
      after(table_grad_kernel<T_, TT_, 1>, grid, 128, 0, st)((const T_*)dout, (TT_*)dtable, p);                        \
      if (joins > 0)                                                                                                   \
        after(table_join_kernel<TT_, 1>, (unsigned)joins, 128 * JOIN_GROUPS, 0, st)((TT_*)dtable, pj);                 \
    }                                                                                                                  \
  } else
  PF_BWD(PF_F32, float, PF_F32, float)
  PF_BWD(PF_F16, __half, PF_F32, float)
  PF_BWD(PF_BF16, __nv_bfloat16, PF_F32, float)
  PF_BWD(PF_F16, __half, PF_F16, __half)
  PF_BWD(PF_BF16, __nv_bfloat16, PF_BF16, __nv_bfloat16)
  return -1;
#undef PF_BWD
  PF_CHECK_LAUNCH();
  return 0;
}
