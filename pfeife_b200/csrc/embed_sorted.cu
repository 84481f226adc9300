// Embedded tokens with a scale, and the gradient of the table by sorted tokens.
//
// out[t] = scale table[id_t];  dtable[v] = scale sum over t with id_t = v of dout[t].
//
// Both are bound by memory: forward the rows that are named and the output, backward dout and the whole gradient
// table, most of whose rows are zeros.  Sums go over the tokens in their order (the sort is stable) in 32 bits, in
// windows of the sorted tokens: a run of one id inside a window is written at once, one that crosses windows
// leaves a part in each, which are added in their order.  So the same tokens give the same bits, a row is written
// once and rounded once, and a padding token that a third of the batch shares is summed by as many CTAs as it has
// windows.  Ids outside the table have zeros and no gradient.
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
// whether rows of D values start on the 8-value accesses of their type
static bool on_rows(const void* p, int D, int dtype) {
  return D % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & (dtype == PF_F32 ? 31 : 15)) == 0;
}

// Four vectors of V values a thread, requested before any is written.
template <typename TT, typename T, int V>
__global__ void __launch_bounds__(256)
scaled_embed_kernel(const TT* __restrict__ table, const long long* __restrict__ ids, T* __restrict__ out,
                    long long total, int per_row, int D, long long words, float scale) {
  after_previous();
  constexpr int U = 4;
  const long long i0 = blockIdx.x * (256ll * U) + threadIdx.x;
  Vec<TT, V> q[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = i0 + u * 256;
    if (i < total) {
      const long long t = total <= 0x7fffffffll ? (unsigned)i / (unsigned)per_row : i / per_row;
      const long long id = ids[t];
      const int c = (int)(i - t * per_row) * V;
      if (id >= 0 && id < words) {
        q[u].load(table + id * D + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) q[u].v[j] = 0.f;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = i0 + u * 256;
    if (i < total) {
      Vec<T, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = q[u].v[j] * scale;
      r.store(out + i * V);                             // rows of D = per_row V values, packed
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
                   int* __restrict__ other, int* __restrict__ keys, unsigned* __restrict__ present) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;                              // [warp][bin]
  int* totals = counts + SORT_WARPS * SORT_BINS;        // [bin], read by the other CTAs
  int* starts = totals + SORT_BINS;
  int* sums = starts + SORT_BINS;
  after_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS > 1 ? (int)cluster_ctarank() : 0;
  const int bins = 1 << bits;
  // stretches of whole rounds of 32 tokens a warp
  const int per_warp = ((N + CTAS * SORT_WARPS - 1) / (CTAS * SORT_WARPS) + 31) / 32 * 32;
  const long long lo = (long long)(rank * SORT_WARPS + warp) * per_warp;
  const int begin = (int)(lo < N ? lo : N), end = (int)(lo + per_warp < N ? lo + per_warp : N);
  for (int i = rank * SORT_THREADS + threadIdx.x; i < (words + 31) / 32; i += CTAS * SORT_THREADS) present[i] = 0;
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
          if (pass == passes - 1) {
            keys[to] = key[u];
            if (key[u] < words) atomicOr(present + (key[u] >> 5), 1u << (key[u] & 31));
          }
        }
        __syncwarp();
        if (in && lane == __ffs(same) - 1) mine[digit] += __popc(same);
        __syncwarp();
      }
    }
    all_sync();
  }
}

// Sums of windows of the sorted tokens.  `lanes` threads (a power of two) share a row of V-wide vectors, 128 / lanes
// windows a CTA; CTAs behind those of the windows write zeros to rows that no token names.
struct TableGrad {
  const int* keys;
  const int* order;
  const unsigned* present;
  int N, words, D, window, lanes_log, slices;
  unsigned work_ctas;
  int zero_rows;                // rows of a CTA that writes zeros
  float scale;
  int accumulate;
  float* parts;                 // [window][2][D]: of the run that came in, of the run that goes on
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
  constexpr int U = V == 1 ? 8 : 4;
  if (blockIdx.x >= p.work_ctas) {
    const long long r0 = (blockIdx.x - p.work_ctas) * (long long)p.zero_rows;
    const long long r1 = r0 + p.zero_rows < p.words ? r0 + p.zero_rows : p.words;
    Vec<TT, V> zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = 0.f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long r = r0 + warp; r < r1; r += 4) {
      if (p.present[r >> 5] >> (r & 31) & 1) continue;
      TT* dst = dtable + r * p.D;
      for (int c = lane * V; c < p.D; c += 32 * V) zero.store(dst + c);
    }
    return;
  }
  const int lanes = 1 << p.lanes_log;
  const int slice = blockIdx.x % p.slices;
  const long long w = (long long)(blockIdx.x / p.slices) * (128 >> p.lanes_log) + (threadIdx.x >> p.lanes_log);
  const long long b = w * p.window;
  const int c = (slice * lanes + (threadIdx.x & (lanes - 1))) * V;
  if (b >= p.N || c >= p.D) return;
  const int begin = (int)b, end = min(p.N, begin + p.window);
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int run = p.keys[begin];
  bool came_in = begin > 0 && p.keys[begin - 1] == run;
  float* part = p.parts + w * 2 * p.D + c;
  auto done = [&]() {                                   // the run has ended inside the window
    if (run >= p.words) return;
    if (came_in) {
#pragma unroll
      for (int j = 0; j < V; ++j) part[j] = acc[j];
    } else {
      Vec<TT, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = acc[j];
      put_row<TT, V>(dtable, p, run, c, r);
    }
  };
  for (int e = begin; e < end; e += U) {
    int key[U];
    Vec<T, V> q[U];
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
          for (int j = 0; j < V; ++j) acc[j] += q[u].v[j];
        }
      }
    }
  }
  const bool goes_on = end < p.N && p.keys[end] == run;
  if (goes_on && !came_in) {
    if (run < p.words) {
#pragma unroll
      for (int j = 0; j < V; ++j) part[p.D + j] = acc[j];
    }
  } else {
    done();                                             // a run through the whole window leaves its part as one that came in
  }
}

// Runs that cross windows: the window in which one starts adds up its parts, JOIN_GROUPS neighbouring stretches of them
// side by side and then those.  A CTA has one window's slice of a row.
constexpr int JOIN_GROUPS = 8;
template <typename TT, int V>
__global__ void __launch_bounds__(128 * JOIN_GROUPS)
table_join_kernel(TT* __restrict__ dtable, const TableGrad p) {
  after_previous();
  __shared__ float sums[JOIN_GROUPS][128 * V];
  const int slice = blockIdx.x % p.slices, w = blockIdx.x / p.slices;
  const int b = w * p.window, e = b + p.window;         // in range: only windows before the last are dealt
  const int run = p.keys[e - 1];
  if (run >= p.words || p.keys[e] != run) return;
  if (b > 0 && p.keys[b] == run && p.keys[b - 1] == run) return;         // it started further ahead
  // the first token behind the run, by 32 looks at a time
  const int lane = threadIdx.x & 31;
  int lo = e, hi = p.N;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at < hi && p.keys[at] == run));
    if (n == 0) break;
    hi = min(hi, lo + n * step);
    lo = lo + (n - 1) * step + 1;
  }
  const int last = (lo - 1) / p.window;
  const int group = threadIdx.x >> 7, x = threadIdx.x & 127, c = (slice * 128 + x) * V;
  const int n = last - w, each = (n + JOIN_GROUPS - 1) / JOIN_GROUPS;
  const bool mine = c < p.D;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (mine) {
    const float* src = p.parts + c;
    const long long size = 2ll * p.D;
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = src[w * size + p.D + j];
    }
    const int k1 = w + 1 + min(n, (group + 1) * each);
    for (int k = w + 1 + group * each; k < k1; k += 4) {
      float q[4][V];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < k1) {
#pragma unroll
          for (int j = 0; j < V; ++j) q[u][j] = src[(k + u) * size + j];
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < k1) {
#pragma unroll
          for (int j = 0; j < V; ++j) s[j] += q[u][j];
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
static int launch_sort(const long long* ids, int N, int words, int* order, int* other, int* keys, unsigned* present,
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
  return (int)LaunchAfter<const long long*, int, int, int, int, int*, int*, int*, unsigned*>{kern, cfg}(
      ids, N, words, per_pass, passes, order, other, keys, present);
}

}  // namespace pf

using namespace pf;

static bool embed_sizes_ok(long long N, long long words, int D) {
  return N >= 0 && N <= (1ll << 30) && words >= 0 && words < (1ll << 30) && D >= 0;
}

// tokens of a window: some 2000 CTAs' worth, at least 8 and at most 256
static int window_of(long long N, int per_cta_slices) {
  long long w = N * per_cta_slices / 2048;
  return (int)(w < 8 ? 8 : w > 256 ? 256 : w);
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
  const long long total = tokens * per_row, ctas = (total + 1023) / 1024;
  if (ctas > 0x7fffffffll) return -3;
  const long long* I = (const long long*)ids;
#define PF_FWD(TD, TT_, OD, OT_)                                                                                       \
  if (table_dtype == TD && out_dtype == OD) {                                                                          \
    if (vec)                                                                                                           \
      after(scaled_embed_kernel<TT_, OT_, 8>, (unsigned)ctas, 256, 0, st)((const TT_*)table, I, (OT_*)out, total,      \
                                                                          per_row, D, words, scale);                   \
    else                                                                                                               \
      after(scaled_embed_kernel<TT_, OT_, 1>, (unsigned)ctas, 256, 0, st)((const TT_*)table, I, (OT_*)out, total,      \
                                                                          per_row, D, words, scale);                   \
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
  const long long bytes = tokens * 12 + (words + 31) / 32 * 4 + windows * 2 * D * 4 + 64;
  const long long kib = (bytes + 1023) / 1024;
  return kib > 0x7fffffffll ? -3 : (int)kib;
}

// dtable [words, D] = (or, in fp32, +=) scale times the sums of dout [tokens, D] by ids, both packed
PF_API int pf_scaled_embed_bwd(const void* dout, const void* ids, void* dtable, void* scratch, long long tokens, int D,
                               long long words, float scale, int accumulate, int dtype, int table_dtype, void* stream) {
  if (!embed_sizes_ok(tokens, words, D)) return -3;
  if (accumulate && table_dtype != PF_F32) return -1;
  if (!on_vectors(scratch)) return -2;
  if (D == 0 || words == 0 || (accumulate && tokens == 0)) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = on_rows(dout, D, dtype) && on_rows(dtable, D, table_dtype);
  const EmbedPlan g = embed_plan(tokens, D, vec);
  TableGrad p;
  const int N = (int)tokens;
  p.parts = static_cast<float*>(scratch);
  int* keys = reinterpret_cast<int*>(p.parts + g.windows * 2 * D);
  int* order = keys + N;
  int* other = order + N;
  unsigned* present = reinterpret_cast<unsigned*>(other + N);
  // one CTA where a second or two of its rounds are all there is
  const int r = N <= 4096 ? launch_sort<1>((const long long*)ids, N, (int)words, order, other, keys, present, st)
                          : launch_sort<8>((const long long*)ids, N, (int)words, order, other, keys, present, st);
  if (r) return r;
  p.keys = keys; p.order = order; p.present = present;
  p.N = N; p.words = (int)words; p.D = D; p.window = g.window; p.lanes_log = g.lanes_log; p.slices = g.slices;
  p.scale = scale; p.accumulate = accumulate;
  const int per_cta = 128 >> g.lanes_log;
  const long long work = (g.windows + per_cta - 1) / per_cta * g.slices;
  p.zero_rows = (int)(words / 2048 < 4 ? 4 : words / 2048);
  const long long zeros = accumulate ? 0 : (words + p.zero_rows - 1) / p.zero_rows;
  if (work + zeros > 0x7fffffffll) return -3;
  p.work_ctas = (unsigned)work;
  const unsigned grid = (unsigned)(work + zeros);
  const int join_slices = (D + 128 * g.V - 1) / (128 * g.V);
  const long long joins = (g.windows - 1) * join_slices;         // a run that crosses starts before the last window
  if (joins > 0x7fffffffll) return -3;
  TableGrad pj = p;
  pj.slices = join_slices;
#define PF_BWD(ID, T_, TD, TT_)                                                                                        \
  if (dtype == ID && table_dtype == TD) {                                                                              \
    if (vec) {                                                                                                         \
      after(table_grad_kernel<T_, TT_, 8>, grid, 128, 0, st)((const T_*)dout, (TT_*)dtable, p);                        \
      if (joins > 0) after(table_join_kernel<TT_, 8>, (unsigned)joins, 128 * JOIN_GROUPS, 0, st)((TT_*)dtable, pj);                \
    } else {                                                                                                           \
      after(table_grad_kernel<T_, TT_, 1>, grid, 128, 0, st)((const T_*)dout, (TT_*)dtable, p);                        \
      if (joins > 0) after(table_join_kernel<TT_, 1>, (unsigned)joins, 128 * JOIN_GROUPS, 0, st)((TT_*)dtable, pj);                \
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
