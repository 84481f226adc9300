// Products on tcgen05 whose epilogue is the operator: the gated feed-forward block in both directions, and the
// output head with its cross entropy, whose logits stay in TMEM.
//
// The main loop is that of gemm_sm100.cu: persistent CTAs, warp 0 the TMA producer, warp 1 the issuer of the
// products, warps 2..9 the epilogue (a row per thread, half the tile's columns per warp), accumulators twice in
// TMEM so that an epilogue runs under the next tile's products.  Tiles are 256 x 256 of a CTA pair
// (cta_group::2) or 128 x 128 of one CTA.
//
// GLU_FWD: a tile has as many gate columns as up columns.  B comes from two tensor maps, the gate and the up rows of
// one weight; of a pair, the even CTA loads the gate rows and the odd one the up rows, so that the accumulator
// of every row has the gate in its left half and up in its right half, and one thread has both values.
// HEAD_STATS: a thread keeps the maximum and the sum of exponentials of its columns; references are integers in
// powers of two, so that joining two parts multiplies by an exact power of two.
// HEAD_DZ computes the logits again, once the sums are known: no logit is ever written.
#include <cstring>
#include "common.cuh"
#include "api.h"
#include "fused_gemm.h"

namespace pf {

int make_tmap_2d_16bit(CUtensorMap* map, const void* base, int fmt, long long inner, long long outer, long long ld,
                       int box_inner, int box_outer);
int make_tmap_out(CUtensorMap* map, const void* base, int out_dtype, long long cols, long long rows, long long ld);

constexpr int FG_BM = 128, FG_BN = 128, FG_BK = 64;      // per CTA and k-block
constexpr int FG_EPI_WARPS = 8;
constexpr int FG_THREADS = 64 + 32 * FG_EPI_WARPS;
constexpr int FG_STAGE_BYTES = (FG_BM + FG_BN) * FG_BK * 2;
constexpr int FG_GROUP_ROWS = 4096;                      // see GROUP_ROWS in gemm_sm100.cu
constexpr int FG_BOX16 = 2048, FG_BOX32 = 4096;          // staged [32 x 32] boxes

// Shared memory of a job: stages of operands, barriers, and what each epilogue warp stages its stores in.
template <int JOB, typename OutT>
struct FusedSmem {
  static constexpr int BOX = sizeof(OutT) == 4 ? FG_BOX32 : FG_BOX16;
  static constexpr int BOXES = JOB == GLU_FWD || JOB == GLU_BWD ? 3 : JOB == HEAD_STATS ? 0 : 1;
  static constexpr int SETS = BOXES == 1 ? 2 : 1;
  static constexpr int PER_WARP = SETS * BOXES * BOX;
  static constexpr int STAGES = BOXES ? 5 : 6;
  static constexpr int BAR_OFFSET = STAGES * FG_STAGE_BYTES;
  static constexpr int STAGING_OFFSET = BAR_OFFSET + 1024;
  static constexpr int TOTAL = STAGING_OFFSET + FG_EPI_WARPS * PER_WARP + 1024;
  static_assert(TOTAL <= 232448, "more than a CTA may have");
};

struct FusedMaps { CUtensorMap a, b, b2, c0, c1, c2; };

struct FusedParams {
  int M, N, K, fmt, group_m;
  const int* rows;
  int* status;
  const void* gu;
  const void* bias;
  int bias_dtype, act, save;
  const int* labels;
  RowStat* parts;
  long long part_pitch;
  float* picked;
  const RowStat* stats;
  const float* factor;
  float unit;
  int first, split, part_rows, accumulate;
  const float *scale, *scale2;
  float scale3;
};

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Activations of a pair and, with SLOPE, their derivatives.  SiLU is z s(z) with s(z) = 1 / (1 + e^-z), and the tanh
// form of GELU is z s(2 u) with u = sqrt(2 / pi) (z + 0.044715 z^3); with q their argument both have the derivative
// s + z s (1 - s) q'.  e^-q overflows to infinity for large negative q, where s is 0.  q' is held to |z| <= 1e3, beyond
// which s (1 - s) is 0 and z^2 may not be finite.
template <bool SLOPE>
__device__ __forceinline__ void sigmoid_act(float z, float q, float dq, float& a, float& d) {
  const float s = rcp_approx(1.f + ex2(-LOG2E * q));
  a = z * s;
  if (SLOPE) d = fmaf(a * (1.f - s), dq, s);
}
template <bool SLOPE>
__device__ __forceinline__ void act2(int act, float z0, float z1, float& a0, float& a1, float& d0, float& d1) {
  if (act == 1) {                                       // GELU with erf
    uint64_t e;
    const uint64_t ny = gelu_neg_tail2(f2_pack(fabsf(z0), fabsf(z1)), e);
    float y0, y1, e0, e1;
    f2_unpack(ny, y0, y1);
    a0 = fmaf(fabsf(z0), y0, fmaxf(z0, 0.f));
    a1 = fmaf(fabsf(z1), y1, fmaxf(z1, 0.f));
    if (SLOPE) {
      f2_unpack(e, e0, e1);
      d0 = fmaf(z0 * 0.3989422804014327f, e0, z0 >= 0.f ? 1.f + y0 : -y0);
      d1 = fmaf(z1 * 0.3989422804014327f, e1, z1 >= 0.f ? 1.f + y1 : -y1);
    }
  } else if (act == 2) {                                // GELU with tanh
    constexpr float c = 2.f * 0.7978845608028654f;
    auto one = [](float z, float& a, float& d) {
      const float z2 = z * z, zc = fminf(z2, 1e6f);
      sigmoid_act<SLOPE>(z, c * fmaf(0.044715f * z2, z, z), c * fmaf(3.f * 0.044715f, zc, 1.f), a, d);
    };
    one(z0, a0, d0);
    one(z1, a1, d1);
  } else {                                              // SiLU
    sigmoid_act<SLOPE>(z0, z0, 1.f, a0, d0);
    sigmoid_act<SLOPE>(z1, z1, 1.f, a1, d1);
  }
}

__device__ __forceinline__ float bias_at(const void* b, int dtype, int i) {
  if (dtype == PF_F32) return __ldg(reinterpret_cast<const float*>(b) + i);
  if (dtype == PF_F16) return __half2float(__ldg(reinterpret_cast<const __half*>(b) + i));
  return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(b) + i));
}

// Row r (32 values) of a [32 x 32] box as a TMA store reads it: 64-byte rows swizzled over 64 bytes (16-bit values),
// 128-byte rows over 128 (fp32).  No two lanes of a warp meet in a bank.
template <typename OutT>
__device__ __forceinline__ void fill_box(uint8_t* box, int r, const float (&v)[32]) {
  constexpr int PER = 16 / sizeof(OutT), NCH = 32 / PER;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    uint4 q;
    OutT* e = reinterpret_cast<OutT*>(&q);
#pragma unroll
    for (int j = 0; j < PER; ++j) e[j] = from_f32<OutT>(v[c * PER + j]);
    const int at = NCH == 4 ? (c ^ ((r >> 1) & 3)) : (c ^ (r & 7));
    *reinterpret_cast<uint4*>(box + r * (NCH * 16) + at * 16) = q;
  }
}

template <typename T, typename OutT, int JOB, bool PAIR>
__global__ void __launch_bounds__(FG_THREADS, 1)
fused_gemm_kernel(const __grid_constant__ FusedMaps maps, const FusedParams p) {
  using S = FusedSmem<JOB, OutT>;
  constexpr bool A_MN = JOB == HEAD_DW;
  constexpr bool B_MN = JOB == GLU_BWD || JOB == HEAD_DX || JOB == HEAD_DW;
  constexpr int BMT = PAIR ? 2 * FG_BM : FG_BM;
  constexpr int BNT = PAIR ? 2 * FG_BN : FG_BN;           // accumulator columns of a tile
  constexpr int NT = JOB == GLU_FWD ? BNT / 2 : BNT;      // output columns of a tile
  constexpr int STAGES = S::STAGES;
  constexpr uint32_t TMEM_COLS = 2 * BNT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::BAR_OFFSET);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = PAIR ? cluster_ctarank() : 0u;
  const int first_tile = PAIR ? (blockIdx.x >> 1) : blockIdx.x;
  const int n_workers = PAIR ? (gridDim.x >> 1) : gridDim.x;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], (PAIR ? 2 : 1) * FG_EPI_WARPS);      // lane 0 of every epilogue warp
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_of(tmem_slot);
  after_previous();

  // The rows that count are known on the device only.  At most p.M (p.K): what lies behind them is not read.
  const int count = p.rows ? min(*p.rows, JOB == HEAD_DW ? p.K : p.M) : 0;
  const int M = p.rows && JOB != HEAD_DW ? count : p.M;
  const int K = p.rows && JOB == HEAD_DW ? count : p.K;
  const int num_m = (M + BMT - 1) / BMT, num_n = (p.N + NT - 1) / NT, num_mn = num_m * num_n;
  const int split = JOB == HEAD_DX ? p.split : 1;
  const int num_items = num_mn * split;
  const int num_kb = (K + FG_BK - 1) / FG_BK;
  // Items are dealt in rounds, every other one in reverse; tiles in bands of group_m rows of tiles, column by column.
  auto item_of = [&](int round) { return round * n_workers + ((round & 1) ? n_workers - 1 - first_tile : first_tile); };
  auto place = [&](int item, int& mt, int& nt, int& kb0, int& kb1) {
    const int ks = split > 1 ? item / num_mn : 0, tile = item - ks * num_mn;
    kb0 = split > 1 ? (int)((long long)num_kb * ks / split) : 0;
    kb1 = split > 1 ? (int)((long long)num_kb * (ks + 1) / split) : num_kb;
    const int per_band = p.group_m * num_n, band = tile / per_band, in_band = tile - band * per_band;
    const int rows = min(p.group_m, num_m - band * p.group_m);
    nt = in_band / rows;
    mt = band * p.group_m + in_band - nt * rows;
    return ks;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full_leader = PAIR ? mapa_u32(full_bar, 0) : 0u;    // both CTAs' bytes count there
      for (int round = 0, item = item_of(0); item < num_items && ok; item = item_of(++round)) {
        int mt, nt, kb0, kb1;
        place(item, mt, nt, kb0, kb1);
        const int m0 = mt * BMT + int(cta_rank) * FG_BM;
        const int n0 = nt * NT + (JOB == GLU_FWD ? 0 : int(cta_rank) * FG_BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, p.status, PF_ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          uint8_t* sa = smem + stage * FG_STAGE_BYTES;
          uint8_t* sb = sa + FG_BM * FG_BK * 2;
          const int k0 = kb * FG_BK;
          if (!PAIR || cta_rank == 0) mbar_expect_tx(&full_bar[stage], (PAIR ? 2 : 1) * FG_STAGE_BYTES);
          auto load = [&](uint8_t* to, const CUtensorMap* map, int x, int y) {
            if (PAIR) tma_load_2d_pair(to, map, full_leader + stage * 8, x, y);
            else tma_load_2d(to, map, &full_bar[stage], x, y);
          };
          if (A_MN) {
            load(sa, &maps.a, m0, k0);
            load(sa + 8192, &maps.a, m0 + 64, k0);
          } else {
            load(sa, &maps.a, k0, m0);
          }
          if (JOB == GLU_FWD) {
            if (PAIR) {
              load(sb, cta_rank ? &maps.b2 : &maps.b, k0, n0);           // 128 rows of one half
            } else {
              load(sb, &maps.b, k0, n0);                                 // 64 rows of each
              load(sb + 8192, &maps.b2, k0, n0);
            }
          } else if (B_MN) {
            load(sb, &maps.b, n0, k0);
            load(sb + 8192, &maps.b, n0 + 64, k0);
          } else {
            load(sb, &maps.b, k0, n0);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (cta_rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16(BMT, BNT, p.fmt, A_MN, B_MN);
      constexpr uint32_t a_adv = (A_MN ? 2048u : 32u) >> 4, b_adv = (B_MN ? 2048u : 32u) >> 4;
      constexpr uint32_t a_lbo = A_MN ? 8192u : 16u, b_lbo = B_MN ? 8192u : 16u;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int round = 0, item = item_of(0); item < num_items && ok; item = item_of(++round)) {
        int mt, nt, kb0, kb1;
        place(item, mt, nt, kb0, kb1);
        if (kb0 == kb1) continue;                      // nothing to add up: the epilogue writes zeros
        ok = PAIR ? mbar_wait_cluster(&tmem_empty[acc], acc_phase ^ 1, p.status, PF_ERR_TIMEOUT_TMEM_EMPTY)
                  : mbar_wait(&tmem_empty[acc], acc_phase ^ 1, p.status, PF_ERR_TIMEOUT_TMEM_EMPTY);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BNT;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, p.status, PF_ERR_TIMEOUT_FULL);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * FG_STAGE_BYTES);
          const uint32_t a_lo = desc_lo(sa, a_lbo), b_lo = desc_lo(sa + FG_BM * FG_BK * 2, b_lbo);
#pragma unroll
          for (int k = 0; k < FG_BK / 16; ++k) {
            const uint32_t on = (kb != kb0) || (k != 0);
            if (PAIR) tc_mma_f16_pair(d_tmem, a_lo + k * a_adv, b_lo + k * b_adv, idesc, on);
            else tc_mma_f16(d_tmem, a_lo + k * a_adv, b_lo + k * b_adv, idesc, on);
          }
          if (PAIR) tc_commit_pair(&empty_bar[stage], 3);
          else tc_commit(&empty_bar[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (PAIR) tc_commit_pair(&tmem_full[acc], 3);
        else tc_commit(&tmem_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quad = warp & 3, side = (warp - 2) >> 2;
    constexpr int HC = NT / 2;                          // output columns of a warp
    const int c_begin = side * HC, c_end = c_begin + HC;
    uint8_t* boxes = smem + S::STAGING_OFFSET + (warp - 2) * S::PER_WARP;
    int set = 0, staged = 0, acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    // the boxes about to be filled: stores that last read them are done with them
    auto free_boxes = [&]() {
      if (staged >= S::SETS) {
        if (lane == 0) {
          if (S::SETS == 2) tma_store_wait_read_but_one();
          else tma_store_wait_read();
        }
        __syncwarp();
      }
      return boxes + set * (S::BOXES * S::BOX);
    };
    auto boxes_sent = [&]() {
      if (lane == 0) tma_store_commit();
      if (staged < S::SETS) ++staged;
      if (S::SETS == 2) set ^= 1;
    };
    float alpha = 1.f;
    if (JOB == HEAD_DW) alpha = (p.scale ? *p.scale : 1.f) * (p.scale2 ? *p.scale2 : 1.f) * p.scale3;

    for (int round = 0, item = item_of(0); item < num_items && ok; item = item_of(++round)) {
      int mt, nt, kb0, kb1;
      const int ks = place(item, mt, nt, kb0, kb1);
      const int row0 = mt * BMT + int(cta_rank) * FG_BM + quad * 32, row = row0 + lane;
      const int n0 = nt * NT;
      const bool row_ok = row < M;

      // what the epilogue reads travels while the products are computed
      [[maybe_unused]] uint4 kept[8];
      auto fetch = [&](int col) {
        if constexpr (JOB == GLU_BWD) {
          const T* g = reinterpret_cast<const T*>(p.gu) + (long long)row * 2 * p.N + col;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = row_ok && col + 8 * i < p.N;              // N is a multiple of 8
            kept[i] = there ? __ldg(reinterpret_cast<const uint4*>(g) + i) : make_uint4(0, 0, 0, 0);
            kept[4 + i] = there ? __ldg(reinterpret_cast<const uint4*>(g + p.N) + i) : make_uint4(0, 0, 0, 0);
          }
        }
      };
      fetch(n0 + c_begin);
      [[maybe_unused]] int label = -1;                  // as a column of this product
      [[maybe_unused]] float ref = 0.f, inv = 0.f, factor = 0.f, total = 0.f;
      if constexpr (JOB == HEAD_STATS || JOB == HEAD_DZ) {
        if (row_ok) label = p.labels[row] - p.first;
        if (JOB == HEAD_STATS) ref = -INFINITY;
        if (JOB == HEAD_DZ && row_ok) {
          const RowStat st = p.stats[row];
          ref = st.ref;
          inv = st.inv;
          factor = p.factor ? p.factor[row] * p.unit : p.unit;
        }
      }

      const bool empty = kb0 == kb1;
      if (!empty) {
        ok = mbar_wait(&tmem_full[acc], acc_phase, p.status, PF_ERR_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t t_row = tmem_base + (uint32_t(quad * 32) << 16) + acc * BNT;
#pragma unroll 1
      for (int c = c_begin; c < c_end; c += 32) {
        const int col = n0 + c;
        if (col >= p.N) break;                          // uniform across the warp
        uint32_t raw[32];
        float v[32];
        if (!empty) {
          tmem_ld32(t_row + c, raw);
          if constexpr (JOB == GLU_FWD) {
            uint32_t raw_up[32];
            float u[32], h[32];
            tmem_ld32(t_row + NT + c, raw_up);
            tmem_ld_wait_for(raw);
            tmem_ld_wait_for(raw_up);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              v[i] = __uint_as_float(raw[i]);
              u[i] = __uint_as_float(raw_up[i]);
            }
            if (p.bias) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i < p.N) {
                  v[i] += bias_at(p.bias, p.bias_dtype, col + i);
                  u[i] += bias_at(p.bias, p.bias_dtype, p.N + col + i);
                }
            }
            uint8_t* box = free_boxes();
            if (p.save) {
              fill_box<OutT>(box + FG_BOX16, lane, v);
              fill_box<OutT>(box + 2 * FG_BOX16, lane, u);
            }
            float none;
            auto all = [&](auto kind) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                act2<false>(kind, v[i], v[i + 1], h[i], h[i + 1], none, none);
                h[i] *= u[i];
                h[i + 1] *= u[i + 1];
              }
            };
            if (p.act == 1) all(std::integral_constant<int, 1>());
            else if (p.act == 2) all(std::integral_constant<int, 2>());
            else all(std::integral_constant<int, 3>());
            fill_box<OutT>(box, lane, h);
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < M) {                // rows and columns that do not exist are clipped
              tma_store_2d(&maps.c0, box, col, row0);
              if (p.save) {
                tma_store_2d(&maps.c1, box + FG_BOX16, col, row0);
                tma_store_2d(&maps.c2, box + 2 * FG_BOX16, col, row0);
              }
            }
            boxes_sent();
            continue;
          } else {
            tmem_ld_wait_for(raw);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }

        if constexpr (JOB == GLU_BWD) {
          float g[32], u[32];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const T* eg = reinterpret_cast<const T*>(&kept[i]);
            const T* eu = reinterpret_cast<const T*>(&kept[4 + i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              g[i * 8 + j] = to_f32<T>(eg[j]);
              u[i * 8 + j] = to_f32<T>(eu[j]);
            }
          }
          if (c + 32 < c_end) fetch(col + 32);
          // v: dh -> d(up) = dh act(gate); u: up -> h = act(gate) up; g: gate -> d(gate) = dh up act'(gate)
          auto all = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float a0, a1, d0, d1;
              act2<true>(kind, g[i], g[i + 1], a0, a1, d0, d1);
              g[i] = v[i] * u[i] * d0;
              g[i + 1] = v[i + 1] * u[i + 1] * d1;
              v[i] *= a0;
              v[i + 1] *= a1;
              u[i] *= a0;
              u[i + 1] *= a1;
            }
          };
          if (p.act == 1) all(std::integral_constant<int, 1>());
          else if (p.act == 2) all(std::integral_constant<int, 2>());
          else all(std::integral_constant<int, 3>());
          uint8_t* box = free_boxes();
          fill_box<OutT>(box, lane, u);
          fill_box<OutT>(box + FG_BOX16, lane, g);
          fill_box<OutT>(box + 2 * FG_BOX16, lane, v);
          fence_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < M) {
            tma_store_2d(&maps.c0, box, col, row0);
            tma_store_2d(&maps.c1, box + FG_BOX16, col, row0);
            tma_store_2d(&maps.c2, box + 2 * FG_BOX16, col, row0);
          }
          boxes_sent();
        } else if constexpr (JOB == HEAD_STATS) {
          const int nvalid = p.N - col;
          if (nvalid < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= nvalid) v[i] = -INFINITY;
          }
          if ((unsigned)(label - col) < 32u) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == label - col) z = v[i];
            p.picked[row] = z;
          }
          // a NaN does not move the maximum but reaches the sum; a part that is -inf so far subtracts 0
          float top = v[0];
#pragma unroll
          for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
          const float now = fmaxf(ref, ceilf(top * LOG2E)), sub = now == -INFINITY ? 0.f : now;
          total *= ex2(ref - sub);
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            s0 += ex2(fmaf(v[i], LOG2E, -sub));
            s1 += ex2(fmaf(v[i + 1], LOG2E, -sub));
          }
          total += s0 + s1;
          ref = now;
        } else if constexpr (JOB == HEAD_DZ) {
          // rows behind the last have neither a sum nor a factor: their gradients are zeros, which the reduction
          // over rows may read
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float pr = ex2(fmaf(v[i], LOG2E, -ref)) * inv;
            v[i] = (pr - (i == label - col ? 1.f : 0.f)) * factor;
          }
          if (!row_ok) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          uint8_t* box = free_boxes();
          fill_box<OutT>(box, lane, v);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&maps.c0, box, col, row0);
          boxes_sent();
        } else {
          if (JOB == HEAD_DW) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = empty ? 0.f : v[i] * alpha;
          }
          uint8_t* box = free_boxes();
          fill_box<OutT>(box, lane, v);
          fence_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < M) {
            if (sizeof(OutT) == 4 && p.accumulate) tma_reduce_add_2d(&maps.c0, box, col, row0);
            else tma_store_2d(&maps.c0, box, col, row0 + ks * p.part_rows);
          }
          boxes_sent();
        }
      }
      if constexpr (JOB == HEAD_STATS) {
        const int part = (n0 + c_begin) / HC;
        if (row_ok && n0 + c_begin < p.N) p.parts[part * p.part_pitch + row] = {ref, total};
      }
      if (!empty) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(mapa_u32(&tmem_empty[acc], 0));
          else mbar_arrive(&tmem_empty[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
    if (lane == 0 && S::BOXES) tma_store_wait_all();
  }

  // every role reaches this point: all waits are bounded
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------- host side
template <typename T, typename OutT, int JOB, bool PAIR>
static int launch_fused(const FusedMaps& maps, const FusedParams& p, int sm_count, cudaStream_t stream) {
  using S = FusedSmem<JOB, OutT>;
  auto kern = fused_gemm_kernel<T, OutT, JOB, PAIR>;
  static bool configured[64] = {};
  static int resident_pairs[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  if (!known || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return (int)e;
    if (known) configured[dev] = true;
  }
  constexpr int BMT = PAIR ? 2 * FG_BM : FG_BM, BNT = PAIR ? 2 * FG_BN : FG_BN, NT = JOB == GLU_FWD ? BNT / 2 : BNT;
  const long long items = (long long)((p.M + BMT - 1) / BMT) * ((p.N + NT - 1) / NT) * p.split;
  if (items > 0x7fffffffll) return -3;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(FG_THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (PAIR) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(2 * (sm_count / 2));
    int most = known ? resident_pairs[dev] : 0;
    if (most == 0) {
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        n = sm_count / 2;
      }
      most = n < sm_count / 2 ? n : sm_count / 2;
      if (known) resident_pairs[dev] = most;
    }
    cfg.gridDim = dim3(2 * (unsigned)(items < most ? items : most));
  } else {
    cfg.gridDim = dim3((unsigned)(items < sm_count ? items : sm_count));
  }
  cudaError_t e = LaunchAfter<FusedMaps, FusedParams>{kern, cfg}(maps, p);
  return (int)e;
}

bool fused_pairs(Job job, long long M, long long N, int sm_count) {
  if (sm_count < 2) return false;
  const long long nt = job == GLU_FWD ? 128 : 256;
  // rounds of pair tiles over half as many pairs as SMs against rounds of single tiles, which take 0.55 of as long
  const long long t2 = ((M + 255) / 256) * ((N + nt - 1) / nt), t1 = ((M + 127) / 128) * ((2 * N + nt - 1) / nt);
  const long long w2 = (t2 + sm_count / 2 - 1) / (sm_count / 2), w1 = (t1 + sm_count - 1) / sm_count;
  return 93 * w2 <= 55 * w1;
}

template <typename T, typename OutT, int JOB>
static int fused_by_tile(const FusedMaps& maps, const FusedParams& p, bool pair, const FusedCall& c) {
  return pair ? launch_fused<T, OutT, JOB, true>(maps, p, c.sm_count, c.stream)
              : launch_fused<T, OutT, JOB, false>(maps, p, c.sm_count, c.stream);
}

template <typename T>
static int fused_by_job(Job job, const FusedMaps& maps, const FusedParams& p, bool pair, const FusedCall& c) {
  switch (job) {
    case GLU_FWD: return fused_by_tile<T, T, GLU_FWD>(maps, p, pair, c);
    case GLU_BWD: return fused_by_tile<T, T, GLU_BWD>(maps, p, pair, c);
    case HEAD_STATS: return fused_by_tile<T, T, HEAD_STATS>(maps, p, pair, c);
    case HEAD_DZ: return fused_by_tile<T, T, HEAD_DZ>(maps, p, pair, c);
    case HEAD_DX: return fused_by_tile<T, float, HEAD_DX>(maps, p, pair, c);
    case HEAD_DW:
      if (c.out_dtype == PF_F32) return fused_by_tile<T, float, HEAD_DW>(maps, p, pair, c);
      return fused_by_tile<T, T, HEAD_DW>(maps, p, pair, c);
  }
  return -1;
}

int fused_gemm(Job job, const FusedCall& c) {
  if (c.M <= 0 || c.N <= 0) return 0;
  if (c.dtype != PF_F16 && c.dtype != PF_BF16) return -1;
  if (c.lda % 8 || c.ldb % 8 || !on_vectors(c.A, c.B, c.C, c.gu, c.dgu)) return -2;
  const int fmt = c.dtype == PF_BF16;
  const bool pair = fused_pairs(job, c.M, c.N, c.sm_count);
  FusedMaps maps;
  memset(&maps, 0, sizeof(maps));
  int r;
  const char* B = static_cast<const char*>(c.B);
  if (job == HEAD_DW) r = make_tmap_2d_16bit(&maps.a, c.A, fmt, c.M, c.K, c.lda, 64, FG_BK);
  else r = make_tmap_2d_16bit(&maps.a, c.A, fmt, c.K, c.M, c.lda, FG_BK, FG_BM);
  if (r) return r;
  if (job == GLU_FWD) {
    const int rows = pair ? FG_BN : FG_BN / 2;
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.K, c.N, c.ldb, FG_BK, rows)) ||
        (r = make_tmap_2d_16bit(&maps.b2, B + c.ldb * 2 * c.N, fmt, c.K, c.N, c.ldb, FG_BK, rows)))
      return r;
  } else if (job == HEAD_STATS || job == HEAD_DZ) {
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.K, c.N, c.ldb, FG_BK, FG_BN))) return r;
  } else {
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.N, c.K, c.ldb, 64, FG_BK))) return r;
  }
  if (job == GLU_FWD || job == GLU_BWD) {
    char* two = static_cast<char*>(job == GLU_FWD ? c.gu : c.dgu);
    if ((r = make_tmap_out(&maps.c0, c.C, c.dtype, c.N, c.M, c.ldc))) return r;
    if (two && ((r = make_tmap_out(&maps.c1, two, c.dtype, c.N, c.M, 2ll * c.N)) ||
                (r = make_tmap_out(&maps.c2, two + 2ll * c.N, c.dtype, c.N, c.M, 2ll * c.N))))
      return r;
  } else if (job == HEAD_DZ) {
    // rows up to the end of the last tile are written
    const int rows = (c.M + 2 * FG_BM - 1) / (2 * FG_BM) * (2 * FG_BM);
    if ((r = make_tmap_out(&maps.c0, c.C, c.dtype, c.N, rows, c.ldc))) return r;
  } else if (job == HEAD_DX) {
    const long long rows = c.split > 1 ? (long long)c.split * c.part_rows : c.M;
    if ((r = make_tmap_out(&maps.c0, c.C, PF_F32, c.N, rows, c.ldc))) return r;
  } else if (job == HEAD_DW) {
    if ((r = make_tmap_out(&maps.c0, c.C, c.out_dtype, c.N, c.M, c.ldc))) return r;
  }
  FusedParams p;
  memset(&p, 0, sizeof(p));
  p.M = c.M; p.N = c.N; p.K = c.K; p.fmt = fmt;
  p.group_m = FG_GROUP_ROWS / (pair ? 2 * FG_BM : FG_BM);
  p.rows = c.rows; p.status = c.status;
  p.gu = c.gu; p.bias = c.bias; p.bias_dtype = c.bias_dtype; p.act = c.act; p.save = job == GLU_FWD && c.gu;
  p.labels = c.labels; p.parts = c.parts; p.part_pitch = c.part_pitch; p.picked = c.picked; p.stats = c.stats;
  p.factor = c.factor; p.unit = c.unit;
  p.first = c.first; p.split = job == HEAD_DX ? c.split : 1; p.part_rows = c.part_rows; p.accumulate = c.accumulate;
  p.scale = c.scale; p.scale2 = c.scale2; p.scale3 = c.scale3;
  return c.dtype == PF_F16 ? fused_by_job<__half>(job, maps, p, pair, c)
                           : fused_by_job<__nv_bfloat16>(job, maps, p, pair, c);
}

}  // namespace pf

using namespace pf;

// h [M, H] = act(x Wg^T + bg) * (x Wu^T + bu) with Wg, Wu the first and the last H rows of w [2H, K]; gu [M, 2H], where
// given, keeps both projections for the backward.  act: 1 GELU (erf), 2 GELU (tanh), 3 SiLU.  K and H are multiples of
// 8, rows of x and w start on 16 bytes; h and gu are packed.
PF_API int pf_glu_linear_fwd(const void* x, const void* w, const void* bias, int bias_dtype, void* h, void* gu, int M,
                             int H, int K, long long ldx, long long ldw, int act, int dtype, int* status, int sm_count,
                             void* stream) {
  if (act < 1 || act > 3) return -1;
  if (H % 8 || K % 8) return -2;
  FusedCall c;
  c.M = M; c.N = H; c.K = K; c.A = x; c.B = w; c.lda = ldx; c.ldb = ldw; c.dtype = dtype;
  c.C = h; c.ldc = H; c.gu = gu; c.bias = bias; c.bias_dtype = bias_dtype; c.act = act; c.status = status;
  c.sm_count = sm_count > 0 ? sm_count : 148; c.stream = reinterpret_cast<cudaStream_t>(stream);
  return fused_gemm(GLU_FWD, c);
}

// From dy [M, K], w2 [K, H] and the kept gu [M, 2H]: dgu [M, 2H], the gradient of gu, and h [M, H] once more.
PF_API int pf_glu_linear_bwd(const void* dy, const void* w2, const void* gu, void* dgu, void* h, int M, int H, int K,
                             long long lddy, long long ldw2, int act, int dtype, int* status, int sm_count,
                             void* stream) {
  if (act < 1 || act > 3) return -1;
  if (H % 8 || K % 8) return -2;
  FusedCall c;
  c.M = M; c.N = H; c.K = K; c.A = dy; c.B = w2; c.lda = lddy; c.ldb = ldw2; c.dtype = dtype;
  c.C = h; c.ldc = H; c.gu = const_cast<void*>(gu); c.dgu = dgu; c.act = act; c.status = status;
  c.sm_count = sm_count > 0 ? sm_count : 148; c.stream = reinterpret_cast<cudaStream_t>(stream);
  return fused_gemm(GLU_BWD, c);
}
