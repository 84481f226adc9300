// Products on tcgen05 whose epilogue is the operator: the gated feed-forward block in both directions, and the
// output head with its cross entropy, whose logits stay in TMEM.
//
// The main loop is that of gemm_sm100.cu: persistent CTAs, warp 0 the TMA producer, warp 1 the issuer of the
// products, the other warps the epilogue (a row per thread), accumulators twice in TMEM so that an epilogue runs
// under the next tile's products.  Tiles are 256 x 256 of a CTA pair (cta_group::2) or 128 x 128 of one CTA.
//
// In short runs on a B200, rows x columns x reduction, bf16:
//   GLU_FWD     2048 x (2 x 11008) x 4096   254 us  1.45 PFLOP/s    16384 x (2 x 2560) x 640   94 us  1.14 PFLOP/s
//   GLU_BWD     2048 x 11008 x 4096         154 us  1.20            16384 x 2560 x 640        117 us  0.46
//   HEAD_STATS  2048 x 32000 x 4096         330 us  1.63            13 x 32000 x 4096          58 us  4.5 TB/s of W
//   HEAD_DZ     the same                    339 us  1.58                                       48 us  5.5 TB/s
//   PARTS_N     2048 x 4096 x 32000         370 us  1.45            13 x 4096 x 32000          42 us  6.2 TB/s
//   HEAD_DW     32000 x 4096 x 2048         345 us  1.56            32000 x 4096 x 13          50 us  5.2 TB/s written
// Products of many rows are bound by the tensor cores, or by rounds that tiles do not fill: PARTS_N above has 128 tiles for
// 74 pairs, 86 % of two rounds.  GLU_BWD moves 10 bytes for each of its values (420 MB for the short reduction, 63 us) and
// has the longest epilogue, which a reduction of 640 does not cover.  Products of few rows are bound by memory.
//
// GLU_FWD: a tile has as many gate columns as up columns.  What is kept of both is saturated: h of a gate of 7e4 and an up
// value of 0.5 is finite in fp16, and a kept infinity would turn its gradients into NaN at any loss scale.  B comes from two tensor maps, the gate and the up rows of
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
// Epilogue warps: a warp has 32 rows and, of a pair's tile, a fourth of its columns, of a single tile's a half.  With half
// as many, two a scheduler that each wait for their own results, an epilogue shows behind reductions of up to 1280 values.
constexpr int epi_warps(bool pair) { return pair ? 16 : 8; }
constexpr int fg_threads(bool pair) { return 64 + 32 * epi_warps(pair); }
constexpr int FG_STAGE_BYTES = (FG_BM + FG_BN) * FG_BK * 2;
constexpr int FG_GROUP_ROWS = 4096;                      // see GROUP_ROWS in gemm_sm100.cu
constexpr long long FG_B_STAYS = 48ll << 20;             // bytes of B that stay in L2 beside what streams through it

// Shared memory of a job: stages of operands, barriers, and the boxes (32 rows of BW columns) in which an epilogue warp
// turns its rows of the accumulator into lines of the output.
template <int JOB, typename OutT, bool PAIR>
struct FusedSmem {
  static constexpr int HC = JOB == GLU_FWD ? 32 : 64;               // output columns of a warp
  static constexpr int BW = sizeof(OutT) == 4 || JOB == GLU_FWD || JOB == GLU_BWD ? 32 : 64;
  static constexpr int BOX = 32 * BW * sizeof(OutT);
  static constexpr int BOXES = JOB == GLU_FWD || JOB == GLU_BWD ? 2 : JOB == HEAD_STATS ? 0 : 1;
  static constexpr int PER_WARP = BOXES * BOX;
  static constexpr int STAGING = epi_warps(PAIR) * PER_WARP;
  static constexpr int STAGES = STAGING <= 32768 ? 6 : 5;
  static constexpr int BAR_OFFSET = STAGES * FG_STAGE_BYTES;
  static constexpr int STAGING_OFFSET = BAR_OFFSET + 1024;
  // With A boxes of fewer rows there are as many stages as have room.  (13 rows over 11008 x 4096 weights, 11 for 6:
  // products with N innermost 40 us for 44, K innermost 34 for 35, GLU_BWD 26 for 30.)
  static constexpr int MOST = PAIR ? STAGES : 12;
  static constexpr int stages(int a_rows) {
    const int n = BAR_OFFSET / ((a_rows + FG_BN) * FG_BK * 2);
    return n < MOST ? n : MOST;
  }
  static constexpr int TOTAL = STAGING_OFFSET + STAGING + 1024;
  static_assert(TOTAL <= 232448, "more than a CTA may have");
};

struct FusedMaps { CUtensorMap a, b, b2, c; };          // c: of an output that is added to

struct FusedParams {
  int M, N, K, fmt, group_m;
  void* C;                       // h | h | - | dz | parts | parts | dW
  void* two;                     // gate and up [M, 2 N], or their gradients
  long long ldc;
  int c_rows;                    // rows of C that may be written
  int a_rows;                    // rows of A that a CTA loads: all of a tile's, or as many as there are, in eights
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
  PartRule rule;
  int* parts_word;
  void* direct;
  const int* list;
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
__device__ __forceinline__ void sigmoid_act2(uint64_t z, uint64_t q, uint64_t dq, uint64_t& a, uint64_t& d) {
  float q0, q1, d0, d1;
  f2_unpack(mul2(q, f2_pack(-LOG2E, -LOG2E)), q0, q1);
  f2_unpack(add2(f2_pack(ex2(q0), ex2(q1)), f2_pack(1.f, 1.f)), d0, d1);
  const uint64_t s = f2_pack(rcp_approx(d0), rcp_approx(d1));
  a = mul2(z, s);
  if (SLOPE) d = fma2(fma2(mul2(a, f2_pack(-1.f, -1.f)), s, a), dq, s);      // s + (a - a s) q'
}
template <int ACT, bool SLOPE>
__device__ __forceinline__ void act2(float z0, float z1, uint64_t& a, uint64_t& d) {
  if constexpr (ACT == 1) {                             // GELU with erf
    uint64_t e;
    const uint64_t az = f2_pack(fabsf(z0), fabsf(z1));
    const uint64_t ny = gelu_neg_tail2(az, e);
    a = fma2(az, ny, f2_pack(fmaxf(z0, 0.f), fmaxf(z1, 0.f)));
    if (SLOPE) {
      float y0, y1, c0, c1;
      f2_unpack(ny, y0, y1);
      f2_unpack(add2(ny, f2_pack(1.f, 1.f)), c0, c1);
      d = fma2(mul2(f2_pack(z0, z1), f2_pack(0.3989422804014327f, 0.3989422804014327f)), e,
               f2_pack(z0 >= 0.f ? c0 : -y0, z1 >= 0.f ? c1 : -y1));
    }
  } else if constexpr (ACT == 2) {                      // GELU with tanh
    constexpr float c = 2.f * 0.7978845608028654f;
    const uint64_t z = f2_pack(z0, z1), z2 = mul2(z, z);
    const uint64_t q = mul2(mul2(z, f2_pack(c, c)), fma2(z2, f2_pack(0.044715f, 0.044715f), f2_pack(1.f, 1.f)));
    uint64_t dq = 0;
    if (SLOPE) {
      float s0, s1;
      f2_unpack(z2, s0, s1);
      dq = fma2(f2_pack(fminf(s0, 1e6f), fminf(s1, 1e6f)), f2_pack(3.f * 0.044715f * c, 3.f * 0.044715f * c),
                f2_pack(c, c));
    }
    sigmoid_act2<SLOPE>(z, q, dq, a, d);
  } else {                                              // SiLU
    const uint64_t z = f2_pack(z0, z1);
    sigmoid_act2<SLOPE>(z, z, f2_pack(1.f, 1.f), a, d);
  }
}

// The values of an accumulator are in registers (tcgen05.wait::ld) and nothing else is handed over with this arrival: a
// release would first wait for the stores that are on their way to memory.  (dW of 13 rows, 262 MB of stores, 72 us with a
// release and 50 so; GLU_FWD over 16384 x 2560 at a reduction of 640 100 and 86.)
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// A bias in its own type, and what it is: apart, so that nothing waits for the load
__device__ __forceinline__ uint32_t bias_bits(const void* b, int dtype, int i) {
  if (dtype == PF_F32) return __ldg(static_cast<const uint32_t*>(b) + i);
  return __ldg(static_cast<const uint16_t*>(b) + i);
}
__device__ __forceinline__ float bias_value(uint32_t bits, int dtype) {
  if (dtype == PF_F32) return __uint_as_float(bits);
  if (dtype == PF_F16) return __half2float(__ushort_as_half((unsigned short)bits));
  return __uint_as_float(bits << 16);
}
// see tmem_ld_wait_for in common.cuh
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15])
      :
      : "memory");
}

// Where 16 bytes lie in a box, as TMA has it for outputs that are added to: chunk c of row r, rows of 128 bytes swizzled
// over 128 or of 64 over 64.
// The 16-byte accesses of eight lanes, of one row or one chunk, meet no bank twice.
template <int ROW_BYTES>
__device__ __forceinline__ uint4* box_at(uint8_t* box, int r, int c) {
  const int at = ROW_BYTES == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3));
  return reinterpret_cast<uint4*>(box + r * ROW_BYTES + at * 16);
}
// 32 columns of a row, from the box's column `c0` on
template <typename OutT, int ROW_BYTES>
__device__ __forceinline__ void fill_box(uint8_t* box, int r, int c0, const float (&v)[32]) {
  constexpr int PER = 16 / sizeof(OutT);
#pragma unroll
  for (int c = 0; c < 32 / PER; ++c) {
    uint4 q;
    OutT* e = reinterpret_cast<OutT*>(&q);
#pragma unroll
    for (int j = 0; j < PER; ++j) e[j] = from_f32<OutT>(v[c * PER + j]);
    *box_at<ROW_BYTES>(box, r, c0 / PER + c) = q;
  }
}

template <typename T, typename OutT, int JOB, bool PAIR>
__global__ void __launch_bounds__(fg_threads(PAIR), 1)
fused_gemm_kernel(const __grid_constant__ FusedMaps maps, const FusedParams p) {
  using S = FusedSmem<JOB, OutT, PAIR>;
  constexpr bool A_MN = JOB == HEAD_DW;
  constexpr bool B_MN = JOB == GLU_BWD || JOB == PARTS_N || JOB == HEAD_DW;
  constexpr bool PARTS = JOB == PARTS_K || JOB == PARTS_N;
  constexpr int BMT = PAIR ? 2 * FG_BM : FG_BM;
  constexpr int BNT = PAIR ? 2 * FG_BN : FG_BN;           // accumulator columns of a tile
  constexpr int NT = JOB == GLU_FWD ? BNT / 2 : BNT;      // output columns of a tile
  const int a_bytes = PAIR || A_MN ? FG_BM * FG_BK * 2 : p.a_rows * FG_BK * 2;
  const int STAGES = PAIR || A_MN ? S::STAGES : S::stages(p.a_rows), stage_bytes = a_bytes + FG_BN * FG_BK * 2;
  constexpr uint32_t TMEM_COLS = 2 * BNT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::BAR_OFFSET);
  uint64_t* empty_bar = full_bar + S::MOST;
  uint64_t* tmem_full = empty_bar + S::MOST;
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
      mbar_init(&tmem_empty[i], (PAIR ? 2 : 1) * epi_warps(PAIR));      // lane 0 of every epilogue warp
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
  const int num_kb = (K + FG_BK - 1) / FG_BK;
  // a last piece of few words adds to the first parts only
  const int split = !PARTS ? 1 : p.rows ? max(1, min(parts_of(p.rule, count), num_kb / 8)) : p.split;
  const int part_rows = PARTS && p.rows ? rows_of_part(count) : p.part_rows;
  if (PARTS && p.parts_word && blockIdx.x == 0 && threadIdx.x == 0) *p.parts_word = split;
  const int num_items = num_mn * split;
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
          uint8_t* sa = smem + stage * stage_bytes;
          uint8_t* sb = sa + a_bytes;
          const int k0 = kb * FG_BK;
          if (!PAIR || cta_rank == 0)
            mbar_expect_tx(&full_bar[stage], (PAIR ? 2 : 1) * stage_bytes);
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
          const uint32_t sa = smem_u32(smem + stage * stage_bytes);
          const uint32_t a_lo = desc_lo(sa, a_lbo), b_lo = desc_lo(sa + a_bytes, b_lbo);
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
    constexpr int HC = S::HC, BW = S::BW, RB = BW * sizeof(OutT);        // columns of a warp, of a box; bytes of a row
    static_assert(HC * epi_warps(PAIR) == 4 * NT, "the warps share a tile's columns");
    const int c_begin = side * HC, c_end = c_begin + HC;
    uint8_t* boxes = smem + S::STAGING_OFFSET + (warp - 2) * S::PER_WARP;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    // A box that the warp has filled, to memory: 16 bytes a lane, whole rows of the box behind one another.
    constexpr int CPR = RB / 16, RPI = 32 / CPR, PER = 16 / sizeof(OutT);      // chunks of a row, rows of an access
    auto store = [&](uint8_t* box, void* C, long long ldc, int col, int row0, int rows) {
      __syncwarp();
      const int r = lane / CPR, c = col + (lane % CPR) * PER;
      OutT* dst = static_cast<OutT*>(C) + (long long)(row0 + r) * ldc + c;
      const long long step = RPI * ldc;
      if (row0 + 32 <= rows && col + BW <= p.N) {
#pragma unroll
        for (int i = 0; i < CPR; ++i, dst += step)
          *reinterpret_cast<uint4*>(dst) = *box_at<RB>(box, i * RPI + r, lane % CPR);
      } else {
#pragma unroll
        for (int i = 0; i < CPR; ++i, dst += step)
          if (row0 + i * RPI + r < rows && c < p.N)
            *reinterpret_cast<uint4*>(dst) = *box_at<RB>(box, i * RPI + r, lane % CPR);
      }
      __syncwarp();
    };
    float alpha = 1.f;
    const bool direct = PARTS && p.direct && split == 1;
    if (JOB == HEAD_DW || direct) alpha = (p.scale ? *p.scale : 1.f) * (p.scale2 ? *p.scale2 : 1.f) * p.scale3;

    // GLU backward: gate and up of one of the warp's two chunks of 32 columns, in boxes whose places their gradients take.
    // The next is asked for as soon as a chunk has left its boxes, 16 bytes a lane and whole rows of a box behind one
    // another: a lane that read its own row would touch 32 lines with every load.  (Two sets of boxes, for both chunks, and
    // three stages of operands: 84 us for 87 over 8192 x 4096 at a reduction of 640, 124 for 115 at 1536, 256 for 228 at
    // 4096.)
    auto fetch = [&](int chunk, int round) {
      if constexpr (JOB == GLU_BWD) {
        const int item = item_of(round);
        if (item < num_items) {
          int mt, nt, kb0, kb1;
          place(item, mt, nt, kb0, kb1);
          const int row0 = mt * BMT + int(cta_rank) * FG_BM + quad * 32;
          const int c = nt * NT + c_begin + 32 * chunk + (lane % CPR) * 8;
          uint8_t* box = boxes;
#pragma unroll
          for (int i = 0; i < CPR; ++i) {
            const int r = i * RPI + lane / CPR;
            uint4 *g = box_at<RB>(box, r, lane % CPR), *u = box_at<RB>(box + S::BOX, r, lane % CPR);
            if (row0 + r < M && c < p.N) {              // N is a multiple of 8
              const T* at = reinterpret_cast<const T*>(p.gu) + (long long)(row0 + r) * 2 * p.N + c;
              cp_async16(g, at);
              cp_async16(u, at + p.N);
            } else {
              *g = *u = make_uint4(0, 0, 0, 0);
            }
          }
        }
        cp_async_commit();
      }
    };
    // GLU forward: a lane has the biases of one gate and one up column of the next tile; they reach the other lanes through
    // those chunks of the first four rows of the box that the same half of the columns takes up.  (As loads behind those of
    // the accumulator, by every lane: 118 us for 99 without biases over 16384 x 2560 at a reduction of 640.)
    uint32_t bias_g = 0, bias_u = 0;
    auto fetch_bias = [&](int round) {
      if constexpr (JOB == GLU_FWD) {
        const int item = item_of(round);
        if (!p.bias || item >= num_items) return;
        int mt, nt, kb0, kb1;
        place(item, mt, nt, kb0, kb1);
        const int c = nt * NT + c_begin + lane;
        if (c < p.N) {
          bias_g = bias_bits(p.bias, p.bias_dtype, c);
          bias_u = bias_bits(p.bias, p.bias_dtype, p.N + c);
        }
      }
    };
    auto bias_box = [&](int half, int quad) { return box_at<RB>(boxes, quad >> 1, 2 * half + (quad & 1)); };
    auto add4 = [](const uint4& b, float (&v)[16], int i) {
      f2_unpack(add2(f2_pack(v[i], v[i + 1]), f2_pack(__uint_as_float(b.x), __uint_as_float(b.y))), v[i], v[i + 1]);
      f2_unpack(add2(f2_pack(v[i + 2], v[i + 3]), f2_pack(__uint_as_float(b.z), __uint_as_float(b.w))), v[i + 2], v[i + 3]);
    };
    fetch_bias(0);
    auto fetch_next = [&](int c, int round) { fetch(c == c_begin, c == c_begin ? round : round + 1); };
    fetch(0, 0);
    for (int round = 0, item = item_of(0); item < num_items && ok; item = item_of(++round)) {
      int mt, nt, kb0, kb1;
      const int ks = place(item, mt, nt, kb0, kb1);
      const int row0 = mt * BMT + int(cta_rank) * FG_BM + quad * 32, row = row0 + lane;
      const int n0 = nt * NT;
      const bool row_ok = row < M;
      [[maybe_unused]] int target = 0;                  // row of `direct` that the lane's row goes to
      if (direct && row_ok) target = p.list[row];

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

      if (JOB == GLU_FWD && p.bias) {
        const int half = lane >> 4, at = lane & 15;
        reinterpret_cast<float*>(bias_box(half, at >> 2))[at & 3] = bias_value(bias_g, p.bias_dtype);
        reinterpret_cast<float*>(bias_box(half, 4 + (at >> 2)))[at & 3] = bias_value(bias_u, p.bias_dtype);
        __syncwarp();
        fetch_bias(round + 1);
      }
      const bool empty = kb0 == kb1;
      if (!empty) {
        ok = mbar_wait(&tmem_full[acc], acc_phase, p.status, PF_ERR_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t t_row = tmem_base + (uint32_t(quad * 32) << 16) + acc * BNT;
      // the accumulator may be written again: called once its last columns are in registers
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) arrive_relaxed(mapa_u32(&tmem_empty[acc], 0));
          else mbar_arrive(&tmem_empty[acc]);
        }
      };
      const int last = min(c_end, (p.N - n0 + 31) / 32 * 32) - 32;      // first of the last 32 columns there are
      if (!empty && last < c_begin) release();          // none: the whole warp is behind the last column
      auto values = [&](const uint32_t (&raw)[32], float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]);
      };
#pragma unroll 1
      for (int c = c_begin; c < c_end; c += BW) {
        const int col = n0 + c;
        if (col >= p.N) {                               // uniform across the warp
          if (JOB == GLU_BWD) fetch_next(c, round);
          continue;
        }
        uint32_t raw[32];
        float v[32];
        if constexpr (JOB == GLU_FWD) {
          uint4 hq[4];                                  // h, which takes the place of the gate once that is stored
#pragma unroll
          for (int s = 0; s < 32; s += 16) {
            uint32_t gate[16], up[16];
            float g[16], u[16];
            tmem_ld16(t_row + c + s, gate);
            tmem_ld16(t_row + NT + c + s, up);
            tmem_ld_wait_for(gate);
            tmem_ld_wait_for(up);
            if (s) release();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              g[i] = __uint_as_float(gate[i]);
              u[i] = __uint_as_float(up[i]);
            }
            if (p.bias) {                                // no lane writes where another still reads
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint4 bg = *bias_box(s / 16, k), bu = *bias_box(s / 16, 4 + k);
                add4(bg, g, 4 * k);
                add4(bu, u, 4 * k);
              }
              __syncwarp();
            }
            auto packed = [&](const float (&v)[16], int k) {
              uint4 q;
              OutT* e = reinterpret_cast<OutT*>(&q);
#pragma unroll
              for (int j = 0; j < 8; ++j) e[j] = from_f32<OutT>(v[8 * k + j]);
              return q;
            };
            if (p.save) {                                // within the type: h may be where a gate is not
              auto kept = [&](const float (&v)[16], int k) {
                const float* e = v + 8 * k;
                return make_uint4(saturated2<OutT>(e[0], e[1]), saturated2<OutT>(e[2], e[3]),
                                  saturated2<OutT>(e[4], e[5]), saturated2<OutT>(e[6], e[7]));
              };
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                *box_at<RB>(boxes, lane, s / 8 + k) = kept(g, k);
                *box_at<RB>(boxes + S::BOX, lane, s / 8 + k) = kept(u, k);
              }
            }
            auto all = [&](auto kind) {
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                uint64_t a, none;
                act2<decltype(kind)::value, false>(g[i], g[i + 1], a, none);
                f2_unpack(mul2(a, f2_pack(u[i], u[i + 1])), g[i], g[i + 1]);
              }
            };
            if (p.act == 1) all(std::integral_constant<int, 1>());
            else if (p.act == 2) all(std::integral_constant<int, 2>());
            else all(std::integral_constant<int, 3>());
            hq[s / 8] = packed(g, 0);
            hq[s / 8 + 1] = packed(g, 1);
          }
          if (p.save) {
            store(boxes, p.two, 2ll * p.N, col, row0, M);
            store(boxes + S::BOX, static_cast<OutT*>(p.two) + p.N, 2ll * p.N, col, row0, M);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) *box_at<RB>(boxes, lane, k) = hq[k];
          store(boxes, p.C, p.ldc, col, row0, M);
        } else if constexpr (JOB == GLU_BWD) {
          uint8_t *gbox = boxes, *ubox = boxes + S::BOX;
          uint4 hq[BW / 8];                             // h, which takes the place of d(gate) once that is stored
          cp_async_wait<0>();
          __syncwarp();
#pragma unroll
          for (int s = 0; s < BW; s += 16) {
            uint32_t part[16];
            tmem_ld16(t_row + c + s, part);
            tmem_ld_wait_for(part);
            if (c + s == last + 16) release();
            auto all = [&](auto kind) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint4 *gp = box_at<RB>(gbox, lane, s / 8 + k), *up = box_at<RB>(ubox, lane, s / 8 + k);
                uint4 g4 = *gp, u4 = *up;
                T *g = reinterpret_cast<T*>(&g4), *u = reinterpret_cast<T*>(&u4), *h = reinterpret_cast<T*>(&hq[s / 8 + k]);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                  const uint64_t dh = f2_pack(__uint_as_float(part[8 * k + j]), __uint_as_float(part[8 * k + j + 1]));
                  const uint64_t uu = f2_pack(to_f32<T>(u[j]), to_f32<T>(u[j + 1]));
                  uint64_t a, slope;
                  act2<decltype(kind)::value, true>(to_f32<T>(g[j]), to_f32<T>(g[j + 1]), a, slope);
                  float x0, x1;
                  f2_unpack(mul2(mul2(dh, uu), slope), x0, x1);        // d(gate) = dh up act'(gate)
                  g[j] = from_f32<T>(x0);
                  g[j + 1] = from_f32<T>(x1);
                  f2_unpack(mul2(a, uu), x0, x1);
                  h[j] = from_f32<T>(x0);
                  h[j + 1] = from_f32<T>(x1);
                  f2_unpack(mul2(dh, a), x0, x1);                      // d(up) = dh act(gate)
                  u[j] = from_f32<T>(x0);
                  u[j + 1] = from_f32<T>(x1);
                }
                *gp = g4;
                *up = u4;
              }
            };
            if (p.act == 1) all(std::integral_constant<int, 1>());
            else if (p.act == 2) all(std::integral_constant<int, 2>());
            else all(std::integral_constant<int, 3>());
          }
          store(gbox, p.two, 2ll * p.N, col, row0, M);
          store(ubox, static_cast<OutT*>(p.two) + p.N, 2ll * p.N, col, row0, M);
#pragma unroll
          for (int k = 0; k < BW / 8; ++k) *box_at<RB>(gbox, lane, k) = hq[k];
          store(gbox, p.C, p.ldc, col, row0, M);
          fetch_next(c, round);
        } else if constexpr (JOB == HEAD_STATS) {
#pragma unroll
          for (int s = 0; s < BW; s += 32) {
            const int at = col + s, nvalid = p.N - at;
            if (s && nvalid <= 0) break;
            tmem_ld32(t_row + c + s, raw);
            tmem_ld_wait_for(raw);
            if (c + s == last) release();
            values(raw, v);
            if (nvalid < 32) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i >= nvalid) v[i] = -INFINITY;
            }
            if ((unsigned)(label - at) < 32u) {
              float z = 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i == label - at) z = v[i];
              p.picked[row] = z;
            }
            // a NaN does not move the maximum but reaches the sum; a part that is -inf so far subtracts 0
            float top = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
            const float now = fmaxf(ref, ceilf(top * LOG2E)), sub = now == -INFINITY ? 0.f : now;
            total *= ex2(ref - sub);
            uint64_t sum = 0;
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float e0, e1;
              f2_unpack(fma2(f2_pack(v[i], v[i + 1]), f2_pack(LOG2E, LOG2E), f2_pack(-sub, -sub)), e0, e1);
              sum = add2(sum, f2_pack(ex2(e0), ex2(e1)));
            }
            float s0, s1;
            f2_unpack(sum, s0, s1);
            total += s0 + s1;
            ref = now;
          }
        } else {
          if (sizeof(OutT) == 4 && p.accumulate) {      // the last box is read before it is filled again
            if (lane == 0) tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int s = 0; s < BW; s += 32) {
            if (s && col + s >= p.N) break;
            if (!empty) {
              tmem_ld32(t_row + c + s, raw);
              tmem_ld_wait_for(raw);
              if (c + s == last) release();
              values(raw, v);
            }
            if (JOB == HEAD_DZ) {
              // (p - onehot) factor; rows behind the last have zeros, which the reduction over rows may read
              const uint64_t times = f2_pack(inv * factor, inv * factor);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float e0, e1;
                f2_unpack(fma2(f2_pack(v[i], v[i + 1]), f2_pack(LOG2E, LOG2E), f2_pack(-ref, -ref)), e0, e1);
                f2_unpack(mul2(f2_pack(ex2(e0), ex2(e1)), times), v[i], v[i + 1]);
              }
              const int at = label - col - s;
              if ((unsigned)at < 32u) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i == at) v[i] -= factor;
              }
              if (row0 + 32 > M && !row_ok) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0.f;
              }
            } else if (JOB == HEAD_DW || direct) {
              if (empty) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0.f;
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 2)
                  f2_unpack(mul2(f2_pack(v[i], v[i + 1]), f2_pack(alpha, alpha)), v[i], v[i + 1]);
              }
            }
            if (direct) fill_box<T, 64>(boxes, lane, 0, v);
            else fill_box<OutT, RB>(boxes, lane, s, v);
          }
          if (direct) {                                 // 16 bytes a lane, 64 of each row
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 8 * i + (lane >> 2), to = __shfl_sync(0xffffffffu, target, r), at = col + (lane & 3) * 8;
              if (row0 + r < M && at < p.N)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.direct) + (long long)to * p.N + at) =
                    *box_at<64>(boxes, r, lane & 3);
            }
            __syncwarp();
            continue;
          }
          const int part = PARTS ? ks * part_rows : 0;
          if (sizeof(OutT) == 4 && p.accumulate) {      // rows and columns that do not exist are clipped
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row0 < M) tma_reduce_add_2d(&maps.c, boxes, col, row0 + part);
              tma_store_commit();
            }
          } else {
            store(boxes, p.C, p.ldc, col, row0 + part, JOB == HEAD_DZ ? p.c_rows : M + part);
          }
        }
      }
      if constexpr (JOB == HEAD_STATS) {
        const int part = (n0 + c_begin) / HC;
        if (row_ok && n0 + c_begin < p.N) p.parts[part * p.part_pitch + row] = {ref, total};
      }
      if (!empty) {
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
    if (lane == 0 && p.accumulate) tma_store_wait_all();
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
  using S = FusedSmem<JOB, OutT, PAIR>;
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
  long long items = (long long)((p.M + BMT - 1) / BMT) * ((p.N + NT - 1) / NT) * p.split;
  if (items > 0x7fffffffll) return -3;
  if (p.rule.rows && items < sm_count) items = sm_count;               // fewer rows may come in more parts
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(fg_threads(PAIR));
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
    // what the device takes is the same for every call, what a call is given is not
    int most = known ? resident_pairs[dev] : 0;
    if (most == 0) {
      if (cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess || most <= 0) {
        (void)cudaGetLastError();
        most = 0;
      }
      if (known) resident_pairs[dev] = most;
    }
    if (most == 0 || most > sm_count / 2) most = sm_count / 2;
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
  // rounds of pair tiles over half as many pairs as SMs against rounds of single tiles (see plan_parts)
  const long long t2 = ((M + 255) / 256) * ((N + nt - 1) / nt), t1 = ((M + 127) / 128) * ((2 * N + nt - 1) / nt);
  const long long w2 = (t2 + sm_count / 2 - 1) / (sm_count / 2), w1 = (t1 + sm_count - 1) / sm_count;
  return 37 * w2 <= 25 * w1;
}

// In microseconds, as measured: a k-block of 64 costs a pair's tile 0.37 and a single one 0.25, or what memory brings of B
// (5.5 TB/s over all that run at once; tiles of one column share it); an item costs 1.5 more of them, parts their way
// through memory and a launch.  (2048 x 4096 outputs never gain by it; over 22016: 512 rows whole 101, in two parts over
// pairs 72; 256 rows 97 and in four 46; 13 rows 115 and in 13 over single tiles 43.)
PartPlan plan_parts(long long M, long long N, long long K, int sm_count, bool joined) {
  PartPlan best;
  double least = 1e30;
  const long long kb = (K + FG_BK - 1) / FG_BK;
  for (int pair = 0; pair <= (M > FG_BM && sm_count >= 2); ++pair) {
    const long long bt = pair ? 2 * FG_BM : FG_BM, slots = pair ? sm_count / 2 : sm_count;
    const long long rows = (M + bt - 1) / bt, tiles = rows * ((N + bt - 1) / bt);
    const double each = pair ? 0.37 : 0.25, fed = (double)(bt * FG_BK * 2) / rows * slots / 5.5e6;
    for (int p = 1; p <= 16 && (p == 1 || (kb >= 8ll * p && p * M * N <= (64ll << 20))); ++p) {
      const long long items = tiles * p, full = items / slots, rest = items % slots;
      const double blocks = (double)((kb + p - 1) / p) + 1.5;
      double t = full * blocks * (each > fed ? each : fed);
      const double last = fed * rest / slots;
      if (rest) t += blocks * (each > last ? each : last);
      if (p > 1 || joined) t += (joined ? 0.0 : 2.0) + (double)p * M * N * 8 / 6e6;
      if (t < least * (p > 1 ? 0.97 : 1.0)) {
        least = t;
        best = {pair, p};
      }
    }
  }
  return best;
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
    case PARTS_K: return fused_by_tile<T, float, PARTS_K>(maps, p, pair, c);
    case PARTS_N: return fused_by_tile<T, float, PARTS_N>(maps, p, pair, c);
    case HEAD_DW:
      if (c.out_dtype == PF_F32) return fused_by_tile<T, float, HEAD_DW>(maps, p, pair, c);
      return fused_by_tile<T, T, HEAD_DW>(maps, p, pair, c);
  }
  return -1;
}

int fused_gemm(Job job, const FusedCall& c) {
  if (c.M <= 0 || c.N <= 0) return 0;
  if (c.dtype != PF_F16 && c.dtype != PF_BF16) return -1;
  if (c.lda % 8 || c.ldb % 8 || c.ldc % 8 || c.N % 8 && job != HEAD_STATS && job != HEAD_DZ ||
      !on_vectors(c.A, c.B, c.C, c.gu, c.dgu))
    return -2;
  const int fmt = c.dtype == PF_BF16;
  const bool pair = c.tile < 0 ? fused_pairs(job, c.M, c.N, c.sm_count) : c.tile;
  // Fewer rows than a tile has are loaded as what they are: rows of accumulators that no row of A fills are not read.  (What
  // lies behind them in shared memory, B's tile, is multiplied, too; it is inside the stage.)
  const int a_rows = pair || c.M >= FG_BM ? FG_BM : (c.M + 7) / 8 * 8;
  FusedMaps maps;
  memset(&maps, 0, sizeof(maps));
  int r;
  const char* B = static_cast<const char*>(c.B);
  if (job == HEAD_DW) r = make_tmap_2d_16bit(&maps.a, c.A, fmt, c.M, c.K, c.lda, 64, FG_BK);
  else r = make_tmap_2d_16bit(&maps.a, c.A, fmt, c.K, c.M, c.lda, FG_BK, a_rows);
  if (r) return r;
  if (job == GLU_FWD) {
    const int rows = pair ? FG_BN : FG_BN / 2;
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.K, c.N, c.ldb, FG_BK, rows)) ||
        (r = make_tmap_2d_16bit(&maps.b2, B + c.ldb * 2 * c.N, fmt, c.K, c.N, c.ldb, FG_BK, rows)))
      return r;
  } else if (job == HEAD_STATS || job == HEAD_DZ || job == PARTS_K) {
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.K, c.N, c.ldb, FG_BK, FG_BN))) return r;
  } else {
    if ((r = make_tmap_2d_16bit(&maps.b, B, fmt, c.N, c.K, c.ldb, 64, FG_BK))) return r;
  }
  if (c.accumulate && (r = make_tmap_out(&maps.c, c.C, PF_F32, c.N, c.M > c.rule.rows ? c.M : c.rule.rows, c.ldc))) return r;
  FusedParams p;
  memset(&p, 0, sizeof(p));
  p.M = c.M; p.N = c.N; p.K = c.K; p.fmt = fmt;
  p.group_m = FG_GROUP_ROWS / (pair ? 2 * FG_BM : FG_BM);
  // Where all of B stays in L2, the tiles in flight are whole rows of the output instead, which DRAM takes better (GLU_FWD
  // over 16384 x 2560 at a reduction of 640: 90 us, 93 in bands; over 8192 x 5120 at 1280: 154 and 156).
  const int bt = pair ? 2 * FG_BM : FG_BM, nt = job == GLU_FWD ? bt / 2 : bt;
  const int columns = (c.N + nt - 1) / nt, workers = pair ? c.sm_count / 2 : c.sm_count;
  if ((long long)c.N * c.K * (job == GLU_FWD ? 4 : 2) <= FG_B_STAYS) p.group_m = (workers + columns - 1) / columns;
  p.rows = c.rows; p.status = c.status;
  p.gu = c.gu; p.bias = c.bias; p.bias_dtype = c.bias_dtype; p.act = c.act; p.save = job == GLU_FWD && c.gu;
  p.labels = c.labels; p.parts = c.parts; p.part_pitch = c.part_pitch; p.picked = c.picked; p.stats = c.stats;
  p.factor = c.factor; p.unit = c.unit;
  p.a_rows = a_rows;
  p.C = c.C; p.ldc = c.ldc; p.two = job == GLU_FWD ? c.gu : c.dgu; p.c_rows = (c.M + 255) / 256 * 256;
  p.first = c.first; p.split = job == PARTS_K || job == PARTS_N ? c.split : 1; p.part_rows = c.part_rows;
  p.accumulate = c.accumulate;
  p.rule = c.rule; p.parts_word = c.parts_word; p.direct = c.direct; p.list = c.list;
  p.scale = c.scale; p.scale2 = c.scale2; p.scale3 = c.scale3;
  return c.dtype == PF_F16 ? fused_by_job<__half>(job, maps, p, pair, c)
                           : fused_by_job<__nv_bfloat16>(job, maps, p, pair, c);
}

}  // namespace pf
