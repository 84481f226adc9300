// Products whose epilogues are more than a store (fused_gemm_sm100.cu), for the entry points of the gated
// feed-forward block and of the head with its loss.
#pragma once
#include <cuda_runtime.h>

namespace pf {

enum Job : int {
  GLU_FWD,      // h = act(x Wg^T + bg) * (x Wu^T + bu), gate and up kept where asked for
  GLU_BWD,      // dh = dy W2, then d(gate), d(up) and h from the kept gate and up
  HEAD_STATS,   // per row and half a tile of z = x W^T: a reference and the sum of 2^(z log2 e - reference)
  HEAD_DZ,      // (softmax(z) - onehot) * factor of some words, in 16 bits
  PARTS_K,      // parts of A B^T in fp32, B with K innermost: products of few rows, split over their reduction
  PARTS_N,      // the same, B with N innermost
  HEAD_DW,      // dz^T x, and any weight's gradient
};

// What a row of the product has of the loss: reference and one over the sum; its label.
struct RowStat { float ref, inv; };

// Parts of a product whose rows are counted on the device: as many as keep `slots` workers busy and have room, none of
// fewer than 8 k-blocks, and no fewer than were planned for all rows.
struct PartRule {
  int tile_rows = 0, columns = 0, slots = 0;      // rows of a tile, tiles side by side
  int kb = 0, planned = 1, rows = 0;              // k-blocks of 64; rows of the parts' memory
};
__host__ __device__ inline int rows_of_part(int count) { return (count + 255) / 256 * 256; }
__host__ __device__ inline int parts_of(const PartRule& r, int count) {
  const int tiles = (count + r.tile_rows - 1) / r.tile_rows * r.columns;
  if (!tiles) return r.planned;
  int p = r.slots / tiles;
  p = p < r.kb / 8 ? p : r.kb / 8;
  p = p < r.rows / rows_of_part(count) ? p : r.rows / rows_of_part(count);
  p = p < 16 ? p : 16;
  return p > r.planned ? p : r.planned;
}

struct FusedCall {
  // product [M, N] over K.  GLU_FWD: N hidden values, each of two columns
  int M = 0, N = 0, K = 0;
  const void* A = nullptr;     // 16-bit; K innermost, but HEAD_DW: M innermost
  const void* B = nullptr;     // GLU_FWD, HEAD_STATS, HEAD_DZ, PARTS_K: K innermost, else N innermost
  long long lda = 0, ldb = 0;
  const int* rows = nullptr;   // device: how many rows there are (HEAD_DW: what to reduce over); M (K) is the most
  int dtype = 0, out_dtype = 0;
  void* C = nullptr;           // h | h | - | dz | fp32 parts | dW
  long long ldc = 0;
  // GLU
  void* gu = nullptr;          // gate and up [M, 2 N]: written (forward, may be null) or read
  void* dgu = nullptr;         // [M, 2 N]
  const void* bias = nullptr;  // [2 N]
  int bias_dtype = 0;
  int act = 0;
  // head
  const int* labels = nullptr;
  int first = 0;               // word of the first column
  RowStat* parts = nullptr;    // [N / HEAD_PART][part_pitch]: reference and sum
  long long part_pitch = 0;
  float* picked = nullptr;     // z at the label
  const RowStat* stats = nullptr;
  const float* factor = nullptr;   // of each row; null: `unit` for all
  float unit = 1.f;
  int split = 1;               // PARTS: parts of the reduction, part i in rows i * part_rows of C on
  int part_rows = 0;
  PartRule rule;               // PARTS with `rows`: its parts, each rows_of_part(*rows) rows behind the one before;
  int* parts_word = nullptr;   // how many they are, for whoever adds them up
  void* direct = nullptr;      // [*, N] 16-bit: where there is one part, its rows go, scaled, to the rows of `list` instead
  const int* list = nullptr;
  int tile = -1;               // 1: tiles of CTA pairs, 0: of one CTA; -1: as fused_pairs has it
  int accumulate = 0;          // PARTS, HEAD_DW in fp32: add to C
  const float* scale = nullptr;    // HEAD_DW, direct: *scale times *scale2 (where given) times scale3
  const float* scale2 = nullptr;
  float scale3 = 1.f;
  int* status = nullptr;
  int sm_count = 148;
  cudaStream_t stream = nullptr;
};

constexpr int HEAD_PART = 64;      // words of a part of HEAD_STATS

// 256 x 256 tiles of CTA pairs instead of 128 x 128 ones
bool fused_pairs(Job job, long long M, long long N, int sm_count);
// Tiles and parts that a product [M, N] over K is best split into; `joined`: its parts are read by a pass that would
// follow in any case.
struct PartPlan { int pair = 0, parts = 1; };
PartPlan plan_parts(long long M, long long N, long long K, int sm_count, bool joined);
int fused_gemm(Job job, const FusedCall& c);

}  // namespace pf
