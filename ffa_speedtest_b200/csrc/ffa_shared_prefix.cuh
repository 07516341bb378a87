// Decode attention over a paged fp8 + fp8-residual cache for batches whose sequences share leading pages: work split,
// partial results and merge.
//
//   o_b = softmax(scale * q_b K_b^T) V_b over the len_b tokens of sequence b,  K = base + residual
//
// The batch is cut into segments: one per sequence, holding its own pages; one per group of sequences with a shared
// prefix and 128 of its query rows (a row = one query head of one sequence), holding the group's shared pages.  A
// segment and a kv-head make a unit of ceil(tokens / 128) tiles; all units in a row are cut into ranges of equal cost,
// one per CTA.  A CTA's part of a unit is a run; every run leaves one partial (maximum, sum, output) per row, and the
// merge adds a row's partials up in the order of the tiles.  Group sizes, prefix lengths and sequence lengths are read
// on the device, so a captured call follows them.
#pragma once

#include "ffa_common.cuh"

namespace ffa {

constexpr int kSpTile = 128;                  // tokens of a tile: two pages
constexpr int kSpRows = 128;                  // query rows of a segment

// one segment of the work list
struct SpSegment {
  int32_t table_row;                          // row of the block table that names its pages
  int32_t row0;                               // first query row: sequence * G + head within the group
  int32_t rows;                               // query rows
  int32_t tiles;
  int32_t page0;                              // first column of the block table
  int32_t end;                                // token position (in the sequence) that ends it
  int32_t own;                                // 0: shared pages of a group, 1: a sequence's own pages
  int32_t pad;
};

struct SpParams {
  const void* q;                              // [B, HQ, 128]
  const uint8_t* k;                           // [n_pages * 64, HKV, 128] fp8
  const uint8_t* r;                           // residual, or null
  const uint8_t* v;                           // [n_pages * 64, HKV, 128] 16 bit
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* group_start;                 // [NG + 1]
  const int32_t* prefix_pages;                // [NG]
  void* out;                                  // [B, HQ, 128] in q's type
  float* partial_out;                         // optional [B, HQ, 129]
  int32_t* status;
  // workspace
  int32_t* hdr;                               // [0] segments, [1] cost of all units of one kv-head, [2] a wait of this call gave up
  SpSegment* seg;                             // [max_seg]: the sequences' own first, then the shared ones
  int32_t* cum;                               // [max_seg + 1] cost of the segments before
  int32_t* start;                             // [n_ctas, 2] first segment and kv-head
  int32_t* seq_seg;                           // [B, 2] first shared segment of the sequence's group (-1: none), its first row
  uint8_t* qp;                                // [pieces, HKV, B * G, 128] q as e4m3 pieces
  float* q_scale;                             // [HKV, B * G] what a dot product with them is multiplied with (log2 units)
  float2* part_ml;                            // [part_rows] maximum (log2 units) and sum
  float* part_o;                              // [part_rows, 128]
  int B, NG, HQ, HKV, G;
  int n_pages, cols, bt_stride;
  int n_ctas;
  int pieces;
  int q_dtype, v_dtype, fp8;
  float scale_log2;
};

// Segments of shared pages: every group begins one, and one more for every 128 rows (at most B groups).
__host__ __device__ inline int64_t sp_max_shared(int64_t B, int64_t G) { return B + B * G / kSpRows + 1; }

// Rows of partials: a run of CTA c in unit (segment, kv-head) writes at
//   shared: row0 * HKV + head * rows + c * 128        (rows before it in the unit order, plus 128 for each CTA before)
//   own:    shared_rows + row0 * HKV + head * G + c * G
// Going on to the next unit or the next CTA moves at least `rows` rows on, so no two runs share a row.
__host__ __device__ inline int64_t sp_shared_rows(int64_t B, int64_t HQ, int64_t n_ctas) { return B * HQ + n_ctas * kSpRows; }
__host__ __device__ inline int64_t sp_part_rows(int64_t B, int64_t HQ, int64_t HKV, int64_t n_ctas) {
  return sp_shared_rows(B, HQ, n_ctas) + B * HQ + n_ctas * (HQ / HKV);
}
__device__ __forceinline__ int64_t sp_part_row(const SpParams& p, const SpSegment& s, int head, int cta) {
  const int64_t at = static_cast<int64_t>(s.row0) * p.HKV + static_cast<int64_t>(head) * s.rows;
  return s.own ? sp_shared_rows(p.B, p.HQ, p.n_ctas) + at + static_cast<int64_t>(cta) * p.G : at + static_cast<int64_t>(cta) * kSpRows;
}

// A unit costs its tiles and kSpUnitCost for being begun (q, the first loads' latency, the partial).  Its tile t stands at
// unit_start + kSpUnitCost + t on the line of all costs, 0 .. W; CTA c has [c * W / n, (c + 1) * W / n).
constexpr int kSpUnitCost = 1;
__host__ __device__ __forceinline__ int sp_cost(int tiles) { return tiles > 0 ? tiles + kSpUnitCost : 0; }
// CTAs that take part: one position each at least, so that every CTA between a unit's first and last has a run of it.
__device__ __forceinline__ int sp_ctas(int64_t W, int n_ctas) { return W < 1 ? 1 : W < n_ctas ? static_cast<int>(W) : n_ctas; }
__device__ __forceinline__ int64_t sp_first(int64_t c, int64_t W, int n) { return c * W / n; }
__device__ __forceinline__ int sp_owner(int64_t x, int64_t W, int n) { return static_cast<int>(((x + 1) * n - 1) / W); }

// ffa_shared_prefix_attend.cu: the attention over the runs that the plan in p.hdr, p.seg, ... lists.
int launch_sp_attend(const SpParams& p, cudaStream_t st);

}  // namespace ffa
