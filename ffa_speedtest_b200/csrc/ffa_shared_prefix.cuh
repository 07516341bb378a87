// Decode attention over a paged fp8 + fp8-residual cache for batches whose sequences share leading pages: work split,
// partial results and merge.
//
//   o_b = softmax(scale * q_b K_b^T) V_b over the len_b tokens of sequence b,  K = base + residual
//
// Items of work: one per sequence (its own pages) and one per group of sequences with a shared prefix (the group's
// pages, all query rows of the group; a row = one query head of one sequence).  An item is cut into units: a kv-head,
// and for groups a block of 128 rows.  A unit has ceil(tokens / 128) tiles.  All units stand in a row on a line of costs,
// which is cut into equal ranges, one per CTA.  A CTA's part of a unit is a run; every run leaves partials (maximum, sum,
// output) for its rows, and the merge adds a row's partials up in the order of the line.  Group sizes, prefix lengths and
// sequence lengths are read on the device, so a captured call follows them; every CTA works out the line for itself.
#pragma once

#include "ffa_common.cuh"

namespace ffa {

constexpr int kSpTile = 128;                  // tokens of a tile: two pages
constexpr int kSpRows = 128;                  // query rows of a unit, at most
constexpr int kSpMaxCtas = 148;

// Costs, in quarters of a tile of few rows: beginning a unit (q, the first loads' latency, its partials), a tile of up to 64
// query rows, a tile of more (the exponentials of 128 rows, and with bfloat16 V twice the MMAs of P V; 1.9 us where a tile of
// few rows takes 1.4).  Over 28 batches of mixed shapes 4, 5, 6 and 8 for the first gave 34.6, 34.3, 34.1 and 34.4 us in
// geometric mean.  4, 5, 6 and 7 for the last: 64 samples of 128K 294, 267, 286 and 307 us, 32 samples of 16K in fp16 45.9,
// 44.0, 43.4 and 46.4, the 28 batches the same within 0.7 %.
constexpr int kSpBegin = 6, kSpNarrowTile = 4, kSpWideTile = 5;
// a tile of an item with so many query rows to a kv-head
__host__ __device__ inline int sp_tile_cost(int rows) { return rows > 64 ? kSpWideTile : kSpNarrowTile; }

// where the merge finds the partials of a sequence's rows: the places of its item and of its group's on the line
struct SpSequence {
  int32_t at, tiles;
  int32_t group_at, group_tiles;              // 0 tiles: no shared part
  int32_t group_first, group_rows;            // first sequence of the group, rows of a kv-head
  int32_t pad[2];
};
struct SpGroup {
  int32_t at, tiles, first, rows;
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
  int32_t* hdr;                               // [0] length of the line, [1] a wait of this call gave up
  SpSequence* sequences;                      // [B]
  SpGroup* groups;                            // [NG]
  uint8_t* qp;                                // [pieces, HKV, B * G, 128] q as e4m3 pieces
  float* q_scale;                             // [HKV, B * G] what a dot product with them is multiplied with (log2 units)
  float2* part_ml;                            // [part_rows] maximum (log2 units) and sum
  float4* part_o;                             // [part_rows, 32]
  int B, NG, HQ, HKV, G;
  int n_pages, cols, bt_stride;
  int n_ctas;
  int pieces;
  int q_dtype, v_dtype, fp8;
  float scale_log2;
};

// Rows of partials.  A run of CTA c in the unit of these rows and this head begins at
//   shared: row0 * HKV + head * rows + c * 128        (rows before it in the order of the line, plus 128 for each CTA before)
//   own:    shared_rows + row0 * HKV + head * G + c * G
// Going on to the next unit or the next CTA moves at least `rows` rows on, so no two runs share a row.  With `at` the run's
// first row, row j's partial is part_ml[at + j], and its channels 4 * c .. 4 * c + 3 are part_o[32 * at + c * rows + j], so
// that the threads that hold a row each write side by side.
__host__ __device__ inline int64_t sp_shared_rows(int64_t B, int64_t HQ) { return B * HQ + static_cast<int64_t>(kSpMaxCtas) * kSpRows; }
__host__ __device__ inline int64_t sp_part_rows(int64_t B, int64_t HQ, int64_t HKV) {
  return sp_shared_rows(B, HQ) + B * HQ + kSpMaxCtas * (HQ / HKV);
}
__device__ __forceinline__ int64_t sp_part_row(const SpParams& p, bool own, int row0, int rows, int head, int cta) {
  const int64_t at = static_cast<int64_t>(row0) * p.HKV + static_cast<int64_t>(head) * rows;
  return own ? sp_shared_rows(p.B, p.HQ) + at + static_cast<int64_t>(cta) * p.G : at + static_cast<int64_t>(cta) * kSpRows;
}

// Cost of a unit of so many tiles.  Tile t of a unit that begins at U stands at U + kSpBegin + t * tile_cost.
__device__ __forceinline__ int sp_unit_cost(int tiles, int tile_cost) { return tiles > 0 ? kSpBegin + tiles * tile_cost : 0; }
// The line is at most this long (the host refuses what could give 2^31 or more): every sequence and every group a unit of few
// rows, and what groups of more rows cost beyond that, which is most for a row if a group has one row more than a block.
__host__ __device__ inline int64_t sp_longest_line(int64_t B, int64_t NG, int64_t HKV, int64_t G, int64_t cols) {
  const int64_t tiles = (cols + 1) / 2;
  return HKV * ((B + NG) * (kSpBegin + tiles * kSpNarrowTile) +
                B * G * (kSpBegin + tiles * (2 * kSpWideTile - kSpNarrowTile)) / kSpRows);
}
// CTAs that take part on a line of length W: each gets 8 on average, 7 at least after rounding, more than a tile, so that
// every CTA between the first and the last of a unit has a tile of it.  CTA c begins at c * (W / n).
__device__ __forceinline__ int sp_ctas(int W, int n_ctas) { return max(1, min(n_ctas, W / 8)); }
__device__ __forceinline__ int sp_first(int c, int W, int n) {
  return c >= n ? W : static_cast<int>(static_cast<float>(c) * (static_cast<float>(W) * __frcp_rn(static_cast<float>(n))));
}
__device__ __forceinline__ int sp_owner(int x, int W, int n) {
  int c = min(n - 1, static_cast<int>(static_cast<float>(x) * (static_cast<float>(n) * __frcp_rn(static_cast<float>(W)))));
  while (c > 0 && sp_first(c, W, n) > x) --c;
  while (c < n - 1 && sp_first(c + 1, W, n) <= x) ++c;
  return c;
}

// Lengths and group bounds come from the caller's device memory and are clamped to the batch and the table, so that
// whatever they hold no access leaves the tensors.
// Group bounds and prefixes, clamped: in the CTA's shared memory as far as they fit there.  Bounds that do not ascend make
// no groups at all (n = 0), so that a row never belongs to two.
constexpr int kSpGroupsNear = 256;
struct SpBounds {
  const SpParams& p;
  int n;                                      // groups
  const int32_t* near_start;                  // [min(NG, kSpGroupsNear) + 1]
  const int32_t* near_pages;
  __device__ __forceinline__ int start(int g) const {
    return g <= kSpGroupsNear ? near_start[g] : min(max(p.group_start[g], 0), p.B);
  }
  __device__ __forceinline__ int pages(int g) const { return g < kSpGroupsNear ? near_pages[g] : min(max(p.prefix_pages[g], 0), p.cols); }
  // the group of sequence b, or -1
  __device__ __forceinline__ int group_of(int b) const {
    int lo = 0, hi = n;                       // last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (start(mid) <= b) lo = mid + 1; else hi = mid;
    }
    return lo > 0 && b < start(lo) ? lo - 1 : -1;
  }
};

// Item i of the line: sequences 0 .. B-1 (len: seq_lens[i]), then groups.
struct SpItem {
  int first, rows;                            // first sequence (its table row), rows of a kv-head, all blocks
  int page0, end, tiles;                      // first column of the block table, token that ends it
  int units;
  int group;                                  // of a sequence: its group
};
__device__ __forceinline__ SpItem sp_item(const SpParams& p, const SpBounds& bounds, int i, int len) {
  SpItem x;
  if (i < p.B) {
    x.group = bounds.group_of(i);
    x.first = i;
    x.rows = p.G;
    x.page0 = x.group >= 0 ? bounds.pages(x.group) : 0;
    x.end = min(max(len, 0), p.cols * kPage);
    x.tiles = (max(x.end - x.page0 * kPage, 0) + kSpTile - 1) / kSpTile;
    x.units = p.HKV;
  } else {
    const int g = i - p.B;
    x.group = -1;
    x.first = bounds.start(g);
    x.rows = (bounds.start(g + 1) - x.first) * p.G;
    x.page0 = 0;
    x.end = x.rows ? bounds.pages(g) * kPage : 0;
    x.tiles = (x.end + kSpTile - 1) / kSpTile;
    x.units = (x.rows + kSpRows - 1) / kSpRows * p.HKV;
  }
  return x;
}

// ffa_shared_prefix_attend.cu: the attention over the runs; it also leaves what the merge has to know of the line.
int launch_sp_attend(const SpParams& p, cudaStream_t st);

}  // namespace ffa
