// Decode attention for batches that share a long prefix: plan, attention over the runs, merge (see
// ffa_shared_prefix.cuh for the split).
#include "ffa_shared_prefix.cuh"

namespace ffa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxBatch = 16384;

__device__ __forceinline__ int block_exclusive(int x, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int w = s_warp[lane];
    int winc = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, winc, d);
      if (lane >= d) winc += y;
    }
    s_warp[lane] = winc - w;
    if (lane == 31) s_warp[32] = winc;
  }
  __syncthreads();
  total = s_warp[32];
  return s_warp[warp] + inc - x;
}

// The work list, by one block.  Lengths and group bounds come from the caller's device memory and are clamped to the
// batch and the table, so that whatever they hold no access leaves the tensors.
__global__ void __launch_bounds__(kPlanThreads) sp_plan_kernel(const __grid_constant__ SpParams p) {
  __shared__ int s_warp[33];
  const int tid = threadIdx.x;
  auto start_of = [&](int g) { return min(max(p.group_start[g], 0), p.B); };
  auto pages_of = [&](int g) { return min(max(p.prefix_pages[g], 0), p.cols); };
  const int max_shared = static_cast<int>(sp_max_shared(p.B, p.G));
  int n_shared = 0;
  for (int g0 = 0; g0 < p.NG; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int first = 0, rows = 0, pages = 0;
    if (g < p.NG) {
      first = start_of(g);
      rows = max(start_of(g + 1) - first, 0) * p.G;
      pages = pages_of(g);
      if (pages == 0) rows = 0;
    }
    int n = (rows + kSpRows - 1) / kSpRows, sum;
    const int at = n_shared + block_exclusive(n, s_warp, sum);
    if (at + n > max_shared) n = 0;           // bounds that do not ascend: more segments than the batch can have
    for (int i = 0; i < n; ++i) {
      SpSegment s{};
      s.table_row = first;
      s.row0 = first * p.G + i * kSpRows;
      s.rows = min(kSpRows, rows - i * kSpRows);
      s.tiles = (pages * kPage + kSpTile - 1) / kSpTile;
      s.end = pages * kPage;
      p.seg[at + i] = s;
    }
    // the sequences of this group learn where its segments begin
    if (g < p.NG)
      for (int b = first; b < start_of(g + 1); ++b) { p.seq_seg[2 * b] = n ? at : -1; p.seq_seg[2 * b + 1] = first * p.G; }
    n_shared += sum;
  }
  n_shared = min(n_shared, max_shared);
  __syncthreads();
  for (int b = tid; b < p.B; b += kPlanThreads) {
    const int len = min(max(p.seq_lens[b], 0), p.cols * kPage);
    int lo = 0, hi = p.NG;                    // last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (start_of(mid) <= b) lo = mid + 1; else hi = mid;
    }
    const int g = lo - 1;
    const int pages = g >= 0 && b < start_of(g + 1) ? pages_of(g) : 0;
    if (g < 0 || b >= start_of(g + 1)) p.seq_seg[2 * b] = -1;
    SpSegment s{};
    s.table_row = b;
    s.row0 = b * p.G;
    s.rows = p.G;
    s.page0 = pages;
    s.tiles = (max(len - pages * kPage, 0) + kSpTile - 1) / kSpTile;
    s.end = len;
    s.own = 1;
    p.seg[n_shared + b] = s;
  }
  const int n_seg = n_shared + p.B;
  __syncthreads();
  int total = 0;
  for (int s0 = 0; s0 < n_seg; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int sum;
    const int before = block_exclusive(s < n_seg ? p.seg[s].tiles : 0, s_warp, sum);
    if (s < n_seg) p.cum[s] = total + before;
    total += sum;
  }
  if (tid == 0) {
    p.cum[n_seg] = total;
    p.hdr[0] = n_seg;
    p.hdr[1] = n_shared;
    p.hdr[2] = total;
    p.hdr[3] = 0;
  }
  __syncthreads();
  const int64_t W = static_cast<int64_t>(total) * p.HKV;
  const int n_used = sp_ctas(W, p.n_ctas);
  for (int c = tid; c < n_used; c += kPlanThreads) {
    const int64_t x = sp_first(c, W, n_used);
    int lo = 0, hi = n_seg;                   // last segment whose first tile is at or before x
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<int64_t>(p.cum[mid]) * p.HKV <= x) lo = mid; else hi = mid;
    }
    const int64_t in = x - static_cast<int64_t>(p.cum[lo]) * p.HKV;
    const int tiles = max(p.seg[lo].tiles, 1);
    p.start[4 * c] = lo;
    p.start[4 * c + 1] = static_cast<int>(in / tiles);
    p.start[4 * c + 2] = static_cast<int>(in % tiles);
  }
}

// One warp per query row: its partials of the shared pages, then of its own, in the order of the tiles.  A row
// without a token gives zeros and a log-sum-exp of -inf.
__global__ void __launch_bounds__(256) sp_merge_kernel(const __grid_constant__ SpParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= static_cast<int64_t>(p.B) * p.HQ) return;
  const int b = static_cast<int>(i / p.HQ), hq = static_cast<int>(i % p.HQ), head = hq / p.G, g = hq % p.G;
  const int64_t W = static_cast<int64_t>(p.hdr[2]) * p.HKV;
  const int n_used = sp_ctas(W, p.n_ctas);
  float m = -INFINITY, l = 0.f, o[4] = {};
  for (int own = 0; own < 2; ++own) {
    int si = p.hdr[1] + b, row = g;
    if (!own) {
      si = p.seq_seg[2 * b];
      if (si < 0) continue;
      row = b * p.G + g - p.seq_seg[2 * b + 1];
      si += row / kSpRows;
      row %= kSpRows;
    }
    const SpSegment s = p.seg[si];
    if (s.tiles == 0) continue;
    const int64_t x = static_cast<int64_t>(p.cum[si]) * p.HKV + static_cast<int64_t>(head) * s.tiles;
    const int c1 = sp_owner(x + s.tiles - 1, W, n_used);
    for (int c = sp_owner(x, W, n_used); c <= c1; ++c) {
      const int64_t part = sp_part_row(p, s, head, c) + row;
      const float2 ml = p.part_ml[part];
      const float4 po = *reinterpret_cast<const float4*>(p.part_o + part * kHeadDim + lane * 4);
      const float top = fmaxf(m, ml.x);
      if (top == -INFINITY) continue;
      const float a = exp2f(m - top), w = exp2f(ml.x - top);
      l = l * a + ml.y * w;
      o[0] = o[0] * a + po.x * w; o[1] = o[1] * a + po.y * w; o[2] = o[2] * a + po.z * w; o[3] = o[3] * a + po.w * w;
      m = top;
    }
  }
  const float inv = p.hdr[3] ? NAN : l == 0.f ? 0.f : 1.f / l;      // NaN: a wait of this call gave up
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] *= inv;
#pragma unroll
  for (int j = 0; j < 4; ++j) store_from_float(p.out, i * kHeadDim + lane * 4 + j, p.q_dtype, o[j]);
  if (p.partial_out) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p.partial_out[i * (kHeadDim + 1) + lane * 4 + j] = o[j];
    if (lane == 0) p.partial_out[i * (kHeadDim + 1) + kHeadDim] = l == 0.f ? -INFINITY : m + log2f(l);
  }
}

int sm_count() {
  static thread_local int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (n[dev] == 0) {
    int x = 0;
    n[dev] = cudaDeviceGetAttribute(&x, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && x > 0 ? x : 148;
  }
  return n[dev];
}

constexpr int kMaxCtas = 192;                 // the workspace is sized for this many, whatever the GPU

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

struct Layout {
  size_t seg, cum, start, seq_seg, ml, o, total;
};
Layout layout(int64_t B, int64_t HQ, int64_t HKV) {
  const int64_t n_seg = sp_max_shared(B, HQ / HKV) + B;
  const int64_t rows = sp_part_rows(B, HQ, HKV, kMaxCtas);
  Layout a{};
  a.seg = 512;                                                       // header and status word before it
  a.cum = a.seg + align256(n_seg * sizeof(SpSegment));
  a.start = a.cum + align256((n_seg + 1) * 4);
  a.seq_seg = a.start + align256(kMaxCtas * 16);
  a.ml = a.seq_seg + align256(B * 8);
  a.o = a.ml + align256(rows * 8);
  a.total = a.o + align256(rows * kHeadDim * 4);
  return a;
}

int last_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FFA_OK : note_cuda_error(e, what);
}

}  // namespace
}  // namespace ffa

using namespace ffa;

extern "C" size_t ffa_shared_prefix_workspace_bytes(int32_t B, int32_t HQ, int32_t HKV) {
  if (B <= 0 || B > kMaxBatch || HKV <= 0 || HQ < HKV || HQ % HKV) return 0;
  return layout(B, HQ, HKV).total;
}

extern "C" int ffa_decode_shared_prefix(const FfaSharedPrefixArgs* a, ffa_stream_t stream) {
  if (!a || !a->q || !a->k_base || !a->v || !a->block_table || !a->seq_lens || !a->group_start || !a->prefix_pages || !a->out ||
      !a->workspace)
    return FFA_E_NULL;
  if (a->use_residual && !a->k_residual) return FFA_E_NULL;
  if (a->B <= 0 || a->HKV <= 0 || a->HQ < a->HKV || a->HQ % a->HKV || a->HQ / a->HKV > 8 || a->head_dim != kHeadDim ||
      a->n_groups <= 0 || a->n_groups > a->B || a->n_pages <= 0 || a->cols <= 0 || a->bt_stride < a->cols ||
      a->cols > INT32_MAX / kPage - 2)
    return FFA_E_SHAPE;
  if (a->B > kMaxBatch || static_cast<int64_t>(a->n_pages) * kPage > INT32_MAX) return FFA_E_LIMIT;
  if ((a->q_dtype != FFA_F16 && a->q_dtype != FFA_BF16 && a->q_dtype != FFA_F32) || (a->v_dtype != FFA_F16 && a->v_dtype != FFA_BF16) ||
      (a->fp8_format != FFA_E5M2 && a->fp8_format != FFA_E4M3))
    return FFA_E_DTYPE;
  const Layout w = layout(a->B, a->HQ, a->HKV);
  if (a->workspace_bytes < w.total) return FFA_E_WORKSPACE;
  for (const void* x : {a->q, a->k_base, a->use_residual ? a->k_residual : nullptr, a->v, static_cast<const void*>(a->out),
                        static_cast<const void*>(a->workspace)})
    if (reinterpret_cast<uintptr_t>(x) & 15u) return FFA_E_ALIGN;
  char* ws = static_cast<char*>(a->workspace);
  SpParams p{};
  p.q = a->q;
  p.k = static_cast<const uint8_t*>(a->k_base);
  p.r = a->use_residual ? static_cast<const uint8_t*>(a->k_residual) : nullptr;
  p.v = static_cast<const uint8_t*>(a->v);
  p.bt = a->block_table; p.seq_lens = a->seq_lens; p.group_start = a->group_start; p.prefix_pages = a->prefix_pages;
  p.out = a->out; p.partial_out = a->partial_out;
  p.status = reinterpret_cast<int32_t*>(ws + 256);
  p.hdr = reinterpret_cast<int32_t*>(ws);
  p.seg = reinterpret_cast<SpSegment*>(ws + w.seg);
  p.cum = reinterpret_cast<int32_t*>(ws + w.cum);
  p.start = reinterpret_cast<int32_t*>(ws + w.start);
  p.seq_seg = reinterpret_cast<int32_t*>(ws + w.seq_seg);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  p.B = a->B; p.NG = a->n_groups; p.HQ = a->HQ; p.HKV = a->HKV; p.G = a->HQ / a->HKV;
  p.n_pages = a->n_pages; p.cols = a->cols; p.bt_stride = a->bt_stride;
  p.n_ctas = sm_count() < kMaxCtas ? sm_count() : kMaxCtas;
  p.q_dtype = a->q_dtype; p.v_dtype = a->v_dtype; p.fp8 = a->fp8_format;
  p.scale_log2 = a->sm_scale * kLog2e;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  sp_plan_kernel<<<1, kPlanThreads, 0, st>>>(p);
  int rc = last_launch("ffa_decode_shared_prefix (plan)");
  if (rc) return rc;
  if ((rc = launch_sp_attend(p, st))) return rc;
  const int64_t rows = static_cast<int64_t>(p.B) * p.HQ;
  sp_merge_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(p);
  return last_launch("ffa_decode_shared_prefix (merge)");
}
