// Decode attention for batches that share a long prefix: plan, attention over the runs, merge (see
// ffa_shared_prefix.cuh for the split).
#include "ffa_numeric.h"
#include "ffa_shared_prefix.cuh"

namespace ffa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxBatch = 4096;

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

// Dynamic shared memory of the plan: cost of every segment, and of every group its first sequence, first segment
// and pages.
__host__ __device__ inline int plan_smem_ints(int B, int G, int NG) {
  return static_cast<int>(B + sp_max_shared(B, G)) + 3 * (NG + 1);
}

// The work list, by one block.  Lengths and group bounds come from the caller's device memory and are clamped to the
// batch and the table, so that whatever they hold no access leaves the tensors.
__device__ void plan(const SpParams& p, int* smem) {
  __shared__ int s_warp[33];
  const int tid = threadIdx.x;
  const int max_shared = static_cast<int>(sp_max_shared(p.B, p.G));
  int* const s_cost = smem;
  int* const s_start = smem + p.B + max_shared;
  int* const s_first = s_start + p.NG + 1;
  int* const s_pages = s_first + p.NG + 1;
  for (int g = tid; g <= p.NG; g += kPlanThreads) {
    s_start[g] = min(max(p.group_start[g], 0), p.B);
    if (g < p.NG) s_pages[g] = min(max(p.prefix_pages[g], 0), p.cols);
  }
  __syncthreads();
  int n_shared = 0;
  for (int g0 = 0; g0 < p.NG; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int first = 0, rows = 0, pages = 0;
    if (g < p.NG) {
      first = s_start[g];
      pages = s_pages[g];
      rows = pages ? max(s_start[g + 1] - first, 0) * p.G : 0;
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
      p.seg[p.B + at + i] = s;
      s_cost[p.B + at + i] = sp_cost(s.tiles);
    }
    if (g < p.NG) s_first[g] = n ? p.B + at : -1;
    n_shared += sum;
  }
  n_shared = min(n_shared, max_shared);
  __syncthreads();
  for (int b = tid; b < p.B; b += kPlanThreads) {
    const int len = min(max(p.seq_lens[b], 0), p.cols * kPage);
    int lo = 0, hi = p.NG;                    // last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (s_start[mid] <= b) lo = mid + 1; else hi = mid;
    }
    const int g = lo - 1;
    const bool in = g >= 0 && b < s_start[g + 1];
    const int pages = in ? s_pages[g] : 0;
    p.seq_seg[2 * b] = in ? s_first[g] : -1;
    p.seq_seg[2 * b + 1] = in ? s_start[g] * p.G : 0;
    SpSegment s{};
    s.table_row = b;
    s.row0 = b * p.G;
    s.rows = p.G;
    s.page0 = pages;
    s.tiles = (max(len - pages * kPage, 0) + kSpTile - 1) / kSpTile;
    s.end = len;
    s.own = 1;
    p.seg[b] = s;
    s_cost[b] = sp_cost(s.tiles);
  }
  const int n_seg = p.B + n_shared;
  __syncthreads();
  int total = 0;
  for (int s0 = 0; s0 < n_seg; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int sum;
    const int before = block_exclusive(s < n_seg ? s_cost[s] : 0, s_warp, sum);
    if (s < n_seg) p.cum[s] = s_cost[s] = total + before;
    total += sum;
  }
  if (tid == 0) {
    p.cum[n_seg] = total;
    p.hdr[0] = n_seg;
    p.hdr[1] = total;
    p.hdr[2] = 0;
  }
  __syncthreads();
  const int64_t W = static_cast<int64_t>(total) * p.HKV;
  const int n_used = sp_ctas(W, p.n_ctas);
  for (int c = tid; c < n_used; c += kPlanThreads) {
    const int64_t x = sp_first(c, W, n_used);
    int lo = 0, hi = n_seg;                   // last segment that starts at or before x
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<int64_t>(s_cost[mid]) * p.HKV <= x) lo = mid; else hi = mid;
    }
    const int cost = (lo + 1 < n_seg ? s_cost[lo + 1] : total) - s_cost[lo];
    p.start[2 * c] = lo;
    p.start[2 * c + 1] = static_cast<int>((x - static_cast<int64_t>(s_cost[lo]) * p.HKV) / max(cost, 1));
  }
}

// q as a sum of e4m3 pieces, exactly: 2^up brings the largest |q| of a row into [128, 256), a piece holds four
// significant bits and the rest goes on to the next: two pieces for the eight of bf16, three for the eleven of fp16 (q
// in fp32 is rounded to fp16, as elsewhere in this library).  What is left of a channel 2^10 below the largest is at
// most 2^-10, that is 2^-17 of the largest.  Eight lanes to a row, 16 channels to a lane.
__device__ void split_q(const SpParams& p, int64_t row_id) {
  const int lane = threadIdx.x & 31, c0 = (lane & 7) * 16;
  const int64_t rows = static_cast<int64_t>(p.B) * p.G;             // of one kv-head
  const bool live = row_id < rows * p.HKV;
  const int head = live ? static_cast<int>(row_id / rows) : 0, row = live ? static_cast<int>(row_id % rows) : 0;
  const int64_t qi = (static_cast<int64_t>(row / p.G) * p.HQ + head * p.G + row % p.G) * kHeadDim + c0;
  float x[16];
  if (p.q_dtype == FFA_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + qi + 4 * e);
      x[4 * e] = f.x; x[4 * e + 1] = f.y; x[4 * e + 2] = f.z; x[4 * e + 3] = f.w;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __half2float(__float2half_rn(x[e]));
  } else {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + qi);
    const uint4 a = src[0], b = src[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p.q_dtype == FFA_BF16) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        const float2 f = unpack_h2(w[e]);
        x[2 * e] = f.x; x[2 * e + 1] = f.y;
      }
    }
  }
  float top = 0.f;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < 16; ++e) { top = fmaxf(top, fabsf(x[e])); finite = finite && fabsf(x[e]) < INFINITY; }
#pragma unroll
  for (int d = 4; d; d >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    finite = __shfl_xor_sync(0xffffffffu, finite ? 1 : 0, d) && finite;
  }
  const int up = top > 0.f ? min(max(7 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100) : 0;
  // a negative softmax scale turns q around, so that the scale of a row is never negative
  const float mul = __uint_as_float(static_cast<uint32_t>(up + 127) << 23) * (p.scale_log2 < 0.f ? -1.f : 1.f);
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = finite ? x[e] * mul : 0.f;
  if (!live) return;
  if ((lane & 7) == 0)                        // infinities and NaN in q make the whole row NaN
    p.q_scale[row_id] = finite ? fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23) : NAN;
  for (int piece = 0; piece < p.pieces; ++piece) {
    uint32_t w[4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[8 * half + e];
      const uint2 z = num::narrow8<num::kE4M3>(y);
      w[2 * half] = z.x; w[2 * half + 1] = z.y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = num::fp8x2_to_f32x2<num::kE4M3>((e < 2 ? z.x : z.y) >> (16 * (e & 1)));
        x[8 * half + 2 * e] -= f.x;
        x[8 * half + 2 * e + 1] -= f.y;
      }
    }
    *reinterpret_cast<uint4*>(p.qp + (piece * rows * p.HKV + row_id) * kHeadDim + c0) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Block 0 plans, the others split q: 128 rows to a block.
__global__ void __launch_bounds__(kPlanThreads) sp_prepare_kernel(const __grid_constant__ SpParams p) {
  extern __shared__ int s_plan[];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (blockIdx.x == 0) plan(p, s_plan);
  else split_q(p, static_cast<int64_t>(blockIdx.x - 1) * (kPlanThreads / 8) + threadIdx.x / 8);
}

// One block per query row: its partials of the shared pages and of its own, in the order of the tiles, a fixed share of
// them to each warp, so that the loads of a row are in flight together.  A row without a token gives zeros and a
// log-sum-exp of -inf.
__global__ void __launch_bounds__(128) sp_merge_kernel(const __grid_constant__ SpParams p) {
  __shared__ float s_o[4][kHeadDim], s_m[4], s_l[4];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = blockIdx.x;
  const int b = static_cast<int>(i / p.HQ), hq = static_cast<int>(i % p.HQ), head = hq / p.G, g = hq % p.G;
  const int64_t W = static_cast<int64_t>(p.hdr[1]) * p.HKV;
  const int gave_up = p.hdr[2], n_used = sp_ctas(W, p.n_ctas);
  // the row's two lists of partials: first row, step from part to part, number
  int64_t at[2] = {0, 0};
  int n[2] = {0, 0};
  const int shared = p.seq_seg[2 * b], group_row = b * p.G + g - p.seq_seg[2 * b + 1];
#pragma unroll
  for (int own = 0; own < 2; ++own) {
    if (!own && shared < 0) continue;
    const int si = own ? b : shared + group_row / kSpRows, row = own ? g : group_row % kSpRows;
    const SpSegment s = p.seg[si];
    if (s.tiles == 0) continue;
    const int64_t x = static_cast<int64_t>(p.cum[si]) * p.HKV + static_cast<int64_t>(head) * sp_cost(s.tiles) + kSpUnitCost;
    const int c = sp_owner(x, W, n_used);
    at[own] = sp_part_row(p, s, head, c) + row;
    n[own] = sp_owner(x + s.tiles - 1, W, n_used) - c + 1;
  }
  auto part_of = [&](int k) { return k < n[0] ? at[0] + static_cast<int64_t>(k) * kSpRows : at[1] + static_cast<int64_t>(k - n[0]) * p.G; };
  const int total = n[0] + n[1];
  float m = -INFINITY, l = 0.f, o[4] = {};
  for (int k0 = warp * 8; k0 < total; k0 += 32) {
    float4 x[8];
    float2 ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
      if (k0 + u < total) {
        const int64_t part = part_of(k0 + u);
        ml[u] = p.part_ml[part];
        x[u] = *reinterpret_cast<const float4*>(p.part_o + part * kHeadDim + lane * 4);
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, ml[u].x);
    const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref);
    l *= keep;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= keep;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (k0 + u >= total) continue;
      const float w = exp2f(ml[u].x - ref);
      l += ml[u].y * w;
      o[0] += x[u].x * w; o[1] += x[u].y * w; o[2] += x[u].z * w; o[3] += x[u].w * w;
    }
    m = top;
  }
  *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = make_float4(o[0], o[1], o[2], o[3]);
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  const int c = threadIdx.x;
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, y = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(s_m[w] - ref);
    sum += s_l[w] * f;
    y += s_o[w][c] * f;
  }
  y = gave_up ? NAN : sum == 0.f ? 0.f : y / sum;
  store_from_float(p.out, i * kHeadDim + c, p.q_dtype, y);
  if (p.partial_out) {
    p.partial_out[i * (kHeadDim + 1) + c] = y;
    if (c == 0) p.partial_out[i * (kHeadDim + 1) + kHeadDim] = gave_up ? NAN : sum == 0.f ? -INFINITY : top + log2f(sum);
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
  size_t seg, cum, start, seq_seg, qp, q_scale, ml, o, total;
};
Layout layout(int64_t B, int64_t HQ, int64_t HKV) {
  const int64_t n_seg = sp_max_shared(B, HQ / HKV) + B;
  const int64_t rows = sp_part_rows(B, HQ, HKV, kMaxCtas);
  Layout a{};
  a.seg = 512;                                                       // header and status word before it
  a.cum = a.seg + align256(n_seg * sizeof(SpSegment));
  a.start = a.cum + align256((n_seg + 1) * 4);
  a.seq_seg = a.start + align256(kMaxCtas * 8);
  a.qp = a.seq_seg + align256(B * 8);
  a.q_scale = a.qp + align256(3 * B * HQ * kHeadDim);
  a.ml = a.q_scale + align256(B * HQ * 4);
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
  p.qp = reinterpret_cast<uint8_t*>(ws + w.qp);
  p.q_scale = reinterpret_cast<float*>(ws + w.q_scale);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part_o = reinterpret_cast<float*>(ws + w.o);
  p.B = a->B; p.NG = a->n_groups; p.HQ = a->HQ; p.HKV = a->HKV; p.G = a->HQ / a->HKV;
  p.n_pages = a->n_pages; p.cols = a->cols; p.bt_stride = a->bt_stride;
  p.n_ctas = sm_count() < kMaxCtas ? sm_count() : kMaxCtas;
  p.pieces = a->q_dtype == FFA_BF16 ? 2 : 3;
  p.q_dtype = a->q_dtype; p.v_dtype = a->v_dtype; p.fp8 = a->fp8_format;
  p.scale_log2 = a->sm_scale * kLog2e;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int smem = 4 * plan_smem_ints(p.B, p.G, p.NG);
  if (smem > 48 * 1024) {                     // the limit belongs to the kernel on this device: raise it to the most that can be asked for
    const cudaError_t e = cudaFuncSetAttribute(sp_prepare_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               4 * plan_smem_ints(kMaxBatch, 8, kMaxBatch));
    if (e != cudaSuccess) return note_cuda_error(e, "cudaFuncSetAttribute(sp_prepare)");
  }
  const int64_t rows = static_cast<int64_t>(p.B) * p.HQ;
  const unsigned split_blocks = static_cast<unsigned>((rows * 8 + kPlanThreads - 1) / kPlanThreads);
  sp_prepare_kernel<<<1 + split_blocks, kPlanThreads, smem, st>>>(p);
  int rc = last_launch("ffa_decode_shared_prefix (plan)");
  if (rc) return rc;
  if ((rc = launch_sp_attend(p, st))) return rc;
  // the merge's blocks are set up while the attention still runs; they wait for its end before they read
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sp_merge_kernel, p);
  return e == cudaSuccess ? FFA_OK : note_cuda_error(e, "ffa_decode_shared_prefix (merge)");
}
