// Decode attention for batches that share a long prefix: q in pieces, attention over the runs
// (ffa_shared_prefix_attend.cu), merge (see ffa_shared_prefix.cuh for the split).
#include "ffa_numeric.h"
#include "ffa_shared_prefix.cuh"

namespace ffa {
namespace {

constexpr int kSplitThreads = 256;
constexpr int kMaxBatch = 4096;

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
  bool finite = fabsf(p.scale_log2) < INFINITY;
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
  // infinities and NaN in q or in the softmax scale make the whole row NaN; the scale stays above zero, so that the -inf of a
  // masked token times it is -inf (1e-30 times a dot product of pieces, 128 times 2^8 times base and residual of up to 57344
  // and so below 2^32, is nothing in a score)
  if ((lane & 7) == 0)
    p.q_scale[row_id] = finite ? fmaxf(fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23), 1e-30f) : NAN;
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

// 32 rows to a block.  Bound by latency (2048 rows of 128 are 0.5 MB), so the attention is set up meanwhile and already
// loads K and V: with that, q split in the plan's place, and a merge by four ways, 8 samples of 32K went from 72 to 47 us.
__global__ void __launch_bounds__(kSplitThreads) sp_split_kernel(const __grid_constant__ SpParams p) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) p.hdr[1] = 0;
  split_q(p, static_cast<int64_t>(blockIdx.x) * (kSplitThreads / 8) + threadIdx.x / 8);
}

// Blocks of a sequence and kv-head and a slice of the channels: 128 * G threads are ways x (G rows x groups of four
// channels).  The partials of a row - of the shared pages, then of its own, in the order of the line - are dealt out in
// turn to the ways, so that many loads are in flight together, and added up in a fixed order.  A row without a token gives
// zeros and a log-sum-exp of -inf.  Bound by latency: a chain of three loads and two exchanges, then some 20 partials a row.
//
// The blocks are given out as SMs fall free of the attention, as many to an SM as it can hold.  So few sequences are cut
// into slices, and a block asks for a share of shared memory that leaves no room for more of them than an even spread needs.
// Replayed as a graph: 10 sequences of one head each over 49K shared tokens 52.8 -> 20 us (their blocks had all gone to the
// SM that finished first), 8 samples of 20K 47.5 -> 40; over 28 batches of mixed shapes 34.3 -> 31.5 in geometric mean.
constexpr int kMergeWays = 4;
template <int SLICES>
__global__ void __launch_bounds__(1024) sp_merge_kernel(const __grid_constant__ SpParams p) {
  extern __shared__ float4 s_o[];             // [threads], then [ways][G] maximum and sum
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  constexpr int ways = kMergeWays * SLICES, channels = 32 / SLICES;
  const int slice = blockIdx.x % SLICES, pair = blockIdx.x / SLICES, b = pair / p.HKV, head = pair % p.HKV, per_way = channels * p.G;
  const int lane_row = threadIdx.x % per_way, way = threadIdx.x / per_way;
  const int c4 = slice * channels + lane_row / p.G, g = lane_row % p.G;
  const SpSequence me = p.sequences[b];
  const int W = p.hdr[0];
  const bool gave_up = p.hdr[1] != 0;
  const int n_used = sp_ctas(W, p.n_ctas);
  // the row's two lists of partials: the first one's place for this thread, and from one to the next
  int64_t at[2] = {0, 0}, o_at[2] = {0, 0};
  int n[2] = {0, 0};
  if (me.group_tiles > 0) {
    const int all = (b - me.group_first) * p.G + g, block = all / kSpRows, row = all % kSpRows;
    const int rows = min(kSpRows, me.group_rows - block * kSpRows);
    const int tile = sp_tile_cost(me.group_rows), x = me.group_at + (block * p.HKV + head) * sp_unit_cost(me.group_tiles, tile) + kSpBegin;
    const int c = sp_owner(x, W, n_used);
    n[0] = sp_owner(x + (me.group_tiles - 1) * tile, W, n_used) - c + 1;
    const int64_t first = sp_part_row(p, false, me.group_first * p.G + block * kSpRows, rows, head, c);
    at[0] = first + row;
    o_at[0] = 32 * first + c4 * rows + row;
  }
  if (me.tiles > 0) {
    const int tile = sp_tile_cost(p.G), x = me.at + head * sp_unit_cost(me.tiles, tile) + kSpBegin, c = sp_owner(x, W, n_used);
    n[1] = sp_owner(x + (me.tiles - 1) * tile, W, n_used) - c + 1;
    const int64_t first = sp_part_row(p, true, b * p.G, p.G, head, c);
    at[1] = first + g;
    o_at[1] = 32 * first + c4 * p.G + g;
  }
  const int total = n[0] + n[1];
  float m = -INFINITY, l = 0.f, o[4] = {};
  constexpr int U = 6;
#pragma unroll 1
  for (int k0 = way; k0 < total; k0 += U * ways) {
    float4 x[U];
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * ways;
      ml[u] = make_float2(-INFINITY, 0.f);
      x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < total) {
        const bool own = k >= n[0];
        const int64_t j = own ? k - n[0] : k, step = own ? p.G : kSpRows;
        ml[u] = p.part_ml[(own ? at[1] : at[0]) + j * step];
        x[u] = p.part_o[(own ? o_at[1] : o_at[0]) + j * step * 32];
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u].x);
    const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref);
    l *= keep;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = exp2f(ml[u].x - ref);
      l += ml[u].y * w;
      o[0] += x[u].x * w; o[1] += x[u].y * w; o[2] += x[u].z * w; o[3] += x[u].w * w;
    }
    m = top;
  }
  float2* const s_ml = reinterpret_cast<float2*>(s_o + blockDim.x);
  s_o[threadIdx.x] = make_float4(o[0], o[1], o[2], o[3]);
  if (lane_row < p.G) s_ml[way * p.G + g] = make_float2(m, l);
  __syncthreads();
  if (way != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < ways; ++w) top = fmaxf(top, s_ml[w * p.G + g].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, y[4] = {};
#pragma unroll
  for (int w = 0; w < ways; ++w) {
    const float2 ml = s_ml[w * p.G + g];
    const float f = exp2f(ml.x - ref);
    const float4 x = s_o[w * per_way + lane_row];
    sum += ml.y * f;
    y[0] += x.x * f; y[1] += x.y * f; y[2] += x.z * f; y[3] += x.w * f;
  }
  const float inv = gave_up ? NAN : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] *= inv;
  const int64_t i = static_cast<int64_t>(b) * p.HQ + head * p.G + g;
  if (p.q_dtype == FFA_F32) {
    reinterpret_cast<float4*>(p.out)[i * 32 + c4] = make_float4(y[0], y[1], y[2], y[3]);
  } else {
    uint2 w;
    if (p.q_dtype == FFA_BF16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
      w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      w = make_uint2(pack_h2(y[0], y[1]), pack_h2(y[2], y[3]));
    }
    reinterpret_cast<uint2*>(p.out)[i * 32 + c4] = w;
  }
  if (p.partial_out) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p.partial_out[i * (kHeadDim + 1) + 4 * c4 + j] = y[j];
    if (c4 == 0) p.partial_out[i * (kHeadDim + 1) + kHeadDim] = gave_up ? NAN : sum == 0.f ? -INFINITY : top + log2f(sum);
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

constexpr size_t kMergeSmem = 228 * 1024;     // of an SM
int allow_merge_smem() {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !configured[dev]) {
    for (void (*f)(SpParams) : {sp_merge_kernel<1>, sp_merge_kernel<2>, sp_merge_kernel<4>}) {
      const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMergeSmem - 1024);
      if (e != cudaSuccess) return note_cuda_error(e, "cudaFuncSetAttribute(sp_merge)");
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return FFA_OK;
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

struct Layout {
  size_t sequences, groups, qp, q_scale, ml, o, total;
};
Layout layout(int64_t B, int64_t HQ, int64_t HKV) {
  const int64_t rows = sp_part_rows(B, HQ, HKV);
  Layout a{};
  a.sequences = 512;                                                 // header and status word before it
  a.groups = a.sequences + align256(B * sizeof(SpSequence));
  a.qp = a.groups + align256(B * sizeof(SpGroup));                   // at most B groups
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
  if (a->B > kMaxBatch || static_cast<int64_t>(a->n_pages) * kPage > INT32_MAX ||
      sp_longest_line(a->B, a->n_groups, a->HKV, a->HQ / a->HKV, a->cols) > INT32_MAX)
    return FFA_E_LIMIT;
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
  p.sequences = reinterpret_cast<SpSequence*>(ws + w.sequences);
  p.groups = reinterpret_cast<SpGroup*>(ws + w.groups);
  p.qp = reinterpret_cast<uint8_t*>(ws + w.qp);
  p.q_scale = reinterpret_cast<float*>(ws + w.q_scale);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part_o = reinterpret_cast<float4*>(ws + w.o);
  p.B = a->B; p.NG = a->n_groups; p.HQ = a->HQ; p.HKV = a->HKV; p.G = a->HQ / a->HKV;
  p.n_pages = a->n_pages; p.cols = a->cols; p.bt_stride = a->bt_stride;
  p.n_ctas = sm_count() < kSpMaxCtas ? sm_count() : kSpMaxCtas;
  p.pieces = a->q_dtype == FFA_BF16 ? 2 : 3;
  p.q_dtype = a->q_dtype; p.v_dtype = a->v_dtype; p.fp8 = a->fp8_format;
  p.scale_log2 = a->sm_scale * kLog2e;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t rows = static_cast<int64_t>(p.B) * p.HQ;
  sp_split_kernel<<<static_cast<unsigned>((rows * 8 + kSplitThreads - 1) / kSplitThreads), kSplitThreads, 0, st>>>(p);
  int rc = last_launch("ffa_decode_shared_prefix (q)");
  if (rc) return rc;
  if ((rc = launch_sp_attend(p, st))) return rc;
  // the merge is launched while the attention still runs: its blocks start on SMs whose CTA has ended (both do not fit on one)
  // and wait there for the end of the others
  const int64_t pairs = static_cast<int64_t>(p.B) * p.HKV;
  const int slices = pairs * 4 <= p.n_ctas ? 4 : pairs * 2 <= p.n_ctas ? 2 : 1;
  const int64_t per_sm = (pairs * slices + p.n_ctas - 1) / p.n_ctas;
  const size_t need = kMergeWays * p.G * (32 * sizeof(float4) + slices * sizeof(float2));
  const size_t share = per_sm > 4 ? 0 : kMergeSmem / per_sm - 1024;           // 1 KiB of each block is the system's
  void (*const merge)(SpParams) = slices == 4 ? sp_merge_kernel<4> : slices == 2 ? sp_merge_kernel<2> : sp_merge_kernel<1>;
  if ((rc = allow_merge_smem())) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * slices));
  cfg.blockDim = dim3(kMergeWays * 32 * p.G);
  cfg.dynamicSmemBytes = share > need ? share : need;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, merge, p);
  return e == cudaSuccess ? FFA_OK : note_cuda_error(e, "ffa_decode_shared_prefix (merge)");
}
