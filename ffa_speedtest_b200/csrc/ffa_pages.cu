// Page bookkeeping of a paged K/V cache on the device: truncate, fork, extend (with copy on first write of a
// shared open page) and compact, plus the copy kernel that moves page contents.  No reference counterpart.
//
// State: block_table [max_seqs, bt_stride] page numbers (-1 = none), seq_lens [max_seqs], refcount [n_pages] (0 =
// free).  A sequence of n tokens holds ceil(n/64) pages.  Free pages are handed out lowest number first, so the
// outcome of a call depends on its arguments and the state alone, never on the order in which threads run.
// Every call checks its arguments on the device before it changes anything; a call that cannot be carried out
// changes nothing and sets a bit of `status`.
//
// Cost: the bookkeeping is a few KiB to a few hundred KiB in L2 and bound by latency; the page copies are bound by
// HBM (every byte read once and written once).  Measured as graphs: truncate, fork and extend for 4 samples of 1K tokens
// 13.7 us together, 3.4 a launch; for 64 samples of 32K and 8 layers (open pages copied: 87 MB read, 87 MB written) 44 us, 25
// of them the copy; compact of 2000 pages in 4 layers 196 us for 1.04 GB, 5.3 TB/s.
#include "ffa_common.cuh"

namespace ffa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxSeqs = 65536;               // one bit each in shared memory while a call looks for repeated numbers
constexpr int kCopyThreads = 256;
constexpr int kChunk = kCopyThreads * 16 * 4; // bytes a block of the copy kernel moves at a time: four 16-byte loads a thread

// scratch: header, then arrays of ints
enum { kHdrOk = 0, kHdrJobs = 1, kHdrLive = 2, kHdrArrive = 3, kHdrInts = 16 };

// Any int: a new length may be as large as the caller likes, and tokens + 63 would wrap to a page far in front of the row.
__device__ __forceinline__ int pages_of(int tokens) { return tokens / kPage + (tokens % kPage > 0); }

// Every kernel here is launched while the one before it in the stream may still run (programmatic dependent launch): it
// is set up meanwhile and waits for that one's end before it reads anything.
__device__ __forceinline__ void begin() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

struct Table {
  int n_pages, max_seqs, cols, stride;
  int32_t* block_table;
  int32_t* seq_lens;
  int32_t* refcount;
  int32_t* status;
  int32_t* scratch;
  __host__ __device__ int32_t* hdr() const { return scratch; }
  __host__ __device__ int32_t* free_list() const { return scratch + kHdrInts; }          // extend: [n_pages]
  __host__ __device__ int32_t* job_src() const { return free_list() + n_pages; }         // [max(n_pages, max_seqs)]
  __host__ __device__ int32_t* job_dst() const { return job_src() + job_cap(); }
  __host__ __device__ int32_t* job_rows() const { return job_dst() + job_cap(); }        // extend: tokens to copy
  __host__ __device__ int32_t* first_new() const { return job_rows() + job_cap(); }      // extend: [max_seqs]
  __host__ __device__ int job_cap() const { return n_pages > max_seqs ? n_pages : max_seqs; }
  __device__ int32_t* row(int s) const { return block_table + static_cast<int64_t>(s) * stride; }
};

size_t scratch_ints(int64_t n_pages, int64_t max_seqs) {
  const int64_t cap = n_pages > max_seqs ? n_pages : max_seqs;
  return static_cast<size_t>(kHdrInts + n_pages + 3 * cap + max_seqs);
}

// Exclusive scan over the block's threads; `total` gets the sum.  s_warp: 33 entries.  64 bits: what a call asks for may be
// far more pages than there are.
__device__ __forceinline__ int64_t block_exclusive(int64_t x, int64_t* s_warp, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  int64_t inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();                            // the previous scan's readers are done
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int64_t w = lane < n_warps ? s_warp[lane] : 0;
    int64_t winc = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, winc, d);
      if (lane >= d) winc += y;
    }
    s_warp[lane] = winc - w;
    if (lane == 31) s_warp[32] = winc;
  }
  __syncthreads();
  total = s_warp[32];
  return s_warp[warp] + inc - x;
}

// Whether the n numbers are in range and, with `distinct`, none comes twice.  Sets their bits in s_bits.
__device__ __forceinline__ bool check_seqs(const int32_t* seqs, int n, int max_seqs, bool distinct, uint32_t* s_bits) {
  for (int i = threadIdx.x; i < (max_seqs + 31) / 32; i += blockDim.x) s_bits[i] = 0u;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = seqs[i];
    if (s < 0 || s >= max_seqs) { bad = true; continue; }
    const uint32_t bit = 1u << (s & 31);
    if ((atomicOr(&s_bits[s >> 5], bit) & bit) && distinct) bad = true;
  }
  return !__syncthreads_or(bad);
}

// ---- truncate -----------------------------------------------------------------------------------------
// One block per listed sequence.  A sequence listed twice is shortened to the smaller length: whichever block
// lowers the length frees exactly the pages between the old and the new one.
__global__ void __launch_bounds__(128) truncate_kernel(Table t, const int32_t* __restrict__ seqs,
                                                       const int32_t* __restrict__ new_lens, int n) {
  __shared__ int s_old;
  begin();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) bad |= seqs[i] < 0 || seqs[i] >= t.max_seqs || new_lens[i] < 0;
  if (__syncthreads_or(bad)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(t.status, FFA_PAGES_BAD_ARGUMENT);
    return;
  }
  const int s = seqs[blockIdx.x], len = new_lens[blockIdx.x];
  if (threadIdx.x == 0) s_old = atomicMin(t.seq_lens + s, len);
  __syncthreads();
  const int to = min(pages_of(s_old), t.cols);
  int32_t* row = t.row(s);
  for (int j = pages_of(len) + threadIdx.x; j < to; j += blockDim.x) {
    const int p = row[j];
    row[j] = -1;
    if (p >= 0 && p < t.n_pages) atomicSub(t.refcount + p, 1);
  }
}

// ---- fork ---------------------------------------------------------------------------------------------
// One block per child.  Every block checks the whole list; the children's lengths are written by the last block to
// finish, so that no block sees another's child as taken.
__global__ void __launch_bounds__(256) fork_kernel(Table t, const int32_t* __restrict__ parents,
                                                   const int32_t* __restrict__ children, int n) {
  extern __shared__ uint32_t s_bits[];
  __shared__ int s_last;
  begin();
  bool ok = check_seqs(children, n, t.max_seqs, true, s_bits);
  if (ok) {
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int p = parents[i];
      if (p < 0 || p >= t.max_seqs || ((s_bits[p >> 5] >> (p & 31)) & 1u) || t.seq_lens[children[i]] != 0) bad = true;
    }
    ok = !__syncthreads_or(bad);
  }
  if (!ok) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(t.status, FFA_PAGES_BAD_ARGUMENT);
    return;
  }
  const int parent = parents[blockIdx.x];
  const int held = min(pages_of(t.seq_lens[parent]), t.cols);
  const int32_t* src = t.row(parent);
  int32_t* dst = t.row(children[blockIdx.x]);
  for (int j = threadIdx.x; j < t.cols; j += blockDim.x) {
    const int p = j < held ? src[j] : -1;
    dst[j] = p;
    if (p >= 0 && p < t.n_pages) atomicAdd(t.refcount + p, 1);
  }
  __syncthreads();                            // every thread of the block has read the lengths
  if (threadIdx.x == 0) s_last = atomicAdd(t.hdr() + kHdrArrive, 1) == n - 1;
  __syncthreads();
  if (!s_last) return;
  for (int i = threadIdx.x; i < n; i += blockDim.x) t.seq_lens[children[i]] = t.seq_lens[parents[i]];
  if (threadIdx.x == 0) t.hdr()[kHdrArrive] = 0;
}

// ---- extend -------------------------------------------------------------------------------------------
// One block: check, count the pages that each sequence needs, find that many free pages (lowest first), hand them
// out in the order of the list.  A sequence whose open page is shared gets a page of its own in its place, and a
// job for the copy kernel.
__global__ void __launch_bounds__(kPlanThreads) extend_plan_kernel(Table t, const int32_t* __restrict__ seqs,
                                                                   const int32_t* __restrict__ n_new, int n) {
  extern __shared__ uint32_t s_bits[];
  __shared__ int64_t s_warp[33];
  __shared__ int s_count[kPlanThreads / 32];
  begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // free pages: every warp counts its stretch of the reference counts (and lists them from its place on, below)
  const int per = (((t.n_pages + 31) / 32 + 31) / 32) * 32;          // a stretch in whole rows of 32
  const int from = min(t.n_pages, warp * per), to = min(t.n_pages, from + per);
  int n_free = 0;
#pragma unroll 4
  for (int p = from + lane; p < to; p += 32) n_free += t.refcount[p] == 0;
  bool ok = check_seqs(seqs, n, t.max_seqs, true, s_bits);
  if (ok) {
    bool bad = false;
    for (int i = tid; i < n; i += kPlanThreads) {
      const int add = n_new[i];
      if (add < 0 || t.seq_lens[seqs[i]] < 0 || static_cast<int64_t>(t.seq_lens[seqs[i]]) + add > static_cast<int64_t>(t.cols) * kPage) bad = true;
    }
    ok = !__syncthreads_or(bad);
  }
  int32_t* const hdr = t.hdr();
  if (!ok) {
    if (tid == 0) { atomicOr(t.status, FFA_PAGES_BAD_ARGUMENT); hdr[kHdrJobs] = 0; }
    return;
  }
  int64_t total = 0;                          // pages that the call needs
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int need = 0;
    if (i < n) {
      const int s = seqs[i], add = n_new[i], len = t.seq_lens[s];
      int src = -1, rows = 0;
      if (add > 0) {
        need = pages_of(len + add) - pages_of(len);
        if (len % kPage) {
          const int p = t.row(s)[len / kPage];
          if (p >= 0 && p < t.n_pages && t.refcount[p] > 1) { src = p; rows = len % kPage; ++need; }
        }
      }
      t.job_src()[i] = src;
      t.job_rows()[i] = rows;
    }
    int64_t sum;
    const int64_t before = block_exclusive(need, s_warp, sum);
    if (i < n) t.first_new()[i] = static_cast<int>(min(total + before, static_cast<int64_t>(t.n_pages)));
    total += sum;
  }
  int found = 0;
  if (total > 0) {
    n_free = __reduce_add_sync(0xffffffffu, n_free);
    if (lane == 0) s_count[warp] = n_free;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at += s_count[w];
      found += s_count[w];
    }
    if (found >= total) {
      for (int p0 = from; p0 < to && at < total; p0 += 32) {
        const bool is_free = p0 + lane < to && t.refcount[p0 + lane] == 0;
        const uint32_t m = __ballot_sync(0xffffffffu, is_free);
        const int k = at + __popc(m & ((1u << lane) - 1u));
        if (is_free && k < total) t.free_list()[k] = p0 + lane;
        at += __popc(m);
      }
    }
  }
  __syncthreads();
  if (found < total) {
    if (tid == 0) { atomicOr(t.status, FFA_PAGES_NO_SPACE); hdr[kHdrJobs] = 0; }
    return;
  }
  // a thread to a sequence; one that needs many pages leaves them to its warp
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int c0 = 0, c1 = 0, first = 0, s = 0;
    if (i < n && n_new[i] > 0) {
      s = seqs[i];
      const int len = t.seq_lens[s], add = n_new[i];
      int32_t* row = t.row(s);
      first = t.first_new()[i];
      if (t.job_src()[i] >= 0) {
        const int p = t.free_list()[first++];
        atomicSub(t.refcount + t.job_src()[i], 1);
        t.job_dst()[i] = p;
        row[len / kPage] = p;
        t.refcount[p] = 1;
      }
      c0 = pages_of(len);
      c1 = pages_of(len + add);
      if (c1 - c0 <= 4) {
        for (; c0 < c1; ++c0, ++first) {
          const int p = t.free_list()[first];
          row[c0] = p;
          t.refcount[p] = 1;
        }
      }
      t.seq_lens[s] = len + add;
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, c0 < c1); todo; todo &= todo - 1) {
      const int from = __ffs(todo) - 1;
      const int a = __shfl_sync(0xffffffffu, c0, from), b = __shfl_sync(0xffffffffu, c1, from), f = __shfl_sync(0xffffffffu, first, from);
      int32_t* row = t.row(__shfl_sync(0xffffffffu, s, from));
      for (int c = a + lane; c < b; c += 32) {
        const int p = t.free_list()[f + c - a];
        row[c] = p;
        t.refcount[p] = 1;
      }
    }
  }
  if (tid == 0) hdr[kHdrJobs] = n;
}

// ---- compact ------------------------------------------------------------------------------------------
// One block: with L live pages in all, the k-th live page numbered L or above goes to the k-th free page below L.
// free_list()[p]: for a free page below L the number k of the job that fills it, for a page at L or above its new
// number.  job_rows(): the reference counts of the moved pages.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(Table t) {
  __shared__ int s_live[32], s_hole[32], s_move[32];
  begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (((t.n_pages + 31) / 32 + 31) / 32) * 32;
  const int from = min(t.n_pages, warp * per), to = min(t.n_pages, from + per);
  int mine = 0;
  for (int p = from + lane; p < to; p += 32) mine += t.refcount[p] != 0;
#pragma unroll
  for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) s_live[warp] = mine;
  __syncthreads();
  int live = 0;
  for (int w = 0; w < 32; ++w) live += s_live[w];
  int holes = 0;
  for (int p = from + lane; p < to; p += 32) holes += p < live && t.refcount[p] == 0;
#pragma unroll
  for (int d = 16; d; d >>= 1) holes += __shfl_xor_sync(0xffffffffu, holes, d);
  // of this stretch's live pages those below `live` stay
  const int below = max(0, min(to, live) - from);
  if (lane == 0) { s_hole[warp] = holes; s_move[warp] = s_live[warp] - (below - holes); }
  __syncthreads();
  int hole = 0, move = 0, jobs = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) { hole += s_hole[w]; move += s_move[w]; }
    jobs += s_move[w];
  }
  for (int p0 = from; p0 < to; p0 += 32) {
    const int p = p0 + lane;
    const int count = p < to ? t.refcount[p] : 0;
    const bool is_hole = p < to && p < live && count == 0, is_move = p < to && p >= live && count != 0;
    const uint32_t mh = __ballot_sync(0xffffffffu, is_hole), mm = __ballot_sync(0xffffffffu, is_move);
    const uint32_t under = (1u << lane) - 1u;
    if (is_hole) {
      const int k = hole + __popc(mh & under);
      t.job_dst()[k] = p;
      t.free_list()[p] = k;
    }
    if (is_move) {
      const int k = move + __popc(mm & under);
      t.job_src()[k] = p;
      t.job_rows()[k] = count;
    } else if (p < to && p >= live) {
      t.free_list()[p] = p;                   // a free page keeps its number, should an entry name it
    }
    hole += __popc(mh);
    move += __popc(mm);
  }
  __syncthreads();                            // holes and moved pages come from different warps
  for (int k = threadIdx.x; k < jobs; k += kPlanThreads) t.free_list()[t.job_src()[k]] = t.job_dst()[k];
  if (threadIdx.x == 0) { t.hdr()[kHdrJobs] = jobs; t.hdr()[kHdrLive] = live; }
}

// Rewrites block table and reference counts entry by entry; out may be the state itself.  Only pages numbered
// `live` or above are renamed, and the reference count of every entry below depends on that entry alone.
__device__ __forceinline__ void compact_apply(const Table& t, int32_t* bt_out, int32_t* rc_out, int block, int blocks) {
  const int live = t.hdr()[kHdrLive], warps = blocks * kCopyThreads / 32, lane = threadIdx.x & 31;
  for (int s = (block * kCopyThreads + threadIdx.x) / 32; s < t.max_seqs; s += warps) {
    const int64_t at = static_cast<int64_t>(s) * t.stride;
    for (int j = lane; j < t.cols; j += 32) {
      const int p = t.block_table[at + j];
      bt_out[at + j] = p >= live && p < t.n_pages ? t.free_list()[p] : p;
    }
  }
  for (int i = block * kCopyThreads + threadIdx.x; i < t.n_pages; i += blocks * kCopyThreads) {
    const int c = t.refcount[i];
    rc_out[i] = i >= live ? 0 : c ? c : t.job_rows()[t.free_list()[i]];
  }
}

// ---- page contents --------------------------------------------------------------------------------------
// Copies the first rows(i) tokens of page src(i) to page dst(i) in every pool, all jobs of the header.  A block takes
// 16 KiB pieces, piece number fastest, so that neighbouring blocks read and write one page together.  COMPACT: whole pages,
// and the first blocks rewrite table and counts before they join in.
constexpr int kApplyBlocks = 64;
template <bool COMPACT>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(Table t, const uint64_t* __restrict__ bases,
                                                                  const int32_t* __restrict__ token_bytes, int n_pools,
                                                                  int pieces, int32_t* bt_out, int32_t* rc_out) {
  begin();
  if (COMPACT && blockIdx.x < kApplyBlocks) compact_apply(t, bt_out, rc_out, blockIdx.x, min(kApplyBlocks, static_cast<int>(gridDim.x)));
  const int jobs = t.hdr()[kHdrJobs];
  const int64_t n_items = static_cast<int64_t>(jobs) * n_pools * pieces;
  for (int64_t item = blockIdx.x; item < n_items; item += gridDim.x) {
    const int piece = static_cast<int>(item % pieces);
    const int pool = static_cast<int>(item / pieces % n_pools);
    const int64_t job = item / pieces / n_pools;
    const int rows = COMPACT ? kPage : t.job_rows()[job];
    const int64_t bytes = static_cast<int64_t>(rows) * token_bytes[pool], page = static_cast<int64_t>(kPage) * token_bytes[pool];
    const int64_t at = static_cast<int64_t>(piece) * kChunk;
    if (at >= bytes) continue;
    const char* src = reinterpret_cast<const char*>(bases[pool]) + t.job_src()[job] * page;
    char* dst = reinterpret_cast<char*>(bases[pool]) + t.job_dst()[job] * page;
    uint4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t o = at + (u * kCopyThreads + threadIdx.x) * 16;
      if (o < bytes) x[u] = *reinterpret_cast<const uint4*>(src + o);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t o = at + (u * kCopyThreads + threadIdx.x) * 16;
      if (o < bytes) *reinterpret_cast<uint4*>(dst + o) = x[u];
    }
  }
}

int make_table(const FfaPageTable* a, Table* t) {
  if (!a || !a->block_table || !a->seq_lens || !a->refcount || !a->status || !a->scratch) return FFA_E_NULL;
  if (a->n_pages <= 0 || a->max_seqs <= 0 || a->cols <= 0 || a->bt_stride < a->cols || a->cols > INT32_MAX / kPage) return FFA_E_SHAPE;
  if (a->max_seqs > kMaxSeqs) return FFA_E_LIMIT;
  if (a->scratch_bytes < 4 * scratch_ints(a->n_pages, a->max_seqs)) return FFA_E_WORKSPACE;
  *t = Table{a->n_pages, a->max_seqs, a->cols, a->bt_stride, a->block_table, a->seq_lens, a->refcount, a->status,
             static_cast<int32_t*>(a->scratch)};
  return FFA_OK;
}

template <typename... P, typename... A>
int launch(const char* what, void (*kernel)(P...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? FFA_OK : note_cuda_error(e, what);
}

template <bool COMPACT>
int launch_copy(const Table& t, const FfaPagePools* pools, int64_t max_jobs, int32_t* bt_out, int32_t* rc_out, cudaStream_t st) {
  if (!COMPACT && pools->n_pools == 0) return FFA_OK;
  const int pieces = static_cast<int>((static_cast<int64_t>(kPage) * pools->max_token_bytes + kChunk - 1) / kChunk);
  const int64_t items = max_jobs * pools->n_pools * pieces, least = COMPACT ? kApplyBlocks : 1;
  const unsigned blocks = static_cast<unsigned>(items > 148 * 8 ? 148 * 8 : items > least ? items : least);
  return launch("ffa_pages (copy)", copy_pages_kernel<COMPACT>, blocks, kCopyThreads, 0, st, t, pools->bases, pools->token_bytes,
                pools->n_pools, pieces, bt_out, rc_out);
}

int check_pools(const FfaPagePools* p) {
  if (!p || p->n_pools < 0 || (p->n_pools > 0 && (!p->bases || !p->token_bytes))) return FFA_E_NULL;
  if (p->n_pools > 0 && (p->max_token_bytes <= 0 || p->max_token_bytes % 16)) return FFA_E_SHAPE;
  return FFA_OK;
}

size_t bits_bytes(int max_seqs) { return (static_cast<size_t>(max_seqs) + 31) / 32 * 4; }

}  // namespace
}  // namespace ffa

using namespace ffa;

extern "C" size_t ffa_pages_scratch_bytes(int32_t n_pages, int32_t max_seqs) {
  if (n_pages <= 0 || max_seqs <= 0) return 0;
  return 4 * scratch_ints(n_pages, max_seqs);
}

extern "C" int ffa_pages_truncate(const FfaPageTable* table, const int32_t* seqs, const int32_t* new_lens, int32_t n,
                                  ffa_stream_t stream) {
  Table t;
  const int rc = make_table(table, &t);
  if (rc) return rc;
  if (!seqs || !new_lens) return FFA_E_NULL;
  if (n <= 0 || n > t.max_seqs) return FFA_E_SHAPE;
  return launch("ffa_pages_truncate", truncate_kernel, n, 128, 0, reinterpret_cast<cudaStream_t>(stream), t, seqs, new_lens, n);
}

extern "C" int ffa_pages_fork(const FfaPageTable* table, const int32_t* parents, const int32_t* children, int32_t n,
                              ffa_stream_t stream) {
  Table t;
  const int rc = make_table(table, &t);
  if (rc) return rc;
  if (!parents || !children) return FFA_E_NULL;
  if (n <= 0 || n > t.max_seqs) return FFA_E_SHAPE;
  return launch("ffa_pages_fork", fork_kernel, n, 256, bits_bytes(t.max_seqs), reinterpret_cast<cudaStream_t>(stream), t, parents, children, n);
}

extern "C" int ffa_pages_extend(const FfaPageTable* table, const FfaPagePools* pools, const int32_t* seqs,
                                const int32_t* n_new, int32_t n, ffa_stream_t stream) {
  Table t;
  int rc = make_table(table, &t);
  if (rc) return rc;
  if ((rc = check_pools(pools))) return rc;
  if (!seqs || !n_new) return FFA_E_NULL;
  if (n <= 0 || n > t.max_seqs) return FFA_E_SHAPE;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if ((rc = launch("ffa_pages_extend", extend_plan_kernel, 1, kPlanThreads, bits_bytes(t.max_seqs), st, t, seqs, n_new, n))) return rc;
  return launch_copy<false>(t, pools, n, nullptr, nullptr, st);
}

extern "C" int ffa_pages_compact(const FfaPageTable* table, const FfaPagePools* pools, int32_t* block_table_out,
                                 int32_t* refcount_out, ffa_stream_t stream) {
  Table t;
  int rc = make_table(table, &t);
  if (rc) return rc;
  if ((rc = check_pools(pools))) return rc;
  if (!block_table_out || !refcount_out) return FFA_E_NULL;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if ((rc = launch("ffa_pages_compact", compact_plan_kernel, 1, kPlanThreads, 0, st, t))) return rc;
  return launch_copy<true>(t, pools, t.n_pages / 2, block_table_out, refcount_out, st);
}
