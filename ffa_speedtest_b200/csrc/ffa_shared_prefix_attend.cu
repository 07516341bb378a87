// Attention over the runs of the shared-prefix decode (ffa_shared_prefix.cuh) on the fifth-generation tensor cores.
//
// One persistent CTA per SM walks its runs tile by tile (128 query rows x 128 tokens):
//
//   S[128 rows, 128 tokens] = sum over pieces of q, base and residual:  Qpiece . K^T    kind::f8f6f4, fp32 in TMEM
//   P = 2^(S * row scale - m)                                                           one row per thread
//   O[128 rows, 128 channels] += P . V                                                  kind::f16, P from TMEM
//
// K is used as it lies in the cache: q comes as e4m3 pieces (ffa_shared_prefix.cu), and the products of every piece with the raw base and residual
// bytes accumulate into one fp32 tile.  That costs 4 (6) fp8 MMAs where a dequantised fp16 K would cost two fp8-MMA
// times one, but K never passes through registers: TMA writes it, the tensor core reads it.
//
// Bound: per 128 tokens and kv-head 64 KiB arrive (about 2800 clocks of an SM's share of HBM); the tensor core needs
// 4 x 256 + 512 clocks, the softmax warps 128 exponentials per row = 1024 clocks of their SM quarter's unit.
//
// Warps: 0 builds the run list and loads K and V; 1 issues MMAs; 2 loads q; 4-7 softmax (TMEM lanes 32 * (warp % 4)).
// A ring of 32 KiB slots holds K tiles (base 16 KiB, residual 16 KiB) and V tiles in the order of use: K0 K1 V0 K2 V1 ...
// QK of tile i+1 is issued before PV of tile i, so the tensor core works on it while the softmax of tile i runs.  S has
// two buffers (P overwrites the S it came from), O has two (a run's O is written out while the next run computes).
// Runs of up to eight query rows (a sequence's own pages) have two small q buffers, larger ones one of 128 rows.
// MMAs complete in the order of issue, which is what keeps QK(i+2) off the buffer until PV(i) has read P from it.
//
// Every wait ends after 0.2 s at most: the CTA then leaves its loops, lets its copies and MMAs in flight finish, and
// marks the call, and the merge writes NaN.
#include <cuda.h>

#include "ffa_shared_prefix.cuh"

namespace ffa {
namespace {

constexpr int kThreads = 256;
constexpr int kSlot = 32 * 1024;
constexpr int kPiece = 16 * 1024;             // 128 rows x 128 bytes
constexpr int kRunChunk = 32;
constexpr unsigned long long kWaitNs = 200ull * 1000 * 1000;

struct Run {
  int32_t table_row, row0, rows, head;
  int32_t tok0, end, tiles;                   // first token, token that ends the segment, tiles
  int32_t small;                              // q of at most eight rows
  int64_t part;                               // first row of its partial
};

template <int NP>                             // pieces of q
struct Smem {
  static constexpr int kSlots = 5;
  static constexpr int kOffSmall = NP * kPiece;                         // [2][NP] of 8 rows x 128 bytes
  static constexpr int kOffRing = kOffSmall + 2 * NP * 1024;
  static constexpr int kOffRuns = kOffRing + kSlots * kSlot;
  static constexpr int kOffHead = kOffRuns + 2 * kRunChunk * static_cast<int>(sizeof(Run));   // 2 x (count, last)
  static constexpr int kOffBars = kOffHead + 16;
  // full[slots], empty[slots], sfull[2], pfull[2], odone, ofree[2], qfull[3], qfree[3], runfull[2], runempty[2], final
  static constexpr int kBars = 2 * kSlots + 2 + 2 + 1 + 2 + 3 + 3 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBars + kBars * 8;                 // TMEM address, abort flag, the same for the last waits
  static constexpr int kBytes = kOffMisc + 16 + 1024;                   // and slack to align to 1024
};
static_assert(Smem<2>::kBytes <= 227 * 1024 && Smem<3>::kBytes <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// A lane's wait for the phase of this parity; gives up after kWaitNs, or when another warp of the CTA has.
__device__ __forceinline__ bool wait_lane(uint32_t bar, uint32_t parity, int* abort_flag) {
  unsigned long long t0 = 0;
  for (int spin = 0;; ++spin) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((spin & 63) == 63) {
      if (*reinterpret_cast<volatile int*>(abort_flag) != 0) return false;
      unsigned long long now;
      asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(now));
      if (t0 == 0) t0 = now;
      else if (now - t0 > kWaitNs) {
        atomicExch(abort_flag, 1);
        return false;
      }
    }
  }
}
// The whole warp waits and every lane gets the same answer.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int* abort_flag) {
  return __all_sync(0xffffffffu, wait_lane(bar, parity, abort_flag)) != 0;
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2, version 1).  K-major: rows of 128 bytes, groups
// of 8 rows 1024 bytes apart.  MN-major (V: channels contiguous, tokens down): 64 channels to a row, the next 64
// channels `lead` bytes on, groups of 8 tokens 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// Instruction descriptor: fp32 accumulator, A and B formats, B transposed (MN-major) or not, M = N = 128.
__host__ __device__ constexpr uint32_t instr(uint32_t a, uint32_t b, uint32_t b_mn) {
  return (1u << 4) | (a << 7) | (b << 10) | (b_mn << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31,%32};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// One lane of the converged warp, by the instruction that tells the compiler that it is one.
__device__ __forceinline__ bool elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int NP, bool VBF16>
__global__ void __launch_bounds__(kThreads, 1) sp_attend_mma_kernel(const __grid_constant__ SpParams p,
                                                                    const __grid_constant__ CUtensorMap map_k,
                                                                    const __grid_constant__ CUtensorMap map_r,
                                                                    const __grid_constant__ CUtensorMap map_v,
                                                                    const __grid_constant__ CUtensorMap map_q,
                                                                    const __grid_constant__ CUtensorMap map_q8) {
  using L = Smem<NP>;
  constexpr int NS = L::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // uniform for the compiler too: MMAs issued under a branch that it takes for divergent cost 100 clocks and more each
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, cta = blockIdx.x;
  const uint32_t s_q = smem_u32(smem), s_ring = s_q + L::kOffRing, bars = s_q + L::kOffBars;
  Run* const runs = reinterpret_cast<Run*>(smem + L::kOffRuns);
  volatile int* const run_head = reinterpret_cast<volatile int*>(smem + L::kOffHead);
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kOffMisc);
  int* const aborted = reinterpret_cast<int*>(smem + L::kOffMisc + 4);
  auto full = [&](uint32_t s) { return bars + 8 * s; };
  auto empty = [&](uint32_t s) { return bars + 8 * (NS + s); };
  const uint32_t rest = bars + 16 * NS;
  auto sfull = [&](uint32_t i) { return rest + 8 * i; };
  auto pfull = [&](uint32_t i) { return rest + 16 + 8 * i; };
  const uint32_t odone = rest + 32;
  auto ofree = [&](uint32_t i) { return rest + 40 + 8 * i; };
  // q buffers: 0 the large one, 1 and 2 the small ones
  auto qfull = [&](uint32_t i) { return rest + 56 + 8 * i; };
  auto qfree = [&](uint32_t i) { return rest + 80 + 8 * i; };
  auto runfull = [&](uint32_t i) { return rest + 104 + 8 * i; };
  auto runempty = [&](uint32_t i) { return rest + 120 + 8 * i; };
  const uint32_t final_bar = rest + 136;
  auto q_buffer = [&](uint32_t i) { return i == 0 ? s_q : s_q + L::kOffSmall + (i - 1) * NP * 1024; };
  const uint32_t q_piece[2] = {kPiece, 1024};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * NS; ++i) mbar_init(bars + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull(i), 1);
      mbar_init(pfull(i), 4);
      mbar_init(ofree(i), 4);
      mbar_init(runfull(i), 1);
      mbar_init(runempty(i), 1 + 1 + 4);
    }
    mbar_init(odone, 1);
    for (int i = 0; i < 3; ++i) { mbar_init(qfull(i), 1); mbar_init(qfree(i), 1); }
    mbar_init(final_bar, 1);
    *aborted = 0;
    aborted[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(s_q + L::kOffMisc) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int64_t W = static_cast<int64_t>(p.hdr[1]) * p.HKV;
  const int n_used = sp_ctas(W, p.n_ctas);
  const bool idle = cta >= n_used || W == 0;
  const uint32_t tmem = *tmem_slot;           // columns: S0 0, S1 128, O0 256, O1 384

  // The next run for a consumer warp, in order; false at the end (or when the CTA gave up).
  int ch = 0, at = 0, count = -1, last = 0;
  auto next_run = [&](Run& r) -> bool {
    for (;;) {
      if (count < 0) {
        if (!wait(runfull(ch & 1), (ch >> 1) & 1, aborted)) return false;
        count = run_head[2 * (ch & 1)];
        last = run_head[2 * (ch & 1) + 1];
        at = 0;
      }
      if (at < count) {
        r = runs[(ch & 1) * kRunChunk + at];
        ++at;
        return true;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(runempty(ch & 1));
      if (last) return false;
      ++ch;
      count = -1;
    }
  };

  uint32_t issued = 0;                        // warp 0: slots filled so far
  if (idle) {
    // nothing for this CTA
  } else if (warp == 0) {
    // ---- run list, K and V ----
    const int64_t x0 = sp_first(cta, W, n_used), x1 = sp_first(cta + 1, W, n_used);
    const int n_seg = p.hdr[0];
    const int64_t n_units = static_cast<int64_t>(n_seg) * p.HKV;
    int64_t unit = static_cast<int64_t>(p.start[2 * cta]) * p.HKV + p.start[2 * cta + 1];
    // a tile whose V still has to be asked for
    int v_pages[2] = {-1, -1}, v_head = 0, v_n = 0;
    bool have_v = false;
    auto slot_for = [&](uint32_t bytes, uint32_t& dst, uint32_t& bar) -> bool {
      const uint32_t s = issued % NS, round = issued / NS;
      if (round > 0 && !wait(empty(s), (round - 1) & 1, aborted)) return false;
      dst = s_ring + s * kSlot;
      bar = full(s);
      if (elect()) mbar_expect_tx(bar, bytes);
      ++issued;
      return true;
    };
    auto load_v = [&]() -> bool {
      uint32_t dst, bar;
      if (!slot_for(v_n * 16384, dst, bar)) return false;
      if (elect())
        for (int i = 0; i < v_n; ++i)
          for (int h = 0; h < 2; ++h)
            tma_load(dst + h * 16384 + i * 8192, &map_v, v_head * 256 + h * 128, v_pages[i] * kPage, bar);
      return true;
    };
    bool ok = true;
    for (int c = 0; ok; ++c) {
      if (c >= 2 && !wait(runempty(c & 1), ((c >> 1) - 1) & 1, aborted)) break;
      const int64_t u = unit + lane;
      Run r{};
      int n = 0;
      bool past = u >= n_units;
      if (!past) {
        const int si = static_cast<int>(u / p.HKV), head = static_cast<int>(u % p.HKV);
        const SpSegment s = p.seg[si];
        const int64_t pos = static_cast<int64_t>(p.cum[si]) * p.HKV + static_cast<int64_t>(head) * sp_cost(s.tiles) + kSpUnitCost;
        past = pos >= x1;
        const int64_t a = pos > x0 ? pos : x0, b = pos + s.tiles < x1 ? pos + s.tiles : x1;
        if (b > a) {
          n = static_cast<int>(b - a);
          r.table_row = s.table_row; r.row0 = s.row0; r.rows = s.rows; r.head = head;
          r.tok0 = s.page0 * kPage + static_cast<int>(a - pos) * kSpTile;
          r.end = s.end;
          r.tiles = n;
          r.small = s.rows <= 8;
          r.part = sp_part_row(p, s, head, cta);
        }
      }
      const uint32_t live = __ballot_sync(0xffffffffu, n > 0);
      const int is_last = __any_sync(0xffffffffu, past) ? 1 : 0, n_runs = __popc(live);
      if (n > 0) runs[(c & 1) * kRunChunk + __popc(live & ((1u << lane) - 1u))] = r;
      if (lane == 0) { run_head[2 * (c & 1)] = n_runs; run_head[2 * (c & 1) + 1] = is_last; }
      __syncwarp();
      if (lane == 0) mbar_arrive(runfull(c & 1));
      unit += 32;
      for (int j = 0; j < n_runs && ok; ++j) {
        const Run q = runs[(c & 1) * kRunChunk + j];
        const int32_t* row = p.bt + static_cast<int64_t>(q.table_row) * p.bt_stride;
        const int col0 = q.tok0 / kPage, cols = (q.end + kPage - 1) / kPage;     // cols <= p.cols
        auto page_at = [&](int col) {
          const int x = col < cols ? row[col] : -1;
          return x >= 0 && x < p.n_pages ? x : -1;     // TMA reads zeros at negative rows
        };
        int ids = page_at(col0 + lane), ids_next = page_at(col0 + 32 + lane);
        for (int t = 0; t < q.tiles; ++t) {
          if (t > 0 && (t & 15) == 0) { ids = ids_next; ids_next = page_at(col0 + 2 * t + 32 + lane); }
          const int n_pages = min(2, cols - (col0 + 2 * t));
          const int pg0 = __shfl_sync(0xffffffffu, ids, (2 * t) & 31), pg1 = __shfl_sync(0xffffffffu, ids, (2 * t + 1) & 31);
          uint32_t dst, bar;
          if (!slot_for(n_pages * (p.r ? 16384 : 8192), dst, bar)) { ok = false; break; }
          if (elect())
            for (int i = 0; i < n_pages; ++i) {
              const int y = (i ? pg1 : pg0) * kPage;
              tma_load(dst + i * 8192, &map_k, q.head * 128, y, bar);
              if (p.r) tma_load(dst + kPiece + i * 8192, &map_r, q.head * 128, y, bar);
            }
          if (have_v && !load_v()) { ok = false; break; }
          v_pages[0] = pg0; v_pages[1] = pg1; v_head = q.head; v_n = n_pages;
          have_v = true;
        }
      }
      if (is_last) break;
    }
    if (ok && have_v) load_v();
  } else if (warp == 1) {
    // ---- MMA ----
    const uint32_t idesc_s = instr(0, p.fp8 == FFA_E4M3 ? 0 : 1, 0), idesc_o = instr(VBF16 ? 1 : 0, VBF16 ? 1 : 0, 1);
    uint32_t used = 0;                        // slots consumed
    uint32_t i = 0;                           // tiles whose QK was issued
    int n_run = 0;
    // the tile whose PV is still to come
    bool have = false, first = false;
    int valid = 0, o_buf = 0, o_round = 0;
    auto pv = [&]() -> bool {
      const uint32_t j = i - 1, s = used % NS;
      if (!wait(full(s), (used / NS) & 1, aborted)) return false;
      const uint32_t v = s_ring + s * kSlot;
      const int steps = (valid + 15) / 16;
      if (valid < steps * 16) {
        // tokens past the end of the sequence: whatever their V holds, 0 * V has to be 0
        for (int x = lane; x < (steps * 16 - valid) * 16; x += 32) {
          const int row = valid + x / 16, h = (x >> 3) & 1, ck = x & 7;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(v + h * 16384 + row * 128 + ck * 16), "r"(0) : "memory");
        }
        fence_async();
        __syncwarp();
      }
      if (first && o_round > 0 && !wait(ofree(o_buf), (o_round - 1) & 1, aborted)) return false;
      if (!wait(pfull(j & 1), (j >> 1) & 1, aborted)) return false;
      fence_after();
      if (elect()) {
        const uint64_t dv = desc(v, 16384);
        for (int k = 0; k < steps; ++k)
          mma_16_tmem(tmem + 256 + 128 * o_buf, tmem + 128 * (j & 1) + 8 * k, dv + 128 * k, idesc_o, !(first && k == 0));
        commit(empty(s));
        commit(odone);
      }
      __syncwarp();
      ++used;
      return true;
    };
    Run r;
    bool ok = true;
    uint32_t q_large = 0, q_small = 0;        // runs of either kind so far
    while (ok && next_run(r)) {
      const uint32_t qb = r.small ? 1 + (q_small & 1) : 0;
      if (!wait(qfull(qb), (r.small ? q_small >> 1 : q_large) & 1, aborted)) break;
      if (r.small) ++q_small; else ++q_large;
      fence_after();
      const uint64_t dq = desc(q_buffer(qb), 16);
      const uint32_t q_step = q_piece[r.small ? 1 : 0] >> 4;
      for (int t = 0; t < r.tiles; ++t) {
        const uint32_t s = used % NS;
        if (!wait(full(s), (used / NS) & 1, aborted)) { ok = false; break; }
        fence_after();
        if (elect()) {
          const uint64_t dk = desc(s_ring + s * kSlot, 16);
          uint32_t acc = 0;
          for (int part = 0; part < (p.r ? 2 : 1); ++part)
#pragma unroll
            for (int piece = 0; piece < NP; ++piece)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                mma_fp8(tmem + 128 * (i & 1), dq + piece * q_step + 2 * k, dk + (part * kPiece >> 4) + 2 * k, idesc_s, acc);
                acc = 1;
              }
          commit(empty(s));
          commit(sfull(i & 1));
          if (t == r.tiles - 1) commit(qfree(qb));
        }
        __syncwarp();
        ++used;
        if (have && !pv()) { ok = false; break; }
        ++i;
        have = true;
        first = t == 0;
        valid = min(kSpTile, r.end - (r.tok0 + t * kSpTile));
        o_buf = n_run & 1;
        o_round = n_run >> 1;
      }
      ++n_run;
    }
    if (ok && have && *reinterpret_cast<volatile int*>(aborted) == 0) pv();
  } else if (warp == 2) {
    // ---- q ----
    uint32_t q_large = 0, q_small = 0;
    const int rows_head = p.B * p.G;
    Run r;
    asm volatile("fence.proxy.async.global;\n" ::: "memory");       // q's pieces were written by ordinary stores
    while (next_run(r)) {
      const uint32_t qb = r.small ? 1 + (q_small & 1) : 0, round = r.small ? q_small >> 1 : q_large;
      if (round > 0 && !wait(qfree(qb), (round - 1) & 1, aborted)) break;
      if (r.small) ++q_small; else ++q_large;
      if (elect()) {
        const uint32_t bytes = q_piece[r.small ? 1 : 0];
        mbar_expect_tx(qfull(qb), NP * bytes);
        for (int piece = 0; piece < NP; ++piece)
          tma_load(q_buffer(qb) + piece * bytes, r.small ? &map_q8 : &map_q, 0, (piece * p.HKV + r.head) * rows_head + r.row0, qfull(qb));
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ---- softmax: one query row per thread ----
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t i = 0;
    int n_run = 0;
    bool have_o = false, o_live = false;      // a finished run whose O is still to be written
    int64_t o_part = 0;
    float o_m = 0.f, o_l = 0.f;
    auto write_o = [&](int buf) {
      if (__any_sync(0xffffffffu, o_live)) {
        float4* dst = reinterpret_cast<float4*>(p.part_o + (o_part + row) * kHeadDim);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t x[32];
          tmem_ld32(x, tmem + lanes + 256 + 128 * buf + 32 * c);
          tmem_wait_ld();
          if (o_live)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[8 * c + e] = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                                           __uint_as_float(x[4 * e + 3]));
        }
        if (o_live) p.part_ml[o_part + row] = make_float2(o_m, o_l);
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree(buf));
    };
    Run r;
    bool ok = true;
    while (ok && next_run(r)) {
      const bool live = row < r.rows, any_live = quarter * 32 < r.rows;
      float m = -INFINITY, l = 0.f, scale = 0.f;
      int end = r.end;
      if (live) {
        scale = p.q_scale[static_cast<int64_t>(r.head) * p.B * p.G + r.row0 + row];
        end = min(end, p.seq_lens[(r.row0 + row) / p.G]);
      }
      for (int t = 0; t < r.tiles; ++t, ++i) {
        const uint32_t s_addr = tmem + lanes + 128 * (i & 1);
        if (!wait(sfull(i & 1), (i >> 1) & 1, aborted)) { ok = false; break; }
        fence_after();
        uint32_t x[128];
        float up = 1.f;                       // factor of what was summed so far
        bool lift = false;
        if (any_live) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(x + 32 * c, s_addr + 32 * c);
          tmem_wait_ld();
          const int lim = end - (r.tok0 + t * kSpTile);
          if (__any_sync(0xffffffffu, lim < kSpTile)) {
#pragma unroll
            for (int e = 0; e < 128; ++e) x[e] = e < lim ? x[e] : 0xff800000u;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 128; ++e) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(x[e]));
          const float tile_top = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
          // the reference point moves only when a weight would pass 2^8: rarely, and O is rescaled only then
          if (tile_top > m + 8.f || m == -INFINITY) {
            const float to = fmaxf(m, tile_top);
            up = m == -INFINITY ? 0.f : ex2(m - to);
            lift = t > 0 && to > m;
            m = to;
          }
          const float neg = m == -INFINITY ? 0.f : -m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 128; e += 2) {
            const float a = ex2(fmaf(__uint_as_float(x[e]), scale, neg)), b = ex2(fmaf(__uint_as_float(x[e + 1]), scale, neg));
            sum[(e >> 1) & 3] += a + b;
            x[e >> 1] = pack16<VBF16>(a, b);
          }
          l = l * up + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
        // PV of the tile before has read its P and finished with O
        if (i > 0 && !wait(odone, (i - 1) & 1, aborted)) { ok = false; break; }
        fence_after();
        if (any_live) {
          if (__any_sync(0xffffffffu, lift)) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t y[32];
              const uint32_t o_addr = tmem + lanes + 256 + 128 * (n_run & 1) + 32 * c;
              tmem_ld32(y, o_addr);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * up);
              tmem_st32(o_addr, y);
            }
          }
          tmem_st32(s_addr, x);
          tmem_st32(s_addr + 32, x + 32);
          tmem_wait_st();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull(i & 1));
        if (t == 0 && have_o) { write_o((n_run - 1) & 1); have_o = false; }
      }
      if (!ok) break;
      have_o = true;
      o_live = live;
      o_part = r.part;
      o_m = m;
      o_l = l;
      ++n_run;
    }
    if (ok && have_o && wait(odone, (i - 1) & 1, aborted)) {
      fence_after();
      write_o((n_run - 1) & 1);
    }
  }

  __syncwarp();
  __syncthreads();
  if (*aborted) {
    // what is still on its way must land before the CTA's memory is given up
    if (warp == 0) {
      for (uint32_t n = issued > NS ? issued - NS : 0; n < issued; ++n) {
        wait_lane(full(n % NS), (n / NS) & 1, aborted + 1);
      }
      if (lane == 0) { p.hdr[2] = 1; atomicExch(p.status, 1); }
    } else if (warp == 1) {
      if (lane == 0) commit(final_bar);
      __syncwarp();
      wait_lane(final_bar, 0, aborted + 1);
    }
    __syncthreads();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// Rows of `row_bytes`; a box is 128 bytes of box_rows of them, 128-byte swizzle.
bool make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t row_bytes, uint32_t box_rows, CUtensorMapL2promotion promo) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  const cuuint32_t box[2] = {128, box_rows}, ones[2] = {1, 1};
  return encode_tiled()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promo,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NP, bool VBF16>
int launch(const SpParams& p, const CUtensorMap* maps, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(sp_attend_mma_kernel<NP, VBF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<NP>::kBytes);
    if (e != cudaSuccess) return note_cuda_error(e, "cudaFuncSetAttribute(sp_attend_mma)");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  // set up while the plan still runs; it waits for the plan's end before it reads
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.n_ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<NP>::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sp_attend_mma_kernel<NP, VBF16>, p, maps[0], maps[1], maps[2], maps[3], maps[4]);
  return e == cudaSuccess ? FFA_OK : note_cuda_error(e, "ffa_decode_shared_prefix");
}

}  // namespace

int launch_sp_attend(const SpParams& p, cudaStream_t st) {
  if (!encode_tiled()) return FFA_E_LAUNCH;
  alignas(64) CUtensorMap maps[5];
  const int64_t rows = static_cast<int64_t>(p.n_pages) * kPage, k_bytes = static_cast<int64_t>(p.HKV) * 128;
  const int64_t q_rows = static_cast<int64_t>(p.pieces) * p.B * p.HQ;
  // L2 promotion no wider than one head's row: the neighbouring heads belong to other units
  if (!make_map(&maps[0], p.k, rows, k_bytes, kPage, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
      !make_map(&maps[1], p.r ? p.r : p.k, rows, k_bytes, kPage, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
      !make_map(&maps[2], p.v, rows, 2 * k_bytes, kPage, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
      !make_map(&maps[3], p.qp, q_rows, 128, kSpRows, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
      !make_map(&maps[4], p.qp, q_rows, 128, 8, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return FFA_E_LAUNCH;
  const bool two = p.q_dtype == FFA_BF16, bf = p.v_dtype == FFA_BF16;
  if (two) return bf ? launch<2, true>(p, maps, st) : launch<2, false>(p, maps, st);
  return bf ? launch<3, true>(p, maps, st) : launch<3, false>(p, maps, st);
}

}  // namespace ffa
