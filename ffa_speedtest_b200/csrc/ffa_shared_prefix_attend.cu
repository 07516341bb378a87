// Attention over the runs of the shared-prefix decode (ffa_shared_prefix.cuh) on the fifth-generation tensor cores.
//
// One persistent CTA per SM walks its runs in steps of 128 query rows x 128 tokens:
//
//   S[128 rows, 128 tokens] = sum over pieces of q, base and residual:  Qpiece . K^T    kind::f8f6f4, fp32 in TMEM
//   P = 2^(S * row scale - m)                                                           one row per thread
//   O[128 rows, 128 channels] += P . V                                                  kind::f16, P from TMEM, in pieces
//                                                                                       too where V is bfloat16
//
// K is used as it lies in the cache: q comes as e4m3 pieces (ffa_shared_prefix.cu), and the products of every piece with
// the raw base and residual bytes accumulate into one fp32 tile.  That costs 4 (6) times the fp8 MMAs of one product,
// twice (three times) what a dequantised 16-bit K would, but K never passes through registers.
//
// Bound: per 128 tokens and kv-head 64 KiB arrive, 1.48 us of an SM's share of HBM.  The tensor core needs 16 (24) + 8 MMAs
// of 64 clocks a step, and 8 more with bfloat16 V and more than 64 rows.  The softmax of a row takes 128 exponentials, 1024
// clocks of the special-function unit of a quarter of the SM, and some 600 clocks around them (exponentials by a polynomial
// on the FMA units were tried: half of them so made a step 600 clocks longer).  Measured, with the kernels before and after
// (bf16, 8 kv-heads, 4 query heads to each; in brackets a GPU under sustained load): 8 samples of 32K tokens 38.9 us (39.0)
// for 147 MB: the first K is there after 6.4, then 1.39 a tile of 128 tokens, 3 to write O, 5 for the merge; 16 sequences that
// share nothing 75.9 us (83.2) for 400 MB, 1.45 a tile; 64 samples of 128K 273 us (323): 256 rows are two units, each of which
// walks the prompt, 1.8 a tile, the tensor core busy for 68 % and the power limit at 1.54 GHz; the second walk finds the
// prompt in L2, 839 MB come from HBM.
// One unit of 256 rows (an S and an O for each half, two softmax groups) was tried: it leaves one S buffer to a half, so
// that S, softmax and P V follow one another: the same time there, 1 to 7 us more elsewhere.  S given back as soon as it is
// in registers, P in columns of its own (then there is room for one O only): 3 us more in the smaller cases, nothing gained
// in the largest.
//
// Code: what is executed is fetched cold at every call, and 127 KB of it took 1 to 6 us longer than 86 do, so what runs once
// or rarely is compiled once (the walk over a unit, the long part of a wait) and its loops are not unrolled.
//
// Warps: 0 lists the runs and loads q, K and V; 1 issues the MMAs of S, 2 those of O (two warps, so that the waits of one
// do not keep the other's from the tensor core); 4-7 softmax (TMEM lanes 32 * (warp % 4)).
// A ring of 16 KiB slots holds, tile after tile, K base, K residual, V of the first and of the second page.  S has two
// buffers, for even and odd steps: S of step i+1 is made while the softmax of step i runs.  P overwrites the S that it came
// from.  O has two buffers, for even and odd runs: a run's O is written out while the next run has begun.
// Runs of up to eight query rows (a sequence's own pages) have two small q buffers, larger ones one of 128 rows.  Up to 32
// (64) rows are spread over the four quarters of the TMEM lanes, eight (sixteen) to each, so that all four softmax warps
// have work, and there four lanes share a row (softmax_16): 32 (64) exponentials a lane and not 128.  Up to 64 rows the
// MMAs have M = 64, which takes as long as 128 but less power, and the clock rises.  16 sequences that share nothing, under
// sustained load, with one bfloat16 to a weight: 94.3 us with a row to a lane and M = 128, 92.5 spread, 83.3 with M = 64.
// The second pieces of bfloat16 weights have the lanes eight (sixteen) further on; with 33 to 64 rows their MMA has M = 128.
//
// The line of costs does not depend on the kernel that splits q, nor do K and V: both are begun while that one runs.
//
// Every wait ends after 0.2 s at most: the CTA then leaves its loops, lets its copies and MMAs in flight finish, and
// marks the call, and the merge writes NaN.
#include <cuda.h>

#include "ffa_shared_prefix.cuh"

namespace ffa {
namespace {

constexpr int kThreads = 256;
constexpr int kSlot = 16 * 1024;
constexpr int kPiece = 16 * 1024;             // 128 rows x 128 bytes
constexpr int kRuns = 8;                      // runs listed ahead
constexpr unsigned long long kWaitNs = 200ull * 1000 * 1000;

struct Run {
  int32_t table_row, row0, rows, head;
  int32_t tok0, end, tiles;                   // first token, token that ends the item, tiles (0: no more runs)
  int32_t spread;                             // rows of a run in each 32 TMEM lanes: 8, 16 or 32; 0: up to 8 rows in all
  int64_t part;                               // first row of its partials
};

template <int NP>                             // pieces of q
struct Smem {
  static constexpr int kSlots = NP == 2 ? 11 : 10;
  static constexpr int kOffSmall = NP * kPiece;                         // after [NP] of 128 rows: [2][NP] of 8 rows
  static constexpr int kOffRing = kOffSmall + 2 * NP * 1024;
  static constexpr int kOffRuns = kOffRing + kSlots * kSlot;
  static constexpr int kOffPlan = kOffRuns + kRuns * static_cast<int>(sizeof(Run));    // [12] sums of the warps; [12], [13] first item, its place; the item
  static constexpr int kOffBounds = kOffPlan + 64 + 48;                     // group bounds and prefixes
  static constexpr int kOffBars = kOffBounds + (2 * kSpGroupsNear + 2) * 4;
  // full[slots], empty[slots], sfull[2], sfree[2], pfull[2], ofree[2], qfull[3], qfree[3], runfull[runs], runempty[runs],
  // final[2]
  static constexpr int kBars = 2 * kSlots + 8 + 6 + 2 * kRuns + 2;
  static constexpr int kOffMisc = kOffBars + kBars * 8;                 // TMEM address, abort flag, the same for the last waits
  static constexpr int kBytes = kOffMisc + 16 + 1024;                   // and slack to align to 1024
};
static_assert(Smem<2>::kBytes <= 227 * 1024 && Smem<3>::kBytes <= 227 * 1024, "shared memory of a CTA");
// K of two tiles and V of one have to fit, or the ring could fill up with what is not needed next
static_assert(Smem<3>::kSlots >= 6, "slots of the ring");

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// A lane's wait for the phase of this parity; gives up after kWaitNs, or when another warp of the CTA has.  What a wait that
// does not end at once needs is a call of its own: inlined at every wait the code no longer fits where instructions are held.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, int* abort_flag) {
  unsigned long long t0 = 0;
#pragma unroll 1
  for (int spin = 0;; ++spin) {
    if (try_wait(bar, parity)) return true;
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
__device__ __forceinline__ bool wait_lane(uint32_t bar, uint32_t parity, int* abort_flag) {
  return try_wait(bar, parity) || wait_on(bar, parity, abort_flag);
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

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2, version 1).  K-major: rows of 128 bytes, groups
// of 8 rows 1024 bytes apart.  MN-major (V: channels contiguous, tokens down): 64 channels to a row, the next 64
// channels `lead` bytes on, groups of 8 tokens 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// Instruction descriptor: fp32 accumulator, A and B formats, B transposed (MN-major) or not, N = 128, M = 128 or 64.  With
// M = 64 rows 16 * i .. 16 * i + 15 are the first 16 lanes of quarter i of the TMEM lanes.
__host__ __device__ constexpr uint32_t instr(uint32_t a, uint32_t b, uint32_t b_mn, uint32_t m) {
  return (1u << 4) | (a << 7) | (b << 10) | (b_mn << 16) | ((128u >> 3) << 17) | ((m >> 4) << 24);
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
__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 TMEM lanes x 128 columns: registers 4 * a .. 4 * a + 3 are columns 8 * a + 2 * (lane % 4), + 1 of row lane / 4, then of
// row lane / 4 + 8; the store of 16-bit pairs has columns 4 * a + lane % 4 of the two rows in registers 2 * a, 2 * a + 1.
__device__ __forceinline__ void tmem_ld_16x256(uint32_t (&r)[64], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]),
        "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]),
        "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]),
        "=r"(r[63])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_16x128(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_16x128(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256(uint32_t (&r)[8], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
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
// two at a time: a * s + t, a + b
__device__ __forceinline__ float2 fma2(float2 a, float s, float t) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%5, %5};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(s), "f"(t));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {       // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Weights as the MMA takes them, two tokens to a word.  float16: eleven bits.  bfloat16 has only eight, so there a weight is
// two of them, the leading eight bits (cut off) and the rest, rounded to eight more: sixteen bits.  Up to 64 query rows the
// rest has rows of the MMA to itself that were idle; with more the MMAs of P V are issued twice.  One piece is faster,
// 38.3 to 39.0 us (8 samples of 32K), 40.1 to 41.6 (ragged prompts), 74.3 to 75.8 (16 private) and, with 128 rows, 260 to 296
// (64 samples of 128K, all tiles counted alike); but its rounding is as large as that of a bfloat16 output, and larger than
// that of any other.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float2 w) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(w.y), "f"(w.x));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(w.y), "f"(w.x));
  return r;
}
__device__ __forceinline__ void two_pieces(float2 w, uint32_t& lead, uint32_t& rest) {
  const uint32_t x = __float_as_uint(w.x), y = __float_as_uint(w.y);
  lead = __byte_perm(x, y, 0x7632);
  rest = pack16<true>(add2(w, make_float2(__uint_as_float((x & 0xffff0000u) ^ 0x80000000u), __uint_as_float((y & 0xffff0000u) ^ 0x80000000u))));
}

// What a softmax thread knows of a query row.
struct Row {
  float m = -INFINITY, l = 0.f;               // reference point (log2 units), sum of the weights so far
  float scale = 0.f;
  int end = 0;                                // token that ends it
  bool live = false;
};
// Takes a tile's maximum in.  The reference point moves only when a weight would pass 2^kMost: rarely, and O is rescaled
// only then.  Returns the factor of what was summed before.
//
// float16 has five bits of exponent, so the largest weight is put at 2^7 (2^15 at most, 65504 is the largest number):
// weights down to 2^-21 of it keep all eleven bits, and one below is off by at most 2^-32 of it.  With the largest at 2^0 the
// weights of tokens 25 bits below one (an attention sink) were off by half, and l has them unrounded.  At 2^9 and 2^11, with
// less room to rise before O is rescaled, 32 samples of 16K took 47.7 and 48.9 us, at 2^7 46.9, at 2^0 47.0.
//
// bfloat16 has the range.  There the largest weight is put at 2^0.3 and not at 1, whose second piece would be zero: a value
// of infinity times it is NaN.
template <bool VBF16>
__device__ __forceinline__ float take_maximum(Row& row, float top, bool have_o, bool& lift) {
  constexpr float kTop = VBF16 ? 0.3f : 7.f, kMost = VBF16 ? 8.f : 15.f;
  top = row.live ? top * row.scale : 0.f;     // the other rows' S is whatever lay in shared memory
  float up = 1.f;
  if (!(top <= row.m + kMost) || row.m == -INFINITY) {
    top -= kTop;
    const float to = top > row.m || top != top ? top : row.m;        // NaN stays and makes the row NaN
    up = row.m == -INFINITY ? 0.f : ex2(row.m - to);
    lift |= have_o && !(to <= row.m);
    row.m = to;
  }
  return up;
}

// S of a tile to P, in place; a row to a lane.  Tile begins at token `at`; bring_down(factor) rescales O.  16 tokens of P are
// eight columns, with two pieces eight and eight.
template <bool VBF16, typename F>
__device__ __forceinline__ bool softmax_32(Row& row, uint32_t s_addr, int at, bool have_o, const F& bring_down) {
  const int lim = row.end - at;
  const bool cut = __any_sync(0xffffffffu, lim < kSpTile);
  uint32_t x[32], y[32], z[32];               // three quarters of S at a time: the last two are read twice
  float top = -INFINITY;
  if (!cut) {
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    auto tops_of = [&](const uint32_t* s) {
#pragma unroll
      for (int i = 0; i < 32; i += 8)
#pragma unroll
        for (int j = 0; j < 4; ++j) tops[j] = max3(tops[j], __uint_as_float(s[i + j]), __uint_as_float(s[i + j + 4]));
    };
    tmem_ld32(x, s_addr + 64);
    tmem_ld32(y, s_addr + 96);
    tmem_wait_ld();
    tmem_ld32(z, s_addr);
    tops_of(x);
    tmem_ld32(x, s_addr + 32);
    tops_of(y);
    tmem_wait_ld();
    tmem_ld32(y, s_addr + 64);
    tops_of(z);
    tops_of(x);
    top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
  } else {
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t y[32];
      tmem_ld32(y, s_addr + 32 * c);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (32 * c + i < lim) top = max3(top, __uint_as_float(y[i]), __uint_as_float(y[i]));
    }
  }
  bool lift = false;
  const float up = take_maximum<VBF16>(row, top, have_o, lift);
  if (__any_sync(0xffffffffu, lift) && !bring_down(up)) return false;
  const float neg = row.m == -INFINITY ? 0.f : -row.m;
  float2 sum = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
  if (!cut) {
    // quarter c of P, over what has been read of S
    auto weights = [&](const uint32_t* s, int c) {
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        float2 a = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), row.scale, neg);
        float2 b = fma2(make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), row.scale, neg);
        a = make_float2(ex2(a.x), ex2(a.y));
        b = make_float2(ex2(b.x), ex2(b.y));
        sum = add2(sum, a);
        sum1 = add2(sum1, b);
        if (VBF16) {
          const int j = i / 16 * 16 + i % 16 / 2;
          two_pieces(a, w[j], w[8 + j]);
          two_pieces(b, w[j + 1], w[8 + j + 1]);
        } else {
          w[i / 2] = pack16<false>(a);
          w[i / 2 + 1] = pack16<false>(b);
        }
      }
      if (VBF16) tmem_st32(s_addr + 32 * c, w);
      else tmem_st16(s_addr + 16 * c, w);
    };
    weights(z, 0);
    tmem_ld32(z, s_addr + 96);
    weights(x, 1);
    tmem_wait_ld();
    weights(y, 2);
    weights(z, 3);
  } else {
    // P of 32 tokens takes 16 or 32 columns, so it never reaches an S that is still to be read
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t y[32];
      tmem_ld32(y, s_addr + 32 * c);
      tmem_wait_ld();
#pragma unroll
      for (int i0 = 0; i0 < 32; i0 += 16) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float2 a = fma2(make_float2(__uint_as_float(y[i0 + i]), __uint_as_float(y[i0 + i + 1])), row.scale, neg);
          a = make_float2(32 * c + i0 + i < lim ? ex2(a.x) : 0.f, 32 * c + i0 + i + 1 < lim ? ex2(a.y) : 0.f);
          sum = add2(sum, a);
          if (VBF16) two_pieces(a, w[i / 2], w[8 + i / 2]);
          else y[(i0 + i) / 2] = pack16<false>(a);
        }
        if (VBF16) tmem_st16(s_addr + 32 * c + i0, w);
      }
      if (!VBF16) tmem_st16(s_addr + 16 * c, y);
    }
  }
  row.l = row.l * up + ((sum.x + sum.y) + (sum1.x + sum1.y));
  tmem_wait_st();
  return true;
}

// The same for up to 8 * H rows in the warp's first 16 TMEM lanes, four lanes of the warp to a row: lane i has columns
// 8 * a + 2 * (i % 4), + 1 of rows i / 4 and i / 4 + 8.  A warp then works out 32 * H exponentials a lane, not 128.  The second
// piece of bfloat16 weights goes to the TMEM lanes 8 * H further on, and so does its part of O.
template <int H, bool VBF16, typename F>
__device__ __forceinline__ bool softmax_16(Row (&row)[2], uint32_t s_addr, int at, bool have_o, const F& bring_down) {
  const int lane = threadIdx.x & 31, col0 = 2 * (lane & 3);
  uint32_t x[64];
  tmem_ld_16x256(x, s_addr);
  tmem_wait_ld();
  const int lim0 = row[0].end - at, lim1 = H > 1 ? row[1].end - at : kSpTile;
  if (__any_sync(0xffffffffu, min(lim0, lim1) < kSpTile)) {
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (8 * (i >> 2) + (i & 1) + col0 >= ((i & 2) ? lim1 : lim0)) x[i] = 0xff800000u;
  }
  bool lift = false;
  float up[2] = {1.f, 1.f};
#pragma unroll
  for (int h = 0; h < H; ++h) {
    float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int a = 0; a < 16; ++a) tops[a & 1] = max3(tops[a & 1], __uint_as_float(x[4 * a + 2 * h]), __uint_as_float(x[4 * a + 2 * h + 1]));
    float top = max3(tops[0], tops[1], tops[1]);
    const float y = __shfl_xor_sync(0xffffffffu, top, 1);
    top = max3(top, y, y);
    const float z = __shfl_xor_sync(0xffffffffu, top, 2);
    up[h] = take_maximum<VBF16>(row[h], max3(top, z, z), have_o, lift);
  }
  if (__any_sync(0xffffffffu, lift)) {
    const float a = __shfl_sync(0xffffffffu, up[0], (lane & 7) * 4), b = __shfl_sync(0xffffffffu, up[H - 1], (lane & 7) * 4);
    if (!bring_down(lane & 8 ? b : a)) return false;
  }
  float neg[H];
  float2 sum[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    neg[h] = row[h].m == -INFINITY ? 0.f : -row[h].m;
    sum[h] = make_float2(0.f, 0.f);
  }
  auto weight = [&](const uint32_t* s, int h, int a) {
    const int i = 4 * a + 2 * h;
    float2 v = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), row[h].scale, neg[h]);
    v = make_float2(ex2(v.x), ex2(v.y));
    sum[h] = add2(sum[h], v);
    return v;
  };
  if (H == 2 && VBF16) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {    // 64 tokens at a time
      uint32_t w[16], rest[16];
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int a = 0; a < 8; ++a) two_pieces(weight(x, h, 8 * part + a), w[2 * a + h], rest[2 * a + h]);
      tmem_st_16x128(s_addr + 32 * part, w);
      tmem_st_16x128(s_addr + 32 * part + (16u << 16), rest);
    }
  } else {
    uint32_t w[32];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int a = 0; a < 16; ++a) {
        if (VBF16) two_pieces(weight(x, h, a), w[2 * a], w[2 * a + 1]);
        else w[2 * a + h] = pack16<false>(weight(x, h, a));
        if (!VBF16 && H == 1) w[2 * a + 1] = 0u;
      }
    tmem_st_16x128(s_addr, w);
  }
#pragma unroll
  for (int h = 0; h < H; ++h) row[h].l = row[h].l * up[h] + (sum[h].x + sum[h].y);
  tmem_wait_st();
  return true;
}

// Sum over the CTA's threads before this one; `total` gets the sum over all.  s: one entry per warp.
__device__ __forceinline__ int cta_exclusive(int x, volatile int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 31) s[warp] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int y = s[w];
    if (w < warp) before += y;
    total += y;
  }
  return before + inc - x;
}

template <int NP, bool VBF16>
__global__ void __launch_bounds__(kThreads, 1) sp_attend_mma_kernel(const __grid_constant__ SpParams p,
                                                                    const __grid_constant__ CUtensorMap map_k,
                                                                    const __grid_constant__ CUtensorMap map_r,
                                                                    const __grid_constant__ CUtensorMap map_v,
                                                                    const __grid_constant__ CUtensorMap map_q,
                                                                    const __grid_constant__ CUtensorMap map_q8) {
  using L = Smem<NP>;
  constexpr uint32_t NS = L::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // uniform for the compiler too: MMAs issued under a branch that it takes for divergent cost 100 clocks and more each
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, cta = blockIdx.x;
  const uint32_t s_q = smem_u32(smem), s_ring = s_q + L::kOffRing, bars = s_q + L::kOffBars;
  Run* const runs = reinterpret_cast<Run*>(smem + L::kOffRuns);
  volatile int* const s_plan = reinterpret_cast<volatile int*>(smem + L::kOffPlan);
  SpItem* const s_first = reinterpret_cast<SpItem*>(smem + L::kOffPlan + 64);
  int* const s_bounds = reinterpret_cast<int*>(smem + L::kOffBounds);
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kOffMisc);
  int* const aborted = reinterpret_cast<int*>(smem + L::kOffMisc + 4);
  auto full = [&](uint32_t s) { return bars + 8 * s; };
  auto empty = [&](uint32_t s) { return bars + 8 * (NS + s); };
  const uint32_t rest = bars + 16 * NS;
  auto sfull = [&](uint32_t i) { return rest + 8 * i; };
  auto sfree = [&](uint32_t i) { return rest + 16 + 8 * i; };
  auto pfull = [&](uint32_t i) { return rest + 32 + 8 * i; };
  auto ofree = [&](uint32_t i) { return rest + 48 + 8 * i; };
  // q buffers: 0 the large one, 1 and 2 the small ones
  auto qfull = [&](uint32_t i) { return rest + 64 + 8 * i; };
  auto qfree = [&](uint32_t i) { return rest + 88 + 8 * i; };
  auto final_bar = [&](uint32_t i) { return rest + 112 + 8 * i; };
  auto runfull = [&](uint32_t i) { return rest + 128 + 8 * i; };
  auto runempty = [&](uint32_t i) { return rest + 128 + 8 * (kRuns + i); };
  auto q_buffer = [&](uint32_t i) { return i == 0 ? s_q : s_q + L::kOffSmall + (i - 1) * NP * 1024; };

  // what the line is worked out from, on its way before anything else
  const int tid = threadIdx.x;
  const int first_len = tid < p.B ? p.seq_lens[tid] : 0;
  {
    // the block table into L2, a line to a thread: its entries are asked for once the line is known
    const int64_t at = (static_cast<int64_t>(cta) * kThreads + tid) * 32;
    if (at < static_cast<int64_t>(p.B - 1) * p.bt_stride + p.cols) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p.bt + at));
  }
  bool falls = false;                         // a bound below the one before it
#pragma unroll 1
  for (int g = tid; g <= p.NG; g += kThreads) {
    const int start = p.group_start[g];
    falls |= g < p.NG && p.group_start[g + 1] < start;
    if (g <= kSpGroupsNear) s_bounds[g] = min(max(start, 0), p.B);
    if (g < min(p.NG, kSpGroupsNear)) s_bounds[kSpGroupsNear + 1 + g] = min(max(p.prefix_pages[g], 0), p.cols);
  }
  if (warp == 2 && lane == 0) {
#pragma unroll 1
    for (uint32_t i = 0; i < 2 * NS; ++i) mbar_init(bars + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull(i), 1);
      mbar_init(sfree(i), 1);
      mbar_init(pfull(i), 4);
      mbar_init(ofree(i), 4);
      mbar_init(final_bar(i), 1);
    }
    for (int i = 0; i < kRuns; ++i) { mbar_init(runfull(i), 1); mbar_init(runempty(i), 1 + 1 + 4); }
    for (int i = 0; i < 3; ++i) { mbar_init(qfull(i), 1); mbar_init(qfree(i), 1); }
    *aborted = 0;
    aborted[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(s_q + L::kOffMisc) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int n_groups = __syncthreads_or(falls) ? 0 : p.NG, n_items = p.B + n_groups;

  // ---- the line: its length, and the item that this CTA's range begins in ----
  const SpBounds bounds{p, n_groups, s_bounds, s_bounds + kSpGroupsNear + 1};
  SpItem mine{};
  int W = 0, my_cost = 0, my_at = 0, first_sum = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < n_items; i0 += kThreads) {
    const int i = i0 + tid;
    SpItem x{};
    if (i < n_items) x = sp_item(p, bounds, i, i0 == 0 ? first_len : i < p.B ? p.seq_lens[i] : 0);
    const int cost = x.units * sp_unit_cost(x.tiles, sp_tile_cost(x.rows));
    int sum;
    const int at = W + cta_exclusive(cost, s_plan, sum);
    if (i0 == 0) { mine = x; my_cost = cost; my_at = at; first_sum = sum; }
    if (cta == 0 && i < n_items) {            // for the merge
      if (i < p.B) p.sequences[i] = SpSequence{at, x.tiles, x.group, 0, 0, 0, {0, 0}};
      else p.groups[i - p.B] = SpGroup{at, x.tiles, x.first, x.rows};
    }
    W += sum;
  }
  if (cta == 0 && tid == 0) p.hdr[0] = W;
  const int n_used = sp_ctas(W, p.n_ctas);
  const bool idle = cta >= n_used || W == 0;
  const int x0 = sp_first(cta, W, n_used), x1 = sp_first(cta + 1, W, n_used);
  if (!idle) {
    if (my_cost > 0 && my_at <= x0 && x0 < my_at + my_cost) { *s_first = mine; s_plan[12] = tid; s_plan[13] = my_at; }
    int before = first_sum;
#pragma unroll 1
    for (int i0 = kThreads; i0 < n_items && before <= x0; i0 += kThreads) {
      const int i = i0 + tid;
      SpItem x{};
      if (i < n_items) x = sp_item(p, bounds, i, i < p.B ? p.seq_lens[i] : 0);
      const int cost = x.units * sp_unit_cost(x.tiles, sp_tile_cost(x.rows));
      int sum;
      const int at = before + cta_exclusive(cost, s_plan, sum);
      before += sum;
      if (cost > 0 && at <= x0 && x0 < at + cost) { *s_first = x; s_plan[12] = i; s_plan[13] = at; }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;           // columns: S0 0, S1 128, O0 256, O1 384

  if (cta == 0 && warp >= 4) {                // these warps have nothing to do yet
#pragma unroll 1
    for (int b = tid - 128; b < p.B; b += kThreads - 128) {
      const int g = p.sequences[b].group_at;  // the group's number so far
      const SpGroup gr = g >= 0 ? p.groups[g] : SpGroup{0, 0, 0, 0};
      p.sequences[b].group_at = gr.at;
      // one that holds nothing has no partials, whatever its q is (the padding of a batch)
      p.sequences[b].group_tiles = p.seq_lens[b] > 0 ? gr.tiles : 0;
      p.sequences[b].group_first = gr.first;
      p.sequences[b].group_rows = gr.rows;
    }
  }

  // The next run for an MMA warp, in order; false at the end (or when the CTA gave up).
  uint32_t runs_read = 0;
  auto next_run = [&](Run& r) -> bool {
    const uint32_t i = runs_read % kRuns;
    if (!wait(runfull(i), (runs_read / kRuns) & 1, aborted)) return false;
    r = runs[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(runempty(i));
    ++runs_read;
    return r.tiles > 0;
  };

  const uint32_t nk = p.r ? 2 : 1;            // slots of a K tile
  uint32_t issued = 0;                        // warp 0: slots filled so far
  uint32_t q_large = 0, q_small = 0;          // warps 0 and 1: runs so far with the large and with a small q buffer
  if (idle) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
  } else if (warp == 0) {
    // ---- run list, q, K and V ----
    // waits for the next slot to be free
    auto take = [&](uint32_t n) -> bool { return n < NS || wait(empty(n % NS), (n / NS - 1) & 1, aborted); };
    bool ok = true;
    uint32_t listed = 0;
    auto list = [&](const Run& r) -> bool {
      const uint32_t i = listed % kRuns, round = listed / kRuns;
      if (round > 0 && !wait(runempty(i), (round - 1) & 1, aborted)) return false;
      if (lane == 0) {
        runs[i] = r;
        mbar_arrive(runfull(i));
      }
      __syncwarp();
      ++listed;
      return true;
    };
    auto load_q = [&](const Run& r) -> bool {
      const bool small = r.spread == 0;
      const uint32_t qb = small ? 1 + (q_small & 1) : 0, round = small ? q_small >> 1 : q_large;
      if (round > 0 && !wait(qfree(qb), (round - 1) & 1, aborted)) return false;
      if (small) ++q_small; else ++q_large;
      if (listed == 1) {                      // before the first q: the kernel that splits it has ended
        asm volatile("griddepcontrol.wait;\n" ::: "memory");
        asm volatile("fence.proxy.async.global;\n" ::: "memory");   // its pieces were written by ordinary stores
      }
      if (elect()) {
        const int rows_head = p.B * p.G;
        const uint32_t dst = q_buffer(qb), step = small ? 1024 : kPiece, bar = qfull(qb);
        if (r.spread == 32) {
          mbar_expect_tx(bar, NP * kPiece);
#pragma unroll 1
          for (int piece = 0; piece < NP; ++piece)
            tma_load(dst + piece * step, &map_q, 0, (piece * p.HKV + r.head) * rows_head + r.row0, bar);
        } else {
          // eight rows at a time, eight or sixteen to a quarter of the 64
          const int boxes = (r.rows + 7) / 8;
          mbar_expect_tx(bar, NP * boxes * 1024);
#pragma unroll 1
          for (int piece = 0; piece < NP; ++piece)
#pragma unroll 1
            for (int i = 0; i < boxes; ++i)
              tma_load(dst + piece * step + i * (r.spread == 16 ? 1024 : 2048), &map_q8, 0,
                       (piece * p.HKV + r.head) * rows_head + r.row0 + 8 * i, bar);
        }
      }
      __syncwarp();
      return true;
    };
    // q is asked for after the run's first tile, which need not wait until the pieces of q are there or a q buffer is free
    auto load = [&](const Run& r) -> bool {
      const int32_t* row = p.bt + static_cast<int64_t>(r.table_row) * p.bt_stride;
      const int col0 = r.tok0 / kPage, cols = (r.end + kPage - 1) / kPage;         // cols <= p.cols
      auto page_at = [&](int col) {
        const int y = col < cols ? row[col] : -1;
        return y >= 0 && y < p.n_pages ? y : -1;       // TMA reads zeros at negative rows
      };
      int ids = page_at(col0 + lane), ids_next = page_at(col0 + 32 + lane);
#pragma unroll 1
      for (int t = 0; t < r.tiles; ++t) {
        if (t > 0 && (t & 15) == 0) { ids = ids_next; ids_next = page_at(col0 + 2 * t + 32 + lane); }
        const int n_pages = min(2, cols - (col0 + 2 * t));
        const int y0 = __shfl_sync(0xffffffffu, ids, (2 * t) & 31) * kPage, y1 = __shfl_sync(0xffffffffu, ids, (2 * t + 1) & 31) * kPage;
        // K base and K residual: a box of 64 tokens x 128 bytes for either page; V of either page: 64 tokens x 2 x 128 bytes
        if (!take(issued) || (nk > 1 && !take(issued + 1))) return false;
        const uint32_t s0 = issued % NS, s1 = (issued + 1) % NS;
        if (elect()) {
          const uint32_t d0 = s_ring + s0 * kSlot, d1 = s_ring + s1 * kSlot;
          mbar_expect_tx(full(s0), n_pages * 8192);
          tma_load(d0, &map_k, r.head * 128, y0, full(s0));
          if (n_pages > 1) tma_load(d0 + 8192, &map_k, r.head * 128, y1, full(s0));
          if (nk > 1) {
            mbar_expect_tx(full(s1), n_pages * 8192);
            tma_load(d1, &map_r, r.head * 128, y0, full(s1));
            if (n_pages > 1) tma_load(d1 + 8192, &map_r, r.head * 128, y1, full(s1));
          }
        }
        issued += nk;
        if (!take(issued) || (n_pages > 1 && !take(issued + 1))) return false;
        const uint32_t s2 = issued % NS, s3 = (issued + 1) % NS;
        if (elect()) {
          mbar_expect_tx(full(s2), 16384);
          tma_load_3d(s_ring + s2 * kSlot, &map_v, 0, y0, 2 * r.head, full(s2));
          if (n_pages > 1) {
            mbar_expect_tx(full(s3), 16384);
            tma_load_3d(s_ring + s3 * kSlot, &map_v, 0, y1, 2 * r.head, full(s3));
          }
        }
        issued += n_pages;
        if (t == 0 && !load_q(r)) return false;
      }
      return true;
    };
    int place = s_plan[13];
    // the runs of one item
    auto runs_of = [&](const SpItem& it, bool own) -> bool {
      const int tile = sp_tile_cost(it.rows), unit = sp_unit_cost(it.tiles, tile), before = x0 - place - kSpBegin - (it.tiles - 1) * tile;
      int k = before <= 0 ? 0 : (before - 1) / unit + 1;                          // units that end before x0 are other CTAs'
      int block = k / p.HKV, head = k - block * p.HKV;
#pragma unroll 1
      for (; k < it.units; ++k) {
        const int first = place + k * unit + kSpBegin;                            // where tile 0 stands
        if (first >= x1) break;
        const int t0 = first >= x0 ? 0 : (x0 - first - 1) / tile + 1;
        const int t1 = min(it.tiles, (x1 - first - 1) / tile + 1);
        Run r;
        r.table_row = it.first;
        r.head = head;
        r.row0 = it.first * p.G + block * kSpRows;
        r.rows = min(kSpRows, it.rows - block * kSpRows);
        r.tok0 = it.page0 * kPage + t0 * kSpTile;
        r.end = it.end;
        r.tiles = t1 - t0;
        r.spread = r.rows <= 8 ? 0 : r.rows <= 32 ? 8 : r.rows <= 64 ? 16 : 32;
        r.part = sp_part_row(p, own, r.row0, r.rows, head, cta);
        if (!list(r) || !load(r)) return false;
        if (++head == p.HKV) { head = 0; ++block; }
      }
      place += it.units * unit;
      return true;
    };
    const int first_item = s_plan[12];
    SpItem it;
#pragma unroll 1
    for (int i0 = first_item; ok && i0 < n_items && place < x1; i0 += i0 == first_item ? 1 : 32) {
      // the first item by itself: it is known; then 32, one to a lane; one that has tiles after the other
      const int i = i0 + lane;
      SpItem x{};
      if (i0 == first_item) { if (lane == 0) x = *s_first; }
      else if (i < n_items) x = sp_item(p, bounds, i, i < p.B ? p.seq_lens[i] : 0);
      uint32_t todo = __ballot_sync(0xffffffffu, x.tiles > 0 && x.units > 0);
#pragma unroll 1
      while (todo && ok && place < x1) {
        const int from = __ffs(todo) - 1;
        todo &= todo - 1;
        it.first = __shfl_sync(0xffffffffu, x.first, from);
        it.rows = __shfl_sync(0xffffffffu, x.rows, from);
        it.page0 = __shfl_sync(0xffffffffu, x.page0, from);
        it.end = __shfl_sync(0xffffffffu, x.end, from);
        it.tiles = __shfl_sync(0xffffffffu, x.tiles, from);
        it.units = __shfl_sync(0xffffffffu, x.units, from);
        ok = runs_of(it, i0 + from < p.B);
      }
    }
    if (ok) {
      Run none{};
      list(none);
    }
  } else if (warp == 1) {
    // ---- S = q K^T ----
    uint32_t pos = 0, e = 0;                  // slots of the tiles before the present one, steps before it
    Run r;
    bool ok = true;
    while (ok && next_run(r)) {
      const bool small = r.spread == 0;
      const uint32_t qb = small ? 1 + (q_small & 1) : 0;
      if (!wait(qfull(qb), (small ? q_small >> 1 : q_large) & 1, aborted)) break;
      if (small) ++q_small; else ++q_large;
      const uint32_t idesc = instr(0, p.fp8 == FFA_E4M3 ? 0 : 1, 0, r.spread == 32 ? 128 : 64);
      const uint64_t dq = desc(q_buffer(qb), 16);
      const uint32_t q_step = (small ? 1024 : kPiece) >> 4;
#pragma unroll 1
      for (int t = 0; t < r.tiles; ++t, ++e) {
        const uint32_t s0 = pos % NS, s1 = (pos + 1) % NS, g = e & 1;
        if (!wait(full(s0), (pos / NS) & 1, aborted)) { ok = false; break; }
        if (nk > 1 && !wait(full(s1), ((pos + 1) / NS) & 1, aborted)) { ok = false; break; }
        if (e >= 2 && !wait(sfree(g), ((e >> 1) - 1) & 1, aborted)) { ok = false; break; }
        fence_after();
        if (elect()) {
          const uint64_t dk0 = desc(s_ring + s0 * kSlot, 16), dk1 = desc(s_ring + s1 * kSlot, 16);
          const uint32_t d = tmem + 128 * g;
#pragma unroll
          for (int piece = 0; piece < NP; ++piece)
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_fp8(d, dq + piece * q_step + 2 * k, dk0 + 2 * k, idesc, piece + k > 0);
          if (nk > 1) {
#pragma unroll
            for (int piece = 0; piece < NP; ++piece)
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_fp8(d, dq + piece * q_step + 2 * k, dk1 + 2 * k, idesc, 1);
          }
          commit(sfull(g));
          commit(empty(s0));
          if (nk > 1) commit(empty(s1));
          if (t == r.tiles - 1) commit(qfree(qb));
        }
        __syncwarp();
        pos += nk + (r.end - (r.tok0 + t * kSpTile) > kPage ? 2 : 1);
      }
    }
  } else if (warp == 2) {
    // ---- O += P V ----
    uint32_t pos = 0, e = 0, n_run = 0;
    Run r;
    bool ok = true;
    while (ok && next_run(r)) {
      const uint32_t o = n_run & 1, d = tmem + 256 + 128 * o;
      const uint32_t type = VBF16 ? 1 : 0, idesc = instr(type, type, 1, r.spread == 32 || (VBF16 && r.spread == 16) ? 128 : 64);
      const bool wide = VBF16 && r.spread == 32;
      if (n_run >= 2 && !wait(ofree(o), ((n_run >> 1) - 1) & 1, aborted)) break;
      ++n_run;
#pragma unroll 1
      for (int t = 0; t < r.tiles && ok; ++t, ++e) {
        const int valid = min(kSpTile, r.end - (r.tok0 + t * kSpTile)), pages = valid > kPage ? 2 : 1;
        const uint32_t g = e & 1;
        pos += nk;
#pragma unroll 1
        for (int i = 0; i < pages && ok; ++i) {
          const uint32_t n = pos + i, v = s_ring + n % NS * kSlot;
          if (!wait(full(n % NS), (n / NS) & 1, aborted)) { ok = false; break; }
          const int here = valid - i * kPage;
          if (here < kPage && here % 16) {
            // tokens past the end of the sequence: whatever their V holds, 0 * V has to be 0
#pragma unroll 1
            for (int x = lane; x < (16 - here % 16) * 16; x += 32) {
              const int row = here + x / 16, h = (x >> 3) & 1, ck = x & 7;
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(v + h * 8192 + row * 128 + ck * 16), "r"(0) : "memory");
            }
            fence_async();
            __syncwarp();
          }
        }
        if (!ok || !wait(pfull(g), (e >> 1) & 1, aborted)) { ok = false; break; }
        fence_after();
        if (elect()) {
          const uint32_t a = tmem + 128 * g;
#pragma unroll 1
          for (int i = 0; i < pages; ++i) {
            const uint64_t dv = desc(s_ring + (pos + i) % NS * kSlot, 8192);
            const int ks = min(4, (valid - i * kPage + 15) / 16);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k < ks) {
                const uint32_t p0 = a + (32 * i + 8 * k) * (wide ? 2 : 1);
                mma_16_tmem(d, p0, dv + 128 * k, idesc, t > 0 || i + k > 0);
                if (wide) mma_16_tmem(d, p0 + 8, dv + 128 * k, idesc, 1);
              }
          }
          commit(sfree(g));
          for (int i = 0; i < pages; ++i) commit(empty((pos + i) % NS));
        }
        __syncwarp();
        pos += pages;
      }
    }
  } else if (warp >= 4) {
    // ---- softmax ----
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t e = 0, n_run = 0;
    // rows of a run in this quarter: lanes for them (a row to a lane with 32, else four lanes to each), first, number
    auto rows_per = [&](int spread) { return spread ? spread : 8; };
    auto rows_here = [&](int spread, int rows) { return spread || quarter == 0 ? min(rows_per(spread), rows - quarter * rows_per(spread)) : 0; };
    // writes the O of the run before and gives the run back
    auto write_o = [&]() {
      const uint32_t n = n_run - 1;
      const Run& done = runs[n % kRuns];
      const int per = rows_per(done.spread), rows = done.rows, here = rows_here(done.spread, rows), first = quarter * per;
      const uint32_t o_addr = lanes + 256 + 128 * (n & 1);
      if (here > 0) {
        if (per == 32) {
          float4* const dst = p.part_o + 32 * done.part + first + lane;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t x[32];
            tmem_ld32(x, o_addr + 32 * c);
            tmem_wait_ld();
            if (lane < here)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                dst[static_cast<int64_t>(8 * c + i) * rows] = make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]),
                                                                          __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3]));
          }
        } else {
          // four lanes to a row, two channels of every eight to a lane; with bfloat16 weights O of the second pieces is added
          float2* const dst = reinterpret_cast<float2*>(p.part_o + 32 * done.part + first + (lane >> 2)) + (lane & 1);
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t x[8], y[8];
            tmem_ld_16x256(x, o_addr + 16 * c);
            if (VBF16 && per == 16) tmem_ld_16x256(y, o_addr + 16 * c + (16u << 16));
            tmem_wait_ld();
            if (VBF16) {
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + __uint_as_float(per == 16 ? y[i] : x[i ^ 2]));
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2)
              if ((lane >> 2) + 4 * (i & 2) < here)
                dst[static_cast<int64_t>(4 * c + 2 * (i >> 2) + ((lane >> 1) & 1)) * 2 * rows + 8 * (i & 2)] =
                    make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ofree(n & 1));
        mbar_arrive(runempty(n % kRuns));
      }
    };
    bool ok = true;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    for (;;) {
      if (!wait(runfull(n_run % kRuns), (n_run / kRuns) & 1, aborted)) break;
      const Run& r = runs[n_run % kRuns];
      const bool more = r.tiles > 0;
      if (!more && n_run == 0) break;
      const int per = rows_per(r.spread);
      const bool any_live = rows_here(r.spread, r.rows) > 0;
      Row row[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = per == 32 ? lane : (lane >> 2) + 8 * h;
        row[h] = Row{};
        row[h].live = j < rows_here(r.spread, r.rows) && (h == 0 || per == 16);
        row[h].end = r.end;
        if (row[h].live) {
          const int at = r.row0 + quarter * per + j;
          row[h].scale = p.q_scale[static_cast<int64_t>(r.head) * p.B * p.G + at];
          row[h].end = min(r.end, p.seq_lens[at / p.G]);
        }
      }
      // after the last run once more, for its O
#pragma unroll 1
      for (int t = 0; t < max(r.tiles, 1); ++t, ++e) {
        const uint32_t g = e & 1, s_addr = lanes + 128 * g;
        if (more && !wait(sfull(g), (e >> 1) & 1, aborted)) { ok = false; break; }
        fence_after();
        // PV of the step before is done: O may be brought down
        bool waited = false;
        auto pv_done = [&]() -> bool {
          if (e > 0 && !waited && !wait(sfree(g ^ 1), ((e - 1) >> 1) & 1, aborted)) return false;
          waited = true;
          fence_after();
          return true;
        };
        // O is rescaled by a factor per row, a row to a lane
        auto bring_down = [&](float up) -> bool {
          if (!pv_done()) return false;
          const uint32_t o_addr = lanes + 256 + 128 * (n_run & 1);
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t y[16];
            tmem_ld16(y, o_addr + 16 * c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * up);
            tmem_st16(o_addr + 16 * c, y);
          }
          return true;
        };
        if (any_live) {
          const int at = r.tok0 + t * kSpTile;
          if (per == 32) ok = softmax_32<VBF16>(row[0], s_addr, at, t > 0, bring_down);
          else if (per == 8) ok = softmax_16<1, VBF16>(row, s_addr, at, t > 0, bring_down);
          else ok = softmax_16<2, VBF16>(row, s_addr, at, t > 0, bring_down);
        }
        if (!ok || !pv_done()) { ok = false; break; }
        fence_before();
        __syncwarp();
        if (more && lane == 0) mbar_arrive(pfull(g));
        if (t == 0 && n_run > 0) write_o();
      }
      if (!ok || !more) break;
      // maxima and sums are written now, O when the next run has begun
      if (per != 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          row[h].l += __shfl_xor_sync(0xffffffffu, row[h].l, 1);
          row[h].l += __shfl_xor_sync(0xffffffffu, row[h].l, 2);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = per == 32 ? lane : (lane >> 2) + 8 * h;
        if (row[h].live && (per == 32 || (lane & 3) == 0)) p.part_ml[r.part + quarter * per + j] = make_float2(row[h].m, row[h].l);
      }
      ++n_run;
    }
  }

  __syncwarp();
  __syncthreads();
  if (*aborted) {
    // what is still on its way must land before the CTA's memory is given up: slots of the ring, and each q buffer's last load
    if (warp == 0) {
      if (q_large > 0) wait_lane(qfull(0), (q_large - 1) & 1, aborted + 1);
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t n = (q_small + 1 - i) / 2;                                  // the small buffers take turns
        if (n > 0) wait_lane(qfull(1 + i), (n - 1) & 1, aborted + 1);
      }
      for (uint32_t n = issued > NS ? issued - NS : 0; n < issued; ++n) wait_lane(full(n % NS), (n / NS) & 1, aborted + 1);
      if (lane == 0) { p.hdr[1] = 1; atomicExch(p.status, 1); }
    } else if (warp == 1) {
      if (elect()) commit(final_bar(0));
      __syncwarp();
      wait_lane(final_bar(0), 0, aborted + 1);
    } else if (warp == 2) {
      if (elect()) commit(final_bar(1));
      __syncwarp();
      wait_lane(final_bar(1), 0, aborted + 1);
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

// Rows of `row_bytes`; a box is 128 bytes of box_rows of them, 128-byte swizzle.  With `chunks` the box has that many
// 128-byte pieces of every row, piece by piece.
bool make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t row_bytes, uint32_t box_rows, CUtensorMapL2promotion promo,
              uint32_t chunks = 0) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(chunks ? 128 : row_bytes), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(row_bytes / 128)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_bytes), 128};
  const cuuint32_t box[3] = {128, box_rows, chunks}, ones[3] = {1, 1, 1};
  return encode_tiled()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, chunks ? 3 : 2, const_cast<void*>(base), dims, strides, box, ones,
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
  // set up while the kernel that splits q still runs; it waits for that one's end before it reads its pieces
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
      !make_map(&maps[2], p.v, rows, 2 * k_bytes, kPage, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, 2) ||
      !make_map(&maps[3], p.qp, q_rows, 128, 128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
      !make_map(&maps[4], p.qp, q_rows, 128, 8, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return FFA_E_LAUNCH;
  const bool two = p.q_dtype == FFA_BF16, bf = p.v_dtype == FFA_BF16;
  if (two) return bf ? launch<2, true>(p, maps, st) : launch<2, false>(p, maps, st);
  return bf ? launch<3, true>(p, maps, st) : launch<3, false>(p, maps, st);
}

}  // namespace ffa
