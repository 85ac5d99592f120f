// attn_chunk.cu — attention of sequences that bring many query rows (a prompt, a chunk of one) over a paged fp16 cache, on tcgen05.
//
// A CTA takes 256 query rows of one sequence and K/V head - the rep heads of a group of tokens - as two tiles of 128, and walks the
// tiles of 128 keys that any of them sees: S = Q K^T, P = 2^(S - m), O = O corr + P V, with the running maximum m of each row.
//
// Bound: the tensor pipe. q and the weights are fp32 values as two fp16 parts each, high and low (error 2^-22, so that the result is as
// good as fp32 products'), which doubles the products: for heads of 128 both row tiles' products of a tile of keys take 4096 clocks.
// A round of both takes some 6000: of a row tile's part 2000 are its own softmax (a warp per scheduler, latency and 32 exponentials per 4
// clocks; with a row's maximum 600), the rest waits for the products of both. 2 x 1000 tokens over 15000 positions of 32 / 8 heads of
// 128: 0.83 ms at first and 0.97 once the power cap has brought the clock down, when the 1002 GFLOP of the parts' products run at 0.75 of what
// cuBLAS sustains in bf16. 1000 tokens with a window of 1024: 53 us, nine tiles of keys per CTA and some 10 us of beginning and end.
//   * The two row tiles alternate: the products of one run while the other's softmax does. One barrier each way per tile: `done` says
//     that S(j + 1) and P V(j) are there, `ready` that P(j) is and both of those have been taken.
//   * P overwrites S in TMEM, 16 columns at a time: 8 of the high parts, 8 of the low ones. It is the A operand of the second product.
//   * Low parts are multiplied first: the tensor core cuts its running sum at every step, and a sum that is still small loses less
//     (error 2.2e-6 with the parts in turn, 0.6e-6 so). For the same reason the output is summed in registers (a row per thread), tile by
//     tile, which also makes the correction by the maximum one FMA. That is done while the exponentials of the next tile run.
//   * K and V come by cp.async into a ring of buffers in the order K, V, K, V, one lane looking up the pages of four rows, and arrive on the
//     buffer's barrier as they land; the issuing warp's proxy fence orders them before the products' reads. They are swizzled as they
//     are written; V is the second product's B operand with its rows as the summed dimension.
//   * Shared memory leaves no L1, so a spilled register costs a trip to L2: what a row's thread seldom needs waits in shared memory,
//     tiles with hidden keys have S overwritten by a loop of its own, and the issuing warp walks its products in fours.
//   * The keys of few row tiles are split over a cluster, whose CTAs put their rows into shared memory and merge a share each.
//   * What is masked for one row but not for another meets a weight of 0, which is NaN if the value is not finite: a row whose result
//     is not finite is computed again key by key, where masked keys are skipped.
#include "attn_rows.cuh"
#include "bulk.cuh"
#include "common.cuh"
#include "pdl.cuh"
#include "per_device.h"

#include <algorithm>
#include <cuda_fp16.h>

namespace tmc {
namespace {

constexpr uint32_t kRows = kChunkRows / 2, kKeys = 128, kThreads = 384, kCols = 512;
constexpr int kNoRow = 0x7ffffffe;
constexpr uint32_t kWarpMma = 0;                             // warps 1-3: the copies; 4-7 and 8-11: the rows of the two tiles

template <int DHP> struct Chunk {
    static constexpr uint32_t Tile = kKeys * DHP * 2;      // bytes of a tile of keys, or of one part of q; 64 dims are 128 bytes
    static constexpr uint32_t Half = kKeys * 128;
    static constexpr uint32_t Buffers = DHP == 128 ? 3 : 6;
    // Heads of 64: the products of 64 keys' weights begin while the other 64 are worked out, O having taken all of the tile before by then (a mixed
    // batch 40.8 -> 38.6 us). Heads of 128 would have to take twice as much in that time, and gain nothing.
    static constexpr bool Early = DHP == 64;
    // registers of the warps that issue and of those that hold rows: of the 384 x 168 that the block is launched with
    static constexpr uint32_t RegsIssue = DHP == 128 ? 56 : 104, RegsRows = DHP == 128 ? 224 : 200;
    static_assert(RegsIssue + 2 * RegsRows <= 3 * 168);
    static constexpr uint32_t Smem = 4 * Tile + Buffers * Tile + 1024;        // q: two tiles of two parts
};

// Operand descriptors: rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes apart. For V the rows are the summed dimension, and the
// next 64 columns lie `half` times 16 bytes on. The low word is the place, in units of 16 bytes.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t at, uint32_t half) { return (at & 0x3ffffu) >> 4 | half << 16; }
// Four products, A and B a fixed step apart. Fours in a loop that is not unrolled: 32 descriptors at a time are more than the issuing
// warp's registers hold.
template <uint32_t A_STEP, uint32_t B_STEP>
__device__ __forceinline__ void mma4_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q, t;\n\t.reg .b32 x, y;\n\t.reg .b64 u, v;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
                 "mov.b64 u, {%1, %8};\n\tmov.b64 v, {%2, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %3, p;\n\t"
                 "add.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\tmov.b64 u, {x, %8};\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %3, t;\n\t"
                 "add.u32 x, x, %6;\n\tadd.u32 y, y, %7;\n\tmov.b64 u, {x, %8};\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %3, t;\n\t"
                 "add.u32 x, x, %6;\n\tadd.u32 y, y, %7;\n\tmov.b64 u, {x, %8};\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], u, v, %3, t;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(A_STEP), "n"(B_STEP), "n"(kDescHi) : "memory");
}
template <uint32_t A_STEP, uint32_t B_STEP>
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q, t;\n\t.reg .b32 x, y;\n\t.reg .b64 v;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
                 "mov.b64 v, {%2, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], v, %3, p;\n\t"
                 "add.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], v, %3, t;\n\t"
                 "add.u32 x, x, %6;\n\tadd.u32 y, y, %7;\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], v, %3, t;\n\t"
                 "add.u32 x, x, %6;\n\tadd.u32 y, y, %7;\n\tmov.b64 v, {y, %8};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], v, %3, t;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(A_STEP), "n"(B_STEP), "n"(kDescHi) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t lead) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// A load's registers may be used behind tmem_landed, which waits for every load before it.
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(t));
}
__device__ __forceinline__ void tmem_landed(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]) :: "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(t));
}
__device__ __forceinline__ void tmem_landed(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) :: "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(t));
}
__device__ __forceinline__ void tmem_landed(uint32_t (&v)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]) :: "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t t, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// x, y as fp16 pairs: the rounded values, and what the rounding left, which fma's mixed form takes from the halves as they are.
__device__ __forceinline__ void parts(float x, float y, uint32_t& hi, uint32_t& lo) {
    float u, v;
    hi = half2_bits(x, y);
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBC00;\n\t"
        "fma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, h, m, %4;\n\t}" : "=f"(u), "=f"(v) : "r"(hi), "f"(x), "f"(y));
    lo = half2_bits(u, v);
}
// Is key j hidden from position p, whose window begins at lo?
__device__ __forceinline__ bool hidden(int j, int p, int lo, int sinks) { return (j > p) | ((j < lo) & (j >= sinks)); }

// mbar_wait without a call in it (a row's 128 sums are live across most of these waits, more than a call may keep in registers), by a whole
// warp, which leaves it together
__device__ __forceinline__ bool wait_for(uint64_t& bar, uint32_t parity, volatile int* gone) {
    const uint32_t at = smem_u32(&bar);
    bool there = mbar_test(at, parity) || mbar_try_wait(at, parity);
    if (!there) {
        const unsigned long long t0 = global_ns();
        for (uint32_t i = 1; !(there = mbar_try_wait(at, parity)); ++i)
            if (i % 64 == 0) {
                if (*gone) break;
                if (global_ns() - t0 > kWaitLimitNs) { *gone = 1; break; }
            }
    }
    return __all_sync(0xffffffffu, there);
}

struct Bars { uint64_t full[6], empty[6], half[2], ready[2], done[2]; };

template <int DHP>
__global__ void __launch_bounds__(kThreads, 1) attn_chunk_kernel(const __grid_constant__ AttnCall a, uint32_t splits) {
    using C = Chunk<DHP>;
    constexpr uint32_t NBUF = C::Buffers;
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) Bars bars;
    __shared__ uint32_t tmem_slot, unit_b, unit_tile, sums[kThreads / 32];
    __shared__ int gone, bad_page;
    __shared__ uint32_t odd[2 * kRows / 32];                 // rows that are computed again
    __shared__ int place[2 * kRows];                         // a row's position (kNoRow: no row), needed now and then: its thread's registers are
                                                             // full, and local memory is slow where shared memory has taken L1's place
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u, tid = threadIdx.x;
    const uint32_t dh = a.c.dh;
    pdl_enter();

    // ---- which sequence, and which of its row tiles: counted from the last one (the longest of a prompt). The host knows how many there are
    // at most; CTAs beyond that come last and leave at once ----
    const uint32_t unit = blockIdx.x / splits, h = unit % a.c.KVH, split = blockIdx.x % splits;
    auto slots_of = [&](uint32_t b, bool note) {
        const KvSeq s = kv_seq(a.c, b);
        if (s.lost && note) note_bad_batch(a.status);
        const unsigned long long rows = (unsigned long long)s.n * a.rep;
        return rows <= a.few ? 0u : (uint32_t)((rows + 2 * kRows - 1) / (2 * kRows));
    };
    if (tid == 0) { unit_b = 0xffffffffu; gone = 0; bad_page = 0; }
    if (tid < 2 * kRows / 32) odd[tid] = 0;
    {
        const uint32_t per = (a.c.B + kThreads - 1) / kThreads, b0 = min(a.c.B, tid * per), b1 = min(a.c.B, b0 + per);
        uint32_t mine = 0;
        for (uint32_t b = b0; b < b1; ++b) mine += slots_of(b, blockIdx.x == 0);
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= (uint32_t)o) incl += y; }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        uint32_t before = incl - mine, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32; ++w) { if (w == warp) before += total; total += sums[w]; }
        const uint32_t slot = total - 1 - unit / a.c.KVH;                // wraps where there is no such unit
        if (slot >= before && slot < before + mine)
            for (uint32_t b = b0; b < b1; ++b) {
                const uint32_t n = slots_of(b, false);
                if (slot < before + n) { unit_b = b; unit_tile = slot - before; break; }
                before += n;
            }
        __syncthreads();
    }
    const uint32_t b = unit_b;
    if (b == 0xffffffffu) return;
    const KvSeq s = kv_seq(a.c, b);
    const uint32_t row0 = unit_tile * 2 * kRows, rows = min(s.n * a.rep - row0, 2 * kRows), tiles2 = rows > kRows ? 2 : 1;
    const bool bad = s.bad || s.n > a.max_q;
    const int p_first = s.first + (int)(row0 / a.rep), p_last = s.first + (int)((row0 + rows - 1) / a.rep);
    KeyTiles<kKeys> kt;
    kt.set(kv_span(a.mask, p_first, p_last), bad);
    const uint32_t t0 = (uint32_t)((unsigned long long)kt.tiles * split / splits), t1 = (uint32_t)((unsigned long long)kt.tiles * (split + 1) / splits), n = t1 - t0;

    auto number_of = [&](uint32_t i) {                                   // of a row in q and out
        const uint32_t tok = (uint32_t)(place[i] - s.first);
        return (size_t)(s.q0 + tok) * a.H + h * a.rep + (row0 + i - tok * a.rep);
    };
    const uint32_t region = (smem_u32(smem_dyn) + 1023u) & ~1023u, ring = region + 4 * C::Tile;
    // where the results go in the end: 16 bytes more than a row, so that threads with a row each store without conflicts
    constexpr uint32_t PITCH = DHP * 4 + 16;
    const uint32_t stats = region + 2 * kRows * PITCH;
    static_assert(2 * kRows * (PITCH + 8) <= (4 + C::Buffers) * C::Tile, "the results fit");
    if (tid == 0) {
        for (uint32_t i = 0; i < NBUF; ++i) { mbar_init(smem_u32(&bars.full[i]), 96); mbar_init(smem_u32(&bars.empty[i]), 1); }
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(smem_u32(&bars.half[i]), 4); mbar_init(smem_u32(&bars.ready[i]), 4); mbar_init(smem_u32(&bars.done[i]), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::RegsIssue));
        if (warp == kWarpMma && n) {
            const uint32_t lead = elect_one();
            constexpr uint32_t idesc_s = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);                    // fp16 x fp16 -> fp32
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DHP >> 3) << 17) | ((kRows >> 4) << 24);      // B with its rows as the summed dimension
            auto wait_full = [&](uint32_t i) {                           // the copies' writes, then the products' reads through the other proxy
                const bool there = wait_for(bars.full[i % NBUF], i / NBUF & 1u, &gone);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                return there;
            };
            // The low parts first: a sum that is still small is cut to less.
            auto scores = [&](uint32_t w, uint32_t i) {                  // S of row tile w and the K tile that is the i-th in the ring
                const uint32_t q = desc_lo(region + w * 2 * C::Tile, 1), k = desc_lo(ring + i % NBUF * C::Tile, 1), d = tmem + w * kKeys;
#pragma unroll 1
                for (uint32_t x = 0; x < 2 * (DHP / 64); ++x) {          // 64 dims of one part
                    const uint32_t off = x % (DHP / 64) * (C::Half >> 4);
                    mma4_ss<2, 2>(d, q + (x < DHP / 64 ? C::Tile >> 4 : 0u) + off, k + off, idesc_s, x, lead);
                }
            };
            auto values = [&](uint32_t w, uint32_t i, uint32_t half) {   // P V of 64 keys
                const uint32_t v = desc_lo(ring + i % NBUF * C::Tile, C::Half >> 4), pt = tmem + w * kKeys, d = tmem + 2 * kKeys + w * kKeys;
#pragma unroll 1
                for (uint32_t x = 0; x < 2; ++x) mma4_ts<16, 128>(d, pt + half * 64u + (x ? 0u : 8u), v + half * 512u, idesc_o, half | x, lead);
            };
            ok = wait_full(0);
            for (uint32_t w = 0; w < tiles2 && ok; ++w) {
                ok = wait_for(bars.ready[w], 0, &gone);                  // q is there
                if (!ok) break;
                fence_after();
                scores(w, 0);
                commit(smem_u32(&bars.done[w]), lead);
            }
            if (ok) commit(smem_u32(&bars.empty[0]), lead);
            for (uint32_t j = 0; j < n && ok; ++j) {
                const uint32_t iv = 2 * j + 1, ik = 2 * j + 2;
                for (uint32_t w = 0; w < tiles2; ++w) {
                    if (C::Early) {
                        ok = wait_for(bars.half[w], j & 1u, &gone) && (w || wait_full(iv));
                        if (!ok) break;
                        fence_after();
                        values(w, iv, 0);
                    }
                    ok = wait_for(bars.ready[w], (j + 1) & 1u, &gone) && (C::Early || w || wait_full(iv));
                    if (!ok) break;
                    fence_after();
                    if (!C::Early) values(w, iv, 0);
                    values(w, iv, 1);
                    if (w + 1 == tiles2) commit(smem_u32(&bars.empty[iv % NBUF]), lead);
                    if (j + 1 < n) {
                        if (!w && !wait_full(ik)) { ok = false; break; }
                        scores(w, ik);
                        if (w + 1 == tiles2) commit(smem_u32(&bars.empty[ik % NBUF]), lead);
                    }
                    commit(smem_u32(&bars.done[w]), lead);
                }
            }
        } else if (warp != kWarpMma) {
            // Three warps share every tile. Offsets of K and V rows are the same; the copies arrive on the tile's barrier as they land.
            const uint32_t mine = warp - 1, chunks = dh / 8;
            constexpr uint32_t CH = DHP / 8, RP = 32 / CH;               // 16-byte pieces of a row, rows of a round
            uint32_t page[4];                                            // of rows 32 r + lane of the tile after this one
            bool missing = false;
            auto slot_of = [&](uint32_t key) { return a.c.page_shift >= 0 ? key >> a.c.page_shift : key / a.c.page; };
            auto look_up = [&](uint32_t j) {
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    const uint32_t place_at = (t0 + j) * kKeys + 32 * r + lane;
                    page[r] = 0;
                    if (a.c.table && j < n && place_at < kt.count) page[r] = (uint32_t)a.c.table[(size_t)b * a.c.table_ld + slot_of(kt.key(place_at))];
                }
            };
            look_up(0);
            for (uint32_t j = 0; j < n && ok; ++j) {
                uint32_t lo[4], hi[4], there[4];
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    const uint32_t place_at = (t0 + j) * kKeys + 32 * r + lane, key = kt.key(place_at);
                    bool have = place_at < kt.count;
                    if (have && page[r] >= a.c.npages) { have = false; missing = true; }
                    const uint32_t row = a.c.table ? key - slot_of(key) * a.c.page : key;
                    const size_t at = have ? (((size_t)page[r] * a.c.KVH + h) * a.c.page + row) * dh * 2 : 0;
                    lo[r] = (uint32_t)at; hi[r] = (uint32_t)(at >> 32);
                    there[r] = __ballot_sync(0xffffffffu, have);
                }
                look_up(j + 1);
#pragma unroll
                for (uint32_t which = 0; which < 2; ++which) {
                    const uint32_t i = 2 * j + which, buf = i % NBUF, dst = ring + buf * C::Tile;
                    const uint8_t* base = (const uint8_t*)(which ? a.c.v : a.c.k);
                    if (!wait_for(bars.empty[buf], (i / NBUF & 1u) ^ 1u, &gone)) { ok = false; break; }
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r)
#pragma unroll 4
                        for (uint32_t k = (mine + r) % 3; k < 32 / RP; k += 3) {
                            const uint32_t src = k * RP + lane / CH, ch = lane % CH, row = 32 * r + src;
                            const size_t off = (size_t)__shfl_sync(0xffffffffu, lo[r], src) | (size_t)__shfl_sync(0xffffffffu, hi[r], src) << 32;
                            const bool have = (there[r] >> src & 1u) && ch < chunks;
                            copy16(dst + (ch >> 3) * C::Half + row * 128u + (((ch & 7u) ^ (row & 7u)) << 4), base + (have ? off + ch * 16 : 0), have ? 16u : 0u);
                        }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&bars.full[buf])) : "memory");
                }
            }
            if (missing) bad_page = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::RegsRows));
        const uint32_t w = (warp - 4) >> 2, r = (warp & 3u) * 32 + lane, row = w * kRows + r;
        if (w < tiles2) {
            int p_min, lo_max;                                           // the least that a row of the warp sees ahead and behind
            {
                const bool is = row < rows;
                const uint32_t gi = row0 + (is ? row : 0u), tok = gi / a.rep;
                const int p = is ? s.first + (int)tok : kNoRow;          // rows that are none see everything, so that they ask for no masks
                place[row] = p;
                p_min = __reduce_min_sync(0xffffffffu, p);
                lo_max = __reduce_max_sync(0xffffffffu, is ? window_from(a.mask, p) : 0);
            }
            // q: a row per turn (two for heads of 64), four dims per lane, so that the loads are whole lines
            constexpr uint32_t LR = DHP / 4, RT = 32 / LR;               // lanes of a row, rows of a turn
            const uint32_t first_row = row - lane, piece = lane % LR;
            float back = 1.f;
            __syncwarp();
            constexpr uint32_t AHEAD = 32 / RT;                          // all loads on their way together: nothing else is in the registers yet
            const float by = a.scale * kLog2e;
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < 32; i0 += AHEAD * RT) {
                float4 ahead[AHEAD];
#pragma unroll
                for (uint32_t n1 = 0; n1 < AHEAD; ++n1) {
                    const uint32_t rr = first_row + i0 + n1 * RT + lane / LR;
                    ahead[n1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (rr < rows && 4 * piece < dh) ahead[n1] = *reinterpret_cast<const float4*>(a.q + number_of(rr) * dh + 4 * piece);
                }
#pragma unroll
                for (uint32_t n1 = 0; n1 < AHEAD; ++n1) {
                    const uint32_t i = i0 + n1 * RT, rq = (first_row + i + lane / LR) % kRows;
                    const float4 f = ahead[n1];
                    float top = fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))) * by;
#pragma unroll
                    for (uint32_t x = LR / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 120);      // the row's largest to [2^13, 2^14)
                    const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                    uint32_t hi[2], low[2];
                    parts(f.x * by * up, f.y * by * up, hi[0], low[0]);
                    parts(f.z * by * up, f.w * by * up, hi[1], low[1]);
                    const uint32_t c = piece / 2, to = region + w * 2 * C::Tile + (c >> 3) * C::Half + rq * 128u + (((c & 7u) ^ (rq & 7u)) << 4) + (piece & 1u) * 8u;
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(hi[0]), "r"(hi[1]) : "memory");
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + C::Tile), "r"(low[0]), "r"(low[1]) : "memory");
#pragma unroll
                    for (uint32_t k = 0; k < RT; ++k) {
                        const int es = __shfl_sync(0xffffffffu, e, k * LR);
                        if (lane == i + k) back = __uint_as_float((uint32_t)(127 - 13 + es) << 23);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            mbar_arrive_if(smem_u32(&bars.ready[w]), lane == 0);
            const uint32_t lanes = (warp & 3u) << 21, st = tmem + w * kKeys + lanes, ot = tmem + 2 * kKeys + w * kKeys + lanes;
            float o[DHP], m = -CUDART_INF_F, l = 0.f, corr = 0.f;
#pragma unroll
            for (uint32_t d = 0; d < DHP; ++d) o[d] = 0.f;
            {                                                            // what the first tile finds as the values of the one before
                uint32_t none[16] = {};
#pragma unroll
                for (uint32_t d = 0; d < DHP; d += 16) tmem_st(ot + d, none);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            auto hand_over = [&](uint64_t& bar) {                        // what has been stored and read, to the issuing warp
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                mbar_arrive_if(smem_u32(&bar), lane == 0);
            };
            // S of the tiles that not every row of the warp sees whole: what a row does not see is -infinity from here on
            auto hide = [&](uint32_t u0) {
                const int p = place[row], lo = window_from(a.mask, p), sinks = (int)a.mask.sinks;
#pragma unroll 1
                for (uint32_t c = 0; c < kKeys / 16; ++c) {
                    const uint32_t u1 = u0 + 16 * c;
                    if (kt.seen(u1, 16, p_min, (uint32_t)lo_max)) continue;
                    uint32_t v[16];
                    tmem_ld(st + 16 * c, v);
                    tmem_landed(v);
#pragma unroll
                    for (uint32_t k = 0; k < 16; ++k)
                        v[k] = hidden((int)kt.key(u1 + k), p, lo, sinks) ? 0xff800000u : v[k];
                    tmem_st(st + 16 * c, v);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            };
            auto maximum = [&]() {
                float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
                uint32_t v[2][16];
                tmem_ld(st, v[0]);
#pragma unroll
                for (uint32_t c = 0; c < kKeys / 16; ++c) {
                    tmem_landed(v[c & 1]);
                    if (c + 1 < kKeys / 16) tmem_ld(st + 16 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
                    for (uint32_t k = 0; k < 16; ++k) top[k & 3u] = fmaxf(top[k & 3u], __uint_as_float(v[c & 1][k]));
                }
                return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            };
            // S in, P out, the sum on the way; and, since the exponentials leave the other pipes idle, P V of the tile before into O. The
            // exponentials of 8 keys are under way while the 8 before them are split and stored.
            auto weights = [&](float base, float now) {
                constexpr uint32_t N = kKeys / 8;
                const float shift = kUp<__half> - base;
                float sum[4] = {}, y[2][8];
                uint32_t v[8], x[16], z[8];
                tmem_ld(st, v);
                tmem_landed(v);
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) y[0][k] = pow2(fmaf(__uint_as_float(v[k]), back, shift));
                tmem_ld(st + 8, v);
                tmem_ld(ot, z);
#pragma unroll
                for (uint32_t c = 0; c < N; ++c) {
                    const uint32_t g = 4 * (c & 1u);
                    tmem_landed(v);
                    if (c + 1 < N) {
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) y[(c + 1) & 1][k] = pow2(fmaf(__uint_as_float(v[k]), back, shift));
                    }
                    if (c < DHP / 8) {
                        tmem_landed(z);
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) o[8 * c + k] = fmaf(o[8 * c + k], corr, __uint_as_float(z[k]));
                    }
                    if (c + 2 < N) tmem_ld(st + 8 * (c + 2), v);
                    if (c + 1 < DHP / 8) tmem_ld(ot + 8 * (c + 1), z);
#pragma unroll
                    for (uint32_t k = 0; k < 8; k += 2) {
                        sum[k >> 1] += y[c & 1][k] + y[c & 1][k + 1];
                        parts(y[c & 1][k], y[c & 1][k + 1], x[g + (k >> 1)], x[8 + g + (k >> 1)]);
                    }
                    if (c & 1u) tmem_st(st + 8 * (c - 1), x);
                    if (C::Early && c + 1 == N / 2) hand_over(bars.half[w]);
                }
                l = fmaf(l, now, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            };
            for (uint32_t j = 0; j < n; ++j) {
                if (!wait_for(bars.done[w], j & 1u, &gone)) { ok = false; break; }
                fence_after();
                if (!kt.seen((t0 + j) * kKeys, kKeys, p_min, (uint32_t)lo_max)) hide((t0 + j) * kKeys);
                const float mn = fmaxf(m, maximum() * back), base = mn == -CUDART_INF_F ? 0.f : mn, now = pow2(m - base);
                m = mn;
                weights(base, now);
                corr = now;
                hand_over(bars.ready[w]);
            }
            if (n && ok) {
                if (wait_for(bars.done[w], n & 1u, &gone)) {
                    fence_after();
#pragma unroll
                    for (uint32_t c = 0; c < DHP / 32; ++c) {
                        uint32_t v[32];
                        tmem_ld(ot + 32 * c, v);
                        tmem_landed(v);
#pragma unroll
                        for (uint32_t k = 0; k < 32; ++k) o[32 * c + k] = fmaf(o[32 * c + k], corr, __uint_as_float(v[k]));
                    }
                }
                else ok = false;
            }
            bool finite = fabsf(l) < CUDART_INF_F;
#pragma unroll
            for (uint32_t d = 0; d < DHP; ++d) finite = finite && fabsf(o[d]) < CUDART_INF_F;
            if (!ok || bad) l = CUDART_NAN_F;
            const uint32_t again = __ballot_sync(0xffffffffu, place[row] != kNoRow && ok && !bad && !finite);
            if (lane == 0) odd[w * 4 + (warp & 3u)] = again;
            // The rows, unnormalised, and their statistics in shared memory, where q and the ring were: no product reads them any more once
            // both row tiles are here.
            asm volatile("bar.sync 1, %0;" ::"r"(tiles2 * 128u) : "memory");
#pragma unroll
            for (uint32_t d = 0; d < DHP; d += 4)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(region + row * PITCH + d * 4), "f"(o[d]), "f"(o[d + 1]), "f"(o[d + 2]), "f"(o[d + 3]) : "memory");
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(stats + row * 8), "f"(m), "f"(l) : "memory");
        }
    }
    if (!ok) { if (a.status) *(volatile int*)a.status = 1; }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_before();
    __syncthreads();
    if (tid == 0 && (bad || bad_page)) note_bad_batch(a.status);
    if (warp == kWarpMma) {
        if (gone)                                                        // products may still be running: their last commits
            for (uint32_t i = 0; i < 2; ++i)
                for (uint32_t par = 0; par < 2; ++par) { int late = 0; (void)mbar_wait(smem_u32(&bars.done[i]), par, &late, 20000000ull); }
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
    }
    // ---- rows that are computed again, or whose pages were not all there ----
    float* const rows_at = reinterpret_cast<float*>(smem_dyn + (region - smem_u32(smem_dyn)));
    float2* const stats_at = reinterpret_cast<float2*>(smem_dyn + (stats - smem_u32(smem_dyn)));
    uint32_t any = 0;
#pragma unroll
    for (uint32_t i = 0; i < 2 * kRows / 32; ++i) any |= odd[i];
    if (warp >= 4 && (any || bad_page || gone))
        for (uint32_t i = warp - 4; i < rows; i += 8) {
            if (bad_page || gone) { if (lane == 0) stats_at[i].y = CUDART_NAN_F; }
            else if (odd[i >> 5] >> (i & 31u) & 1u) row_again<__half>(a, b, h, place[i], kt, t0, t1, a.q + number_of(i) * dh, rows_at + i * (PITCH / 4), stats_at + i);
        }
    // ---- the parts of the cluster's CTAs together: each takes every splits-th turn of a warp, whole lines at a time ----
    if (splits > 1) cluster_sync(); else __syncthreads();
    constexpr uint32_t LR = DHP / 4, RT = 32 / LR;                       // lanes of a row, rows of a turn
    const uint32_t piece = lane % LR;
    if (warp >= 4) {
        auto finish = [&](uint32_t rr, float4 y, float L) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            if (rr < rows && 4 * piece < dh)
                *reinterpret_cast<float4*>(a.out + number_of(rr) * dh + 4 * piece) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        };
        if (splits == 1) {
#pragma unroll 4
            for (uint32_t i = (warp - 4) * RT; i < rows; i += 8 * RT) {
                const uint32_t rr = i + lane / LR;
                finish(rr, *reinterpret_cast<const float4*>(rows_at + rr * (PITCH / 4) + piece * 4), stats_at[rr].y);
            }
        } else {
            for (uint32_t i = ((warp - 4) * splits + split) * RT; i < rows; i += 8 * splits * RT) {
                const uint32_t rr = i + lane / LR;
                float M = -CUDART_INF_F, L = 0.f;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                for (uint32_t k = 0; k < splits; k += 2) {               // a power of two, so two at a time
                    const float2 m0 = ld_cta2(map_cta(stats + rr * 8, k)), m1 = ld_cta2(map_cta(stats + rr * 8, k + 1));
                    const float4 x0 = ld_cta4(map_cta(region + rr * PITCH + piece * 16, k)), x1 = ld_cta4(map_cta(region + rr * PITCH + piece * 16, k + 1));
                    const float mn = fmaxf(M, fmaxf(m0.x, m1.x)), base = mn == -CUDART_INF_F ? 0.f : mn, f = pow2(M - base), f0 = pow2(m0.x - base), f1 = pow2(m1.x - base);
                    L = fmaf(L, f, fmaf(f0, m0.y, f1 * m1.y));
                    y.x = fmaf(y.x, f, fmaf(f0, x0.x, f1 * x1.x)); y.y = fmaf(y.y, f, fmaf(f0, x0.y, f1 * x1.y));
                    y.z = fmaf(y.z, f, fmaf(f0, x0.z, f1 * x1.z)); y.w = fmaf(y.w, f, fmaf(f0, x0.w, f1 * x1.w));
                    M = mn;
                }
                finish(rr, y, L);
            }
        }
    }
    if (splits > 1) cluster_sync();                                      // nobody leaves while its shared memory is read
}

template <int DHP>
bool go(const AttnCall& a, const ChunkPlan& pl, cudaStream_t st) {
    auto* kernel = attn_chunk_kernel<DHP>;
    static PerDevice<bool> ready;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || !ready.get(dev, [=](bool&) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Chunk<DHP>::Smem) == cudaSuccess; }))
        return fail("attention: shared memory attribute: %s", cudaGetErrorString(cudaGetLastError()));
    const unsigned long long units = (unsigned long long)a.c.KVH * pl.slots;
    if (units * pl.splits > 0x7fffffffull) return fail("attention: %llu tiles of query rows", units);
    if (!launch_units(kernel, (unsigned)units, pl.splits, kThreads, Chunk<DHP>::Smem, st, a, pl.splits)) return false;
    note_launch();
    return check_launch("attn_chunk");
}

}  // namespace

ChunkPlan plan_attn_chunk(uint32_t T, uint32_t B, uint32_t KVH, uint32_t rep, uint32_t few, uint32_t row_tile) {
    const unsigned long long rows = (unsigned long long)T * rep, least = (rows + row_tile - 1) / row_tile;
    ChunkPlan pl;
    pl.slots = (uint32_t)(rows / row_tile + std::min<unsigned long long>(B, rows / (few + 1ull)));
    pl.splits = 1;
    const uint32_t ctas = row_tile == kChunkRows ? 148 : 296;           // that run at a time
    while (pl.splits < 8 && 2 * pl.splits * least * KVH <= ctas) pl.splits *= 2;
    return pl;
}

bool launch_attn_chunk(const AttnCall& a, const ChunkPlan& pl, cudaStream_t st) {
    return a.c.dh <= 64 ? go<64>(a, pl, st) : go<128>(a, pl, st);
}

}  // namespace tmc
