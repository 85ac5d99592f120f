// attn_chunk.cu — attention of sequences that bring many query rows (a prompt, a chunk of one) over a paged fp16 cache, on tcgen05.
//
// A CTA takes 256 query rows of one sequence and K/V head - the rep heads of a group of tokens - as two tiles of 128, and walks the
// tiles of 128 keys that any of them sees: S = Q K^T, P = 2^(S - m), O = O corr + P V, with the running maximum m of each row.
//
// Bound: the tensor pipe. q and the weights are fp32 values as two fp16 parts each, high and low (error 2^-22, so that the result is as
// good as fp32 products'), which doubles the products: for heads of 128 a tile of 128 x 128 takes 4 x 512 clocks, against 1024 for its
// exponentials and about 1200 of the four schedulers' issue for the softmax and the output's update.
//   * The two row tiles alternate: the products of one run while the other's softmax does. One barrier each way per tile: `done` says
//     that S(j + 1) and P V(j) are there, `ready` that P(j) is and both of those have been taken.
//   * P overwrites S in TMEM, 16 columns at a time: 8 of the high parts, 8 of the low ones. It is the A operand of the second product.
//   * The output is summed in registers (a row per thread), tile by tile: a tensor core's own running sum is cut, not rounded, at every
//     step, which over thousands of keys costs more than the parts' rounding; and the correction by the maximum is then one FMA.
//   * K and V come by cp.async, one lane looking up the pages of four rows, into a ring of buffers in the order K, V, K, V. They are
//     swizzled as they are written; V is the second product's B operand with its rows as the summed dimension.
//   * What is masked for one row but not for another meets a weight of 0, which is NaN if the value is not finite: a row whose result
//     is not finite is computed again key by key, where masked keys are skipped.
#include "attn_rows.cuh"
#include "bulk.cuh"
#include "common.cuh"
#include "per_device.h"

#include <algorithm>
#include <cuda_fp16.h>

namespace tmc {
namespace {

constexpr uint32_t kRows = 128, kKeys = 128, kThreads = 384, kCols = 512;
constexpr uint32_t kWarpMma = 0, kWarpK = 1, kWarpV = 2;     // warps 4-7 and 8-11: the rows of the two tiles

template <int DHP> struct Chunk {
    static constexpr uint32_t Tile = kKeys * DHP * 2;      // bytes of a tile of keys, or of one part of q; 64 dims are 128 bytes
    static constexpr uint32_t Half = kKeys * 128;
    static constexpr uint32_t Buffers = DHP == 128 ? 3 : 6;
    static constexpr uint32_t Smem = 4 * Tile + Buffers * Tile + 1024;        // q: two tiles of two parts
};

// K-major rows of 128 bytes, 128-byte swizzle, 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k(uint32_t at) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return (uint64_t)hi << 32 | (uint64_t)((at & 0x3ffffu) >> 4 | 1u << 16);
}
// The same bytes with the rows as the summed dimension: 8 rows 1024 bytes apart, the next 64 columns `half` bytes on
template <uint32_t HALF> __device__ __forceinline__ uint64_t desc_mn(uint32_t at) {
    constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return (uint64_t)hi << 32 | (uint64_t)((at & 0x3ffffu) >> 4 | (HALF >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
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
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(t));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(t));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
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
// The high part is the value cut to 11 bits, so that it converts as it is; what is left has 13 and is rounded to 11.
__device__ __forceinline__ float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// Is key j = j0 + i hidden from position p? lo: where p's window begins.
__device__ __forceinline__ bool hidden(int j, int p, int lo, int sinks) { return j > p || (j < lo && j >= sinks); }

// mbar_wait without a call in it: a row's 128 sums are live across most of these waits, more than a call may keep in registers
__device__ __forceinline__ bool wait_for(uint64_t& bar, uint32_t parity, volatile int* gone) {
    const uint32_t at = smem_u32(&bar);
    if (mbar_test(at, parity) || mbar_try_wait(at, parity)) return true;
    const unsigned long long t0 = global_ns();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(at, parity)) return true;
        if (i % 64 == 0) {
            if (*gone) return false;
            if (global_ns() - t0 > kWaitLimitNs) { *gone = 1; return false; }
        }
    }
}

struct Bars { uint64_t full[6], empty[6], ready[2], done[2]; };

template <int DHP>
__global__ void __launch_bounds__(kThreads, 1) attn_chunk_kernel(const __grid_constant__ AttnCall a, uint32_t splits, float* part, float2* stat) {
    using C = Chunk<DHP>;
    constexpr uint32_t NBUF = C::Buffers;
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) Bars bars;
    __shared__ uint32_t tmem_slot, unit_b, unit_tile, sums[kThreads / 32];
    __shared__ int gone, bad_page;
    __shared__ uint32_t odd[2 * kRows / 32];                 // rows that are computed again
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u, tid = threadIdx.x;
    const uint32_t dh = a.c.dh;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- which sequence, and which of its row tiles: counted from the last one (the longest of a prompt) ----
    const uint32_t at_once = a.c.KVH * splits, slot = (gridDim.x - 1 - blockIdx.x) / at_once, h = blockIdx.x % at_once % a.c.KVH, split = blockIdx.x % at_once / a.c.KVH;
    auto slots_of = [&](uint32_t b, bool note) {
        const KvSeq s = kv_seq(a.c, b);
        if (s.lost && note) note_bad_batch(a.status);
        const unsigned long long rows = (unsigned long long)s.n * a.rep;
        return rows <= a.few ? 0u : (uint32_t)((rows + 2 * kRows - 1) / (2 * kRows));
    };
    if (tid == 0) { unit_b = 0xffffffffu; gone = 0; bad_page = 0; }
    if (tid < 2 * kRows / 32) odd[tid] = 0;
    if (a.c.B == 1) {
        if (tid == 0 && slot < slots_of(0, true)) { unit_b = 0; unit_tile = slot; }
        __syncthreads();
    } else {
        const uint32_t per = (a.c.B + kThreads - 1) / kThreads, b0 = min(a.c.B, tid * per), b1 = min(a.c.B, b0 + per);
        uint32_t mine = 0;
        for (uint32_t b = b0; b < b1; ++b) mine += slots_of(b, blockIdx.x == 0);
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= (uint32_t)o) incl += y; }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        uint32_t before = incl - mine;
        for (uint32_t w = 0; w < warp; ++w) before += sums[w];
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

    const uint32_t region = (smem_u32(smem_dyn) + 1023u) & ~1023u, ring = region + 4 * C::Tile;
    if (tid == 0) {
        for (uint32_t i = 0; i < NBUF; ++i) { mbar_init(smem_u32(&bars.full[i]), 1); mbar_init(smem_u32(&bars.empty[i]), 1); }
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(smem_u32(&bars.ready[i]), 4); mbar_init(smem_u32(&bars.done[i]), 1); }
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
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kWarpMma && n) {
            const uint32_t lead = elect_one();
            constexpr uint32_t idesc_s = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);                    // fp16 x fp16 -> fp32
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DHP >> 3) << 17) | ((kRows >> 4) << 24);      // B with its rows as the summed dimension
            auto wait_full = [&](uint32_t i) { return wait_for(bars.full[i % NBUF], i / NBUF & 1u, &gone); };
            auto scores = [&](uint32_t w, uint32_t i) {                  // S of row tile w and the K tile that is the i-th in the ring
                const uint32_t q = region + w * 2 * C::Tile, k = ring + i % NBUF * C::Tile, d = tmem + w * kKeys;
#pragma unroll
                for (uint32_t p = 0; p < 2; ++p)
#pragma unroll
                    for (uint32_t x = 0; x < DHP / 16; ++x) {
                        const uint32_t off = (x >> 2) * C::Half + (x & 3u) * 32u;
                        mma_ss(d, desc_k(q + p * C::Tile + off), desc_k(k + off), idesc_s, p | x, lead);
                    }
            };
            auto values = [&](uint32_t w, uint32_t i) {                  // P V
                const uint32_t v = ring + i % NBUF * C::Tile, pt = tmem + w * kKeys, d = tmem + 2 * kKeys + w * kKeys;
#pragma unroll
                for (uint32_t x = 0; x < kKeys / 16; ++x)
#pragma unroll
                    for (uint32_t p = 0; p < 2; ++p)
                        mma_ts(d, pt + x * 16u + p * 8u, desc_mn<C::Half>(v + x * 2048u), idesc_o, p | x, lead);
            };
            ok = wait_full(0);
            for (uint32_t w = 0; w < tiles2 && ok; ++w) {
                ok = wait_for(bars.ready[w], 0, &gone);      // q is there
                if (!ok) break;
                fence_after();
                scores(w, 0);
                commit(smem_u32(&bars.done[w]), lead);
            }
            if (ok) commit(smem_u32(&bars.empty[0]), lead);
            for (uint32_t j = 0; j < n && ok; ++j) {
                const uint32_t iv = 2 * j + 1, ik = 2 * j + 2;
                for (uint32_t w = 0; w < tiles2; ++w) {
                    ok = wait_for(bars.ready[w], (j + 1) & 1u, &gone) && (w || wait_full(iv));
                    if (!ok) break;
                    fence_after();
                    values(w, iv);
                    if (w + 1 == tiles2) commit(smem_u32(&bars.empty[iv % NBUF]), lead);
                    if (j + 1 < n) {
                        if (!w && !wait_full(ik)) { ok = false; break; }
                        scores(w, ik);
                        if (w + 1 == tiles2) commit(smem_u32(&bars.empty[ik % NBUF]), lead);
                    }
                    commit(smem_u32(&bars.done[w]), lead);
                }
            }
        } else if (warp == kWarpK || warp == kWarpV) {
            const uint32_t which = warp - kWarpK, chunks = dh / 8;
            const uint8_t* base = (const uint8_t*)(which ? a.c.v : a.c.k);
            bool missing = false;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t i = 2 * j + which, buf = i % NBUF, dst = ring + buf * C::Tile, j0 = kt.key(t0 + j);
                uint32_t lo[4], hi[4], there[4];
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {                       // the page of row 32 r + lane
                    const uint32_t key = j0 + 32 * r + lane;
                    size_t at = 0;
                    bool have = key < kt.end;
                    if (have && !kv_row(a.c, b, key, &at)) { have = false; missing = true; }
                    at = (at + (size_t)h * a.c.page * dh) * 2;
                    lo[r] = (uint32_t)at; hi[r] = (uint32_t)(at >> 32);
                    there[r] = __ballot_sync(0xffffffffu, have);
                }
                if (!wait_for(bars.empty[buf], (i / NBUF & 1u) ^ 1u, &gone)) { ok = false; break; }
                constexpr uint32_t CH = DHP / 8, RP = 32 / CH;           // 16-byte pieces of a row, rows of a round
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r)
#pragma unroll 8
                    for (uint32_t k = 0; k < 32 / RP; ++k) {
                        const uint32_t src = k * RP + lane / CH, ch = lane % CH, row = 32 * r + src;
                        const size_t off = (size_t)__shfl_sync(0xffffffffu, lo[r], src) | (size_t)__shfl_sync(0xffffffffu, hi[r], src) << 32;
                        const bool have = (there[r] >> src & 1u) && ch < chunks;
                        copy16(dst + (ch >> 3) * C::Half + row * 128u + (((ch & 7u) ^ (row & 7u)) << 4), base + (have ? off + ch * 16 : 0), have ? 16u : 0u);
                    }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                mbar_arrive_if(smem_u32(&bars.full[buf]), lane == 0);
            }
            if (missing) bad_page = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const uint32_t w = (warp - 4) >> 2, r = (warp & 3u) * 32 + lane, row = w * kRows + r;
        if (w < tiles2) {
            const bool is = row < rows;
            const uint32_t gi = row0 + (is ? row : 0u), tok = gi / a.rep;
            const size_t at = ((size_t)(s.q0 + tok) * a.H + h * a.rep + gi % a.rep) * dh;
            const int p = is ? s.first + (int)tok : 0x7ffffffe, lo = a.mask.window && p >= (int)a.mask.window ? p - (int)a.mask.window + 1 : 0, sinks = (int)a.mask.sinks;
            // rows that are none see everything, so that they ask for no masks
            const int p_min = __reduce_min_sync(0xffffffffu, p), lo_max = __reduce_max_sync(0xffffffffu, is ? lo : 0);
            float back;
            {
                float top = 0.f;
                for (uint32_t d = 0; d < dh; d += 4) {
                    const float4 f = is ? *reinterpret_cast<const float4*>(a.q + at + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y))), fmaxf(fabsf(f.z), fabsf(f.w)));
                }
                top *= a.scale * kLog2e;
                const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 120);          // the row's largest to [2^13, 2^14)
                const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                back = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll 4
                for (uint32_t c = 0; c < DHP / 8; ++c) {
                    float f[8];
#pragma unroll
                    for (uint32_t k = 0; k < 8; k += 4) {
                        const float4 x = is && c * 8 < dh ? *reinterpret_cast<const float4*>(a.q + at + c * 8 + k) : make_float4(0.f, 0.f, 0.f, 0.f);
                        f[k] = x.x; f[k + 1] = x.y; f[k + 2] = x.z; f[k + 3] = x.w;
                    }
                    uint32_t hi[4], low[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const float x = f[2 * k] * (a.scale * kLog2e) * up, y = f[2 * k + 1] * (a.scale * kLog2e) * up, xh = high_part(x), yh = high_part(y);
                        hi[k] = half2_bits(xh, yh); low[k] = half2_bits(x - xh, y - yh);
                    }
                    const uint32_t to = region + w * 2 * C::Tile + (c >> 3) * C::Half + r * 128u + (((c & 7u) ^ (r & 7u)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + C::Tile), "r"(low[0]), "r"(low[1]), "r"(low[2]), "r"(low[3]) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                mbar_arrive_if(smem_u32(&bars.ready[w]), lane == 0);
            }
            const uint32_t lanes = (warp & 3u) << 21, st = tmem + w * kKeys + lanes, ot = tmem + 2 * kKeys + w * kKeys + lanes;
            float o[DHP], m = -CUDART_INF_F, l = 0.f, corr = 0.f;
#pragma unroll
            for (uint32_t d = 0; d < DHP; ++d) o[d] = 0.f;
            auto add_values = [&]() {                                    // O = O corr + P V
#pragma unroll
                for (uint32_t c = 0; c < DHP / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld(ot + 32 * c, v);
#pragma unroll
                    for (uint32_t k = 0; k < 32; ++k) o[32 * c + k] = fmaf(o[32 * c + k], corr, __uint_as_float(v[k]));
                }
            };
            for (uint32_t j = 0; j < n; ++j) {
                if (!wait_for(bars.done[w], j & 1u, &gone)) { ok = false; break; }
                fence_after();
                const int j0 = (int)kt.key(t0 + j);
                const bool whole = j0 + (int)kKeys - 1 <= p_min && (j0 >= lo_max || j0 + (int)kKeys <= sinks);
                float top = -CUDART_INF_F;
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld(st + 32 * c, v);
                    if (!whole) {
#pragma unroll
                        for (uint32_t k = 0; k < 32; ++k)
                            if (hidden(j0 + (int)(32 * c + k), p, lo, sinks)) v[k] = 0xff800000u;
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 32; ++k) top = fmaxf(top, __uint_as_float(v[k]));
                }
                const float mn = fmaxf(m, top * back), base = mn == -CUDART_INF_F ? 0.f : mn, now = pow2(m - base);
                m = mn;
                const float shift = kUp - base;
                float sum[4] = {};
#pragma unroll
                for (uint32_t c = 0; c < kKeys / 16; ++c) {
                    uint32_t v[16], x[16];
                    tmem_ld(st + 16 * c, v);
#pragma unroll
                    for (uint32_t k = 0; k < 16; k += 2) {
                        float y = pow2(fmaf(__uint_as_float(v[k]), back, shift)), z = pow2(fmaf(__uint_as_float(v[k + 1]), back, shift));
                        if (!whole) {
                            if (hidden(j0 + (int)(16 * c + k), p, lo, sinks)) y = 0.f;
                            if (hidden(j0 + (int)(16 * c + k + 1), p, lo, sinks)) z = 0.f;
                        }
                        sum[k >> 1 & 3u] += y + z;
                        const float yh = high_part(y), zh = high_part(z);
                        x[k >> 1] = half2_bits(yh, zh);
                        x[8 + (k >> 1)] = half2_bits(y - yh, z - zh);
                    }
                    tmem_st(st + 16 * c, x);
                }
                l = fmaf(l, now, (sum[0] + sum[1]) + (sum[2] + sum[3]));
                if (j) add_values();
                corr = now;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                mbar_arrive_if(smem_u32(&bars.ready[w]), lane == 0);
            }
            if (n && ok) {
                if (wait_for(bars.done[w], n & 1u, &gone)) { fence_after(); add_values(); }
                else ok = false;
            }
            bool finite = fabsf(l) < CUDART_INF_F;
#pragma unroll
            for (uint32_t d = 0; d < DHP; ++d) finite = finite && fabsf(o[d]) < CUDART_INF_F;
            if (!ok || bad) l = CUDART_NAN_F;
            const uint32_t again = __ballot_sync(0xffffffffu, is && ok && !bad && !finite);
            if (lane == 0) odd[w * 4 + (warp & 3u)] = again;
            if (is) {
                const size_t to = splits > 1 ? ((size_t)split * a.c.T * a.H) * dh + at : at;
                float* out = (splits > 1 ? part : a.out) + to;
                const float by = splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (uint32_t d = 0; d < DHP; d += 4)
                    if (d < dh) *reinterpret_cast<float4*>(out + d) = make_float4(o[d] * by, o[d + 1] * by, o[d + 2] * by, o[d + 3] * by);
                if (splits > 1) stat[to / dh] = make_float2(m, l);
            }
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
    if (warp >= 4)
        for (uint32_t i = warp - 4; i < rows; i += 8) {
            if (!bad_page && !(odd[i >> 5] >> (i & 31u) & 1u)) continue;
            const uint32_t gi = row0 + i, tok = gi / a.rep;
            const size_t at = (size_t)(s.q0 + tok) * a.H + h * a.rep + gi % a.rep, to = splits > 1 ? (size_t)split * a.c.T * a.H + at : at;
            float* out = (splits > 1 ? part : a.out) + to * dh;
            if (bad_page) {
                for (uint32_t d = lane; d < dh; d += 32) out[d] = CUDART_NAN_F;
                if (splits > 1 && lane == 0) stat[to] = make_float2(0.f, CUDART_NAN_F);
            } else {
                row_again<__half>(a, b, h, s.first + (int)tok, kt, t0, t1, a.q + at * dh, out, splits > 1 ? stat + to : nullptr);
            }
        }
}

// A warp per row: its parts, weighted by their maxima.
__global__ void __launch_bounds__(256) attn_chunk_merge_kernel(const __grid_constant__ AttnCall a, uint32_t splits, const float* part, const float2* stat) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u, dh = a.c.dh;
    const size_t rows = (size_t)a.c.T * a.H, row = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const uint32_t t = (uint32_t)(row / a.H), b = kv_find_seq(a.c, t);
    if (b >= a.c.B) return;
    const KvSeq s = kv_seq(a.c, b);
    if (s.lost || t < s.q0 || t - s.q0 >= s.n || (unsigned long long)s.n * a.rep <= a.few) return;
    float M = -CUDART_INF_F, L = 0.f;
    for (uint32_t i = 0; i < splits; ++i) M = fmaxf(M, stat[i * rows + row].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t i = 0; i < splits; ++i) {
        const float2 ml = stat[i * rows + row];
        const float w = ml.x == -CUDART_INF_F ? 0.f : pow2(ml.x - M);
        L = fmaf(w, ml.y, L);
        if (4 * lane < dh) {
            const float4 x = *reinterpret_cast<const float4*>(part + (i * rows + row) * dh + 4 * lane);
            o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
        }
    }
    const float by = L == 0.f ? 0.f : 1.f / L;
    if (4 * lane < dh) *reinterpret_cast<float4*>(a.out + row * dh + 4 * lane) = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
}

template <int DHP>
bool go(const AttnCall& a, const ChunkPlan& pl, float* scratch, cudaStream_t st) {
    auto* kernel = attn_chunk_kernel<DHP>;
    static PerDevice<bool> ready;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || !ready.get(dev, [=](bool&) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Chunk<DHP>::Smem) == cudaSuccess; }))
        return fail("attention: shared memory attribute: %s", cudaGetErrorString(cudaGetLastError()));
    const unsigned long long ctas = (unsigned long long)a.c.KVH * pl.splits * pl.slots;
    if (ctas > 0x7fffffffull) return fail("attention: %llu tiles of query rows", ctas);
    const size_t rows = (size_t)a.c.T * a.H;
    float* part = scratch;
    float2* stat = reinterpret_cast<float2*>(part + pl.splits * rows * a.c.dh);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = Chunk<DHP>::Smem; cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, a, pl.splits, part, stat);
    note_launch();
    if (!check_launch("attn_chunk")) return false;
    if (pl.splits == 1) return true;
    cfg.gridDim = dim3((unsigned)((rows + 7) / 8)); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
    cudaLaunchKernelEx(&cfg, attn_chunk_merge_kernel, a, pl.splits, (const float*)part, (const float2*)stat);
    note_launch();
    return check_launch("attn_chunk_merge");
}

}  // namespace

ChunkPlan plan_attn_chunk(uint32_t T, uint32_t B, uint32_t KVH, uint32_t rep, uint32_t few) {
    const unsigned long long rows = (unsigned long long)T * rep, least = (rows + 2 * kRows - 1) / (2 * kRows);
    ChunkPlan pl;
    pl.slots = (uint32_t)(rows / (2 * kRows) + std::min<unsigned long long>(B, rows / (few + 1ull)));
    pl.splits = (uint32_t)std::max<unsigned long long>(1, std::min<unsigned long long>(148 / (least * KVH), 16));
    return pl;
}

size_t attn_chunk_scratch(const ChunkPlan& pl, uint32_t T, uint32_t H, uint32_t dh) {
    return pl.splits == 1 ? 0 : (size_t)pl.splits * T * H * (dh * sizeof(float) + sizeof(float2));
}

bool launch_attn_chunk(const AttnCall& a, const ChunkPlan& pl, float* scratch, cudaStream_t st) {
    return a.c.dh <= 64 ? go<64>(a, pl, scratch, st) : go<128>(a, pl, scratch, st);
}

}  // namespace tmc
