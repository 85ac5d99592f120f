// attn_few.cu — attention of sequences that bring few query rows (a decode step, a handful of drafted tokens) over a paged cache.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m), s = scale log2(e) q k, with the running maximum m of one pass over the keys.
//
// Bound: HBM, every visible K and V row is read once for all the query rows of its head: 64 sequences of 150 to 8100 positions, 32 / 8 heads of
// 128 in fp16, 1.10 GB in 185 us, 5.9 TB/s (0.91 of the copy rate); fp32 caches 4.4 TB/s. Short calls are bound by their trips to memory
// one after the other (lengths, page, rows, merge): one token at 601 positions 7.0 us.
//   * LIST: the work of the whole batch - (sequence, K/V head, tile of keys), tiles in order - is one list of which every CTA takes an
//     equal stretch, whatever the lengths are; a CTA finishes the units that lie in its stretch and leaves a partial of the one or two that
//     it shares, which a second kernel merges. Else, where the host can tell that few tiles are in reach, a unit is a cluster's, which
//     merges through distributed shared memory in the same launch (one token at 601 positions 8.9 -> 7.0 us, 4096 keys of one 13.3 -> 11.4).
//   * A warp takes 16 (8) keys of every tile through a ring of its own (cp.async, one lane looks up one row's page), so nothing in the
//     loop waits for another warp.
//   * Both products run on mma.sync with the query rows as its 16 rows: the keys' and values' bytes are the traffic, so the padding
//     costs nothing that counts. Results are to be as good as fp32's, so an fp32 operand is two fp16 parts (two tf32 parts against
//     fp32 caches), high and low: error 2^-22. With at most 8 rows the parts are the two halves of the 16 rows: one product.
//     Against fp16 caches q is scaled by a power of two per row and weights by 2^14 (kUp).
//   * The output is summed in fp32 registers, a step's keys at a time: a tensor core's own running sum is cut, not rounded, at every step.
//   * Over fp32 caches the same kernel takes longer chunks, 16 rows at a time (a.tiled): 700 tokens with a window of 255, 32 / 4 heads of 64,
//     76 us, bound by the instructions that split K and V for every 16 rows.
//   * A value that is masked for one row but not for another meets a weight of 0 in the product, which is NaN if the value is not
//     finite. So a result that is not finite is computed again row by row, where masked keys are skipped; one beyond 2^100, too, lest
//     the sum of an fp32 cache's largest values be infinite where their mean is not.
#include "attn_rows.cuh"
#include "common.cuh"
#include "pdl.cuh"
#include "per_device.h"

#include <algorithm>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <type_traits>

namespace tmc {
namespace {

constexpr uint32_t kWarps = 4;                              // of a CTA; each takes its share of every tile
// One launch may walk so many tiles more than two would: a tile takes some 0.6 us, the second launch 3 to 4.
constexpr uint32_t kClusterTiles = 6;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// x, y as fp16 pairs: the rounded values and what the rounding left
__device__ __forceinline__ void parts(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = half2_bits(x - f.x, y - f.y);
}
__device__ __forceinline__ void parts(float x, uint32_t& hi, uint32_t& lo) {             // as tf32, both rounded: the product would cut
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}

// ---- the list of work ------------------------------------------------------------------------------------------------
template <uint32_t TILE> struct Unit : KeyTiles<TILE> {
    KvSeq s;
    bool bad;                       // its rows are NaN
};
__device__ __forceinline__ uint32_t row_tiles(const AttnCall& a, uint32_t b, bool note) {        // 16 rows each, of a sequence with more than `few`
    const KvSeq s = kv_seq(a.c, b);
    if (s.lost && note) note_bad_batch(a.status);
    return s.n * a.rep <= a.few ? 0u : (s.n * a.rep + kFewRows - 1) / kFewRows;
}
// The rows of sequence b together (r0 = 0 and not more than `few`), or 16 of them from r0 on
template <uint32_t TILE> __device__ Unit<TILE> unit_of(const AttnCall& a, uint32_t b, uint32_t r0) {
    Unit<TILE> u;
    u.s = kv_seq(a.c, b);
    u.bad = u.s.bad || u.s.n > a.max_q;
    if (a.tiled) {
        u.set(kv_span(a.mask, u.s.first + (int)(r0 / a.rep), u.s.first + (int)((min(r0 + kFewRows, u.s.n * a.rep) - 1) / a.rep)), u.bad);
        return u;
    }
    const uint32_t rows = u.s.n <= a.few ? u.s.n * a.rep : a.few + 1;       // no overflow
    if (u.s.n == 0 || (rows > a.few && a.others)) { u.tiles = 0; return u; }
    u.set(kv_span(a.mask, u.s.first, (int)u.s.len - 1), u.bad);
    return u;
}

struct Part { int b, h, last, first; };     // of CTA c: the unit in whose middle its stretch begins, the CTA that ends it, whether c is the first that begins in it

// Two CTAs per SM: 700 tokens of 32 / 4 heads of 64 in fp32 took 144 us with one (four stages), 84 with two (three). fp32 rows of 128 dims come
// eight keys at a time for that: 32 sequences of 500 to 4000 positions, 32 / 8 heads, 240 us with 16 and one CTA, 138 so.
template <typename T, int DHP, bool PAIR> struct Few {
    static constexpr uint32_t Step = sizeof(T) == 4 && DHP == 128 ? 8 : 16, Tile = kWarps * Step;        // keys of a warp's share of a tile; of a tile
    static constexpr uint32_t Rows = PAIR ? 8 : 16;
    static constexpr uint32_t RowBytes = DHP * sizeof(T), StageBytes = 2 * Step * RowBytes;      // K and V of a warp's step
    static constexpr uint32_t Stages = sizeof(T) == 4 ? (DHP == 128 && !PAIR ? 2 : 3) : (PAIR ? 3 : 2) * (128 / DHP);
    static constexpr uint32_t Ring = kWarps * Stages * StageBytes, Merge = kWarps * Rows * DHP * 4;
    static constexpr uint32_t Smem = Ring + Merge;
    static constexpr uint32_t PerSm = 2;
    static_assert(Smem <= 114688, "two fit an SM");
};

// LIST: the stretches of the list. Else a unit per cluster of `splits` CTAs, which share its keys and merge through distributed shared
// memory: the rows of a sequence and K/V head, or (a.tiled) 16 of them.
template <typename T, int DHP, bool PAIR, bool LIST>
__global__ void __launch_bounds__(32 * kWarps, Few<T, DHP, PAIR>::PerSm) attn_few_kernel(const __grid_constant__ AttnCall a, float* part, float2* stat, Part* meta, uint32_t splits) {
    using F = Few<T, DHP, PAIR>;
    constexpr uint32_t kTile = F::Tile, kStep = F::Step, KB = kStep / 8;        // blocks of 8 keys of a step
    constexpr bool kHalf = sizeof(T) == 2;
    static_assert(!kHalf || KB == 2);
    constexpr uint32_t RB = F::RowBytes, SB = F::StageBytes, S = F::Stages, ROWS = F::Rows, NB = DHP / 8, NR = PAIR ? 1 : 2;
    constexpr uint32_t KS = DHP / 16;                       // 16 dims at a time, whatever the type
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ unsigned long long sums[kWarps];
    __shared__ uint32_t at_b, at_h, at_t;
    __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS];
    __shared__ int sm_bad[2];
    __shared__ float2 cta_ml[ROWS];                         // what a cluster's CTAs merge: maxima and sums; the outputs lie in the ring
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
    pdl_enter();
    const uint32_t dh = a.c.dh, KVH = a.c.KVH;

    // ---- this CTA's stretch of the list ----
    unsigned long long x0, x1, total;
    uint32_t r0 = 0;                                        // a.tiled: the unit's first row
    const uint32_t split = LIST ? 0u : blockIdx.x % splits;
    Unit<kTile> u0;
    if constexpr (!LIST) {
        const uint32_t unit = blockIdx.x / splits;
        uint32_t b = unit / KVH;
        if (tid == 0) { at_h = unit % KVH; sm_bad[0] = sm_bad[1] = 0; }
        if (a.tiled) {
            if (tid == 0) at_b = a.c.B;
            const uint32_t per = (a.c.B + blockDim.x - 1) / blockDim.x, b0 = min(a.c.B, tid * per), b1 = min(a.c.B, b0 + per);
            uint32_t mine = 0;
            for (uint32_t i = b0; i < b1; ++i) mine += row_tiles(a, i, blockIdx.x == 0);
            uint32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= (uint32_t)o) incl += y; }
            if (lane == 31) sums[warp] = incl;
            __syncthreads();
            uint32_t before = incl - mine, all = 0;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) { if (w == warp) before += all; all += (uint32_t)sums[w]; }
            const uint32_t slot = all - 1 - unit / KVH;     // from the last on; wraps where there is no such unit
            if (slot >= before && slot < before + mine)
                for (uint32_t i = b0; i < b1; ++i) {
                    const uint32_t n = row_tiles(a, i, false);
                    if (slot < before + n) { at_b = i; at_t = slot - before; break; }
                    before += n;
                }
            __syncthreads();
            b = at_b;
            if (b == a.c.B) return;                         // the whole cluster
            r0 = at_t * kFewRows;
        }
        u0 = unit_of<kTile>(a, b, r0);
        if (u0.s.lost && at_h == 0 && tid == 0 && split == 0) note_bad_batch(a.status);
        if (u0.tiles == 0) return;
        x0 = (unsigned long long)u0.tiles * split / splits; x1 = (unsigned long long)u0.tiles * (split + 1) / splits;
        __syncthreads();
        if (tid == 0) { at_b = b; at_t = (uint32_t)x0; }
        __syncthreads();
    } else {
        const uint32_t per = (a.c.B + blockDim.x - 1) / blockDim.x, b0 = min(a.c.B, tid * per), b1 = min(a.c.B, b0 + per);
        unsigned long long mine = 0;
        for (uint32_t b = b0; b < b1; ++b) {
            const Unit<kTile> u = unit_of<kTile>(a, b, 0);
            if (u.s.lost && blockIdx.x == 0) note_bad_batch(a.status);
            mine += (unsigned long long)u.tiles * KVH;
        }
        unsigned long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= (uint32_t)o) incl += y; }
        if (lane == 31) sums[warp] = incl;
        if (tid == 0) { at_b = a.c.B; at_h = at_t = 0; sm_bad[0] = sm_bad[1] = 0; }
        __syncthreads();
        total = 0;
        unsigned long long before = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) { if (w == warp) before = total; total += sums[w]; }
        const unsigned long long per_cta = total / gridDim.x, rem = total % gridDim.x, c = blockIdx.x;
        x0 = c * per_cta + min(c, rem); x1 = x0 + per_cta + (c < rem ? 1 : 0);
        unsigned long long x = before + incl - mine;
        if (x0 >= x && x0 < x + mine) {                     // the stretch begins in one of this thread's sequences
            for (uint32_t b = b0; b < b1; ++b) {
                const Unit<kTile> u = unit_of<kTile>(a, b, 0);
                const unsigned long long n = (unsigned long long)u.tiles * KVH;
                if (x0 < x + n) {
                    const uint32_t h = (uint32_t)((x0 - x) / u.tiles), t = (uint32_t)((x0 - x) % u.tiles);
                    at_b = b; at_h = h; at_t = t;
                    Part p{-1, 0, 0, 0};
                    if (t && x1 > x0) {
                        const unsigned long long start = x0 - t, end = start + u.tiles - 1, line = rem * (per_cta + 1);
                        p.b = (int)b; p.h = (int)h;
                        p.last = (int)(end < line ? end / (per_cta + 1) : rem + (end - line) / per_cta);
                        const unsigned long long back = x0 - per_cta - (c - 1 < rem ? 1 : 0);         // where CTA c - 1 begins
                        p.first = start >= back;
                    }
                    meta[blockIdx.x] = p;
                    break;
                }
                x += n;
            }
        }
        __syncthreads();
        if (x1 == x0) {
            if (tid == 0) meta[blockIdx.x] = Part{-1, 0, 0, 0};
            return;
        }
    }

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (S * SB);
    float* const merge = reinterpret_cast<float*>(smem + F::Ring);
    if (dh < DHP) {                                         // dims that no copy writes
        for (uint32_t i = tid * 16; i < F::Ring; i += blockDim.x * 16) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    // ---- the copies: a cursor of their own, Stages - 1 tiles ahead ----
    uint32_t lb = at_b, lh = at_h, lt = at_t, left = (uint32_t)(x1 - x0), slot = 0;
    uint32_t no_page = 0;                                   // bit of a stage: a page was not there
    Unit<kTile> lu = !LIST ? u0 : unit_of<kTile>(a, lb, 0);
    auto request = [&]() {
        if (left) {
            const uint32_t place = lt * kTile + warp * kStep + lane % kStep;
            size_t at = 0;
            const bool in = place < lu.count;
            bool ok = true;
            if (in) ok = kv_row(a.c, lb, lu.key(place), &at);
            no_page = no_page & ~(1u << slot) | (__any_sync(0xffffffffu, !ok) ? 1u << slot : 0u);
            at = (at + (size_t)lh * a.c.page * dh) * sizeof(T);
            const uint32_t chunks = dh * (uint32_t)sizeof(T) / 16, lo = (uint32_t)at, hi = (uint32_t)(at >> 32);
            const uint32_t there = __ballot_sync(0xffffffffu, in && ok);
            constexpr uint32_t C = RB / 16, RP = 32 / C > 0 ? 32 / C : 1;            // chunks of a row; rows of a round
            const uint32_t dst = ring + slot * SB;
#pragma unroll
            for (uint32_t i = 0; i < kStep / RP; ++i) {
                const uint32_t r = i * RP + lane / C, ch = lane % C;
                const size_t off = (size_t)__shfl_sync(0xffffffffu, lo, r) | (size_t)__shfl_sync(0xffffffffu, hi, r) << 32;
                if (ch < chunks) {
                    const uint32_t n = there >> r & 1u ? 16u : 0u;
                    const uint32_t kx = kHalf ? r & 7u : (r & 3u) << 1 | (r >> 2 & 1u);
                    copy16(dst + r * RB + ((ch ^ kx) << 4), (const uint8_t*)a.c.k + off + ch * 16, n);
                    copy16(dst + kStep * RB + r * RB + ((ch ^ (r & 7u)) << 4), (const uint8_t*)a.c.v + off + ch * 16, n);
                }
            }
            if (--left && ++lt == lu.tiles) {
                lt = 0;
                if (++lh == KVH) {
                    lh = 0;
                    lu.tiles = 0;
                    while (lu.tiles == 0 && ++lb < a.c.B) lu = unit_of<kTile>(a, lb, 0);
                    if (lb >= a.c.B) left = 0;              // the arrays are not what they were: nothing behind them is read
                }
            }
        }
        if (++slot == S) slot = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (uint32_t i = 0; i + 1 < S; ++i) request();

    auto number_of = [&](const Unit<kTile>& u, uint32_t h, uint32_t r) {        // of a row of a unit in q and out
        const uint32_t i = r / a.rep;
        return (size_t)(u.s.q0 + i) * a.H + h * a.rep + (r - i * a.rep);
    };
    // ---- the units of the stretch ----
    uint32_t b = at_b, h = at_h, t = at_t, todo = (uint32_t)(x1 - x0), use = 0, turn = 0;
    Unit<kTile> u = !LIST ? u0 : unit_of<kTile>(a, b, 0);
    for (;;) {
        const uint32_t t0 = t, t1 = min(u.tiles, t + todo), rows = min(u.s.n * a.rep - r0, ROWS);
        int pos[NR];
        float back[NR], m[NR], l[NR], o[NB][2 * NR];        // back: what undoes q's power of two
        uint32_t qf[NR][KS][4];                             // fp16: the fragments, both parts; fp32: the values of a row, or their high parts
        constexpr bool KEEP = !kHalf && (DHP == 64 || PAIR);  // fp32: q's low parts are kept too, where registers are left
        uint32_t qlow[KEEP ? NR : 1][KEEP ? KS : 1][4];
        {
            const float* qp[NR];
#pragma unroll
            for (uint32_t n = 0; n < NR; ++n) {
                const uint32_t r = r0 + g + 8 * n, i = r / a.rep;
                const bool is = g + 8 * n < rows;
                pos[n] = is ? u.s.first + (int)i : -1;
                qp[n] = is ? a.q + number_of(u, h, r) * dh : nullptr;
                m[n] = -CUDART_INF_F; l[n] = 0.f; back[n] = 1.f;
                float2 raw[2 * KS];
#pragma unroll
                for (uint32_t k = 0; k < 2 * KS; ++k) {
                    const uint32_t d = k * 8 + 2 * t4;
                    raw[k] = make_float2(0.f, 0.f);
                    if (is && d < dh) raw[k] = *reinterpret_cast<const float2*>(qp[n] + d);
                    raw[k].x *= a.scale * kLog2e; raw[k].y *= a.scale * kLog2e;
                }
                if constexpr (kHalf) {
                    float top = 0.f;
#pragma unroll
                    for (uint32_t k = 0; k < 2 * KS; ++k) top = fmaxf(top, fmaxf(fabsf(raw[k].x), fabsf(raw[k].y)));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 120);      // the row's largest to [2^13, 2^14)
                    const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                    back[n] = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
                    for (uint32_t k = 0; k < 2 * KS; ++k) {
                        uint32_t hi, lo;
                        parts(raw[k].x * up, raw[k].y * up, hi, lo);
                        if constexpr (PAIR) { qf[0][k / 2][2 * (k & 1)] = hi; qf[0][k / 2][2 * (k & 1) + 1] = lo; }
                        else { qf[0][k / 2][2 * (k & 1) + n] = hi; qf[NR - 1][k / 2][2 * (k & 1) + n] = lo; }
                    }
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 2 * KS; ++k) {
                        if constexpr (KEEP) {
                            parts(raw[k].x, qf[n][k / 2][2 * (k & 1)], qlow[n][k / 2][2 * (k & 1)]);
                            parts(raw[k].y, qf[n][k / 2][2 * (k & 1) + 1], qlow[n][k / 2][2 * (k & 1) + 1]);
                        } else { qf[n][k / 2][2 * (k & 1)] = __float_as_uint(raw[k].x); qf[n][k / 2][2 * (k & 1) + 1] = __float_as_uint(raw[k].y); }
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < NB; ++i)
#pragma unroll
            for (uint32_t k = 0; k < 2 * NR; ++k) o[i][k] = 0.f;
        bool lost_page = false;
        const int p_least = u.s.first + (int)(r0 / a.rep);
        const uint32_t from = (uint32_t)window_from(a.mask, (int)u.end - 1);       // the last row's window begins last

        for (; t < t1; ++t) {
            request();
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            __syncwarp();
            const uint32_t kat = ring + use * SB, vat = kat + kStep * RB, u0 = t * kTile + warp * kStep;        // the first place of this warp's step
            if (no_page >> use & 1u) lost_page = true;
            if (u0 < u.count) {
                float s[KB][4] = {}, low[KB][4] = {};         // what the low parts add is summed apart: every step cuts the sum that it adds to
                if constexpr (kHalf) {
                    const uint32_t key = (lane >> 4) * 8 + (lane & 7u), row = kat + key * RB, c0 = lane >> 3 & 1u;
#pragma unroll
                    for (uint32_t k = 0; k < KS; ++k) {
                        uint32_t f[4];
                        ldsm4(f, row + (((2 * k + c0) ^ (key & 7u)) << 4));
#pragma unroll
                        for (uint32_t n = 0; n < NR; ++n) { mma_f16(n ? low[0] : s[0], qf[n][k], f[0], f[1]); mma_f16(n ? low[1] : s[1], qf[n][k], f[2], f[3]); }
                    }
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 2 * KS; ++k) {
                        uint32_t ah[4], al[4];              // PAIR: ah holds both parts
#pragma unroll
                        for (uint32_t n = 0; n < NR; ++n) {
                            uint32_t h0 = qf[n][k / 2][2 * (k & 1)], h1 = qf[n][k / 2][2 * (k & 1) + 1], l0, l1;
                            if constexpr (KEEP) { l0 = qlow[n][k / 2][2 * (k & 1)]; l1 = qlow[n][k / 2][2 * (k & 1) + 1]; }
                            else {
                                asm volatile("" : "+r"(h0), "+r"(h1));       // split here, at every tile: split once, outside, they would not fit the registers
                                parts(__uint_as_float(h0), h0, l0); parts(__uint_as_float(h1), h1, l1);
                            }
                            if constexpr (PAIR) { ah[0] = h0; ah[1] = l0; ah[2] = h1; ah[3] = l1; }
                            else { ah[n] = h0; al[n] = l0; ah[2 + n] = h1; al[2 + n] = l1; }
                        }
#pragma unroll
                        for (uint32_t nb = 0; nb < KB; ++nb) {
                            const uint32_t key = nb * 8 + g, kx = (key & 3u) << 1 | (key >> 2 & 1u);
                            float2 f;
                            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(kat + key * RB + (((2 * k + (t4 >> 1)) ^ kx) << 4) + (t4 & 1u) * 8));
                            uint32_t h0, l0, h1, l1;
                            parts(f.x, h0, l0); parts(f.y, h1, l1);
                            mma_tf32(s[nb], ah, h0, h1);
                            mma_tf32(low[nb], ah, l0, l1);
                            if constexpr (!PAIR) mma_tf32(low[nb], al, h0, h1);
                        }
                    }
                }
                if constexpr (!kHalf || !PAIR) {
#pragma unroll
                    for (uint32_t i = 0; i < 4 * KB; ++i) s[i >> 2][i & 3] += low[i >> 2][i & 3];
                }
                const bool whole = u.seen(u0, kStep, p_least, from);
                float corr[NR];
                uint32_t ph[NR][2 * KB];                         // the weights as the second product's rows: PAIR: [0] both parts; else high, low
#pragma unroll
                for (uint32_t n = 0; n < NR; ++n) {
                    float x[2 * KB];
#pragma unroll
                    for (uint32_t i = 0; i < 2 * KB; ++i) {
                        if constexpr (PAIR) x[i] = (s[i >> 1][i & 1] + s[i >> 1][2 + (i & 1)]) * back[0];
                        else x[i] = s[i >> 1][2 * n + (i & 1)] * back[n];
                    }
                    if (!whole) {
#pragma unroll
                        for (uint32_t i = 0; i < 2 * KB; ++i)
                            if (!kv_sees(a.mask, pos[n], (int)u.key(u0 + (i >> 1) * 8 + 2 * t4 + (i & 1)))) x[i] = -CUDART_INF_F;
                    }
                    float mn = fmaxf(x[0], x[1]);
                    if constexpr (KB == 2) mn = fmaxf(mn, fmaxf(x[2], x[3]));
                    mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
                    mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
                    mn = fmaxf(mn, m[n]);
                    const float base = mn == -CUDART_INF_F ? 0.f : mn;
                    corr[n] = pow2(m[n] - base);
                    m[n] = mn;
#pragma unroll
                    for (uint32_t i = 0; i < 2 * KB; ++i) x[i] = pow2(x[i] - base + kUp<T>);
                    float add = x[0] + x[1];
                    if constexpr (KB == 2) add += x[2] + x[3];
                    l[n] = fmaf(l[n], corr[n], add);
                    if constexpr (kHalf) {
                        if constexpr (PAIR) { parts(x[0], x[1], ph[0][0], ph[0][1]); parts(x[2], x[3], ph[0][2], ph[0][3]); }
                        else { parts(x[0], x[1], ph[0][n], ph[NR - 1][n]); parts(x[2], x[3], ph[0][2 + n], ph[NR - 1][2 + n]); }
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 2 * KB; ++i) ph[n][i] = __float_as_uint(x[i]);
                    }
                }
                if constexpr (kHalf) {
                    const uint32_t key = (lane >> 3 & 1u) * 8 + (lane & 7u), row = vat + key * RB, c0 = lane >> 4;
#pragma unroll
                    for (uint32_t i = 0; i < NB / 2; ++i) {
                        uint32_t f[4];
                        ldsm4_t(f, row + (((2 * i + c0) ^ (key & 7u)) << 4));
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            float d[4] = {};
#pragma unroll
                            for (uint32_t n = 0; n < NR; ++n) mma_f16(d, ph[n], f[2 * k], f[2 * k + 1]);
                            float (&to)[2 * NR] = o[2 * i + k];
                            if constexpr (PAIR) { to[0] = fmaf(to[0], corr[0], d[0] + d[2]); to[1] = fmaf(to[1], corr[0], d[1] + d[3]); }
                            else {
#pragma unroll
                                for (uint32_t e = 0; e < 4; ++e) to[e] = fmaf(to[e], corr[NR == 1 ? 0 : e >> 1], d[e]);
                            }
                        }
                    }
                } else {
                    uint32_t ah[KB][4], al[KB][4];            // key 2 t of a block of 8 is row t of the product's operand, key 2 t + 1 row t + 4
#pragma unroll
                    for (uint32_t nb = 0; nb < KB; ++nb)
#pragma unroll
                        for (uint32_t n = 0; n < NR; ++n) {
                            uint32_t h0, l0, h1, l1;
                            parts(__uint_as_float(ph[n][2 * nb]), h0, l0);
                            parts(__uint_as_float(ph[n][2 * nb + 1]), h1, l1);
                            if constexpr (PAIR) { ah[nb][0] = h0; ah[nb][1] = l0; ah[nb][2] = h1; ah[nb][3] = l1; }
                            else { ah[nb][n] = h0; al[nb][n] = l0; ah[nb][2 + n] = h1; al[nb][2 + n] = l1; }
                        }
#pragma unroll
                    for (uint32_t i = 0; i < NB; ++i) {
                        float d[4] = {};
#pragma unroll
                        for (uint32_t nb = 0; nb < KB; ++nb) {
                            uint32_t vh[2], vl[2];
#pragma unroll
                            for (uint32_t k = 0; k < 2; ++k) {
                                const uint32_t key = nb * 8 + 2 * t4 + k;
                                float f;
                                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(vat + key * RB + (((2 * i + (g >> 2)) ^ (key & 7u)) << 4) + (g & 3u) * 4));
                                parts(f, vh[k], vl[k]);
                            }
                            mma_tf32(d, ah[nb], vh[0], vh[1]);
                            mma_tf32(d, ah[nb], vl[0], vl[1]);
                            if constexpr (!PAIR) mma_tf32(d, al[nb], vh[0], vh[1]);
                        }
                        float (&to)[2 * NR] = o[i];
                        if constexpr (PAIR) { to[0] = fmaf(to[0], corr[0], d[0] + d[2]); to[1] = fmaf(to[1], corr[0], d[1] + d[3]); }
                        else {
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) to[e] = fmaf(to[e], corr[NR == 1 ? 0 : e >> 1], d[e]);
                        }
                    }
                }
            }
            __syncwarp();                                   // the stage is free for the next request
            if (++use == S) use = 0;
        }

        // ---- the warps' results together ----
#pragma unroll
        for (uint32_t n = 0; n < NR; ++n) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
            if (t4 == 0) { sm_m[warp][g + 8 * n] = m[n]; sm_l[warp][g + 8 * n] = l[n]; }
#pragma unroll
            for (uint32_t i = 0; i < NB; ++i)
                *reinterpret_cast<float2*>(merge + ((size_t)warp * ROWS + g + 8 * n) * DHP + i * 8 + 2 * t4) = make_float2(o[i][2 * n], o[i][2 * n + 1]);
        }
        if ((lost_page || u.bad) && lane == 0) sm_bad[turn] = 1;
        __syncthreads();
        const bool bad = sm_bad[turn], all = LIST ? t0 == 0 && t1 == u.tiles : splits == 1;
        const size_t slot = 2 * (size_t)blockIdx.x + (t0 == 0);            // of a unit that began before: 0; that goes on behind: 1
        float* const po = LIST ? part + slot * ROWS * dh : reinterpret_cast<float*>(smem);
        float2* const ps = LIST ? stat + slot * ROWS : cta_ml;
        bool again = false;
        if (tid < dh) {
            for (uint32_t r = 0; r < rows; ++r) {
                float M = -CUDART_INF_F, x = 0.f, L = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][r]);
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) {
                    const float f = sm_m[w][r] == -CUDART_INF_F ? 0.f : pow2(sm_m[w][r] - M);
                    x = fmaf(f, merge[((size_t)w * ROWS + r) * DHP + tid], x);
                    L = fmaf(f, sm_l[w][r], L);
                }
                again = again || !in_reach<T>(x) || !(fabsf(L) < CUDART_INF_F);
                if (bad) L = CUDART_NAN_F;
                if (all) {
                    a.out[number_of(u, h, r0 + r) * dh + tid] = L == 0.f ? 0.f : x / L;
                } else {
                    po[(size_t)r * dh + tid] = x;
                    if (tid == 0) ps[r] = make_float2(M, L);
                }
            }
            if (!a.tiled && bad)                            // more rows than were promised
                for (uint32_t r = rows; r < u.s.n * a.rep; ++r) a.out[number_of(u, h, r) * dh + tid] = CUDART_NAN_F;
        }
        if (bad && tid == 0) note_bad_batch(a.status);
        if (tid == 0) sm_bad[turn ^ 1u] = 0;
        if (__syncthreads_or(again && !bad)) {
            for (uint32_t r = warp; r < rows; r += kWarps) {
                const size_t row = number_of(u, h, r0 + r);
                row_again<T, kTile>(a, b, h, u.s.first + (int)((r0 + r) / a.rep), u, t0, t1, a.q + row * dh, all ? a.out + row * dh : po + (size_t)r * dh, all ? nullptr : ps + r);
            }
            if (!LIST) __syncthreads();
        }
        if constexpr (!LIST) {
            if (splits == 1) return;
            cluster_sync();
            const uint32_t at_o = (uint32_t)__cvta_generic_to_shared(smem), at_ml = (uint32_t)__cvta_generic_to_shared(cta_ml);
            for (uint32_t i = split * blockDim.x + tid; i < rows * dh; i += splits * blockDim.x) {
                const uint32_t r = i / dh;
                float M = -CUDART_INF_F, L = 0.f, y = 0.f;
#pragma unroll 4
                for (uint32_t k = 0; k < splits; k += 2) {  // a power of two, so two at a time
                    const float2 m0 = ld_cta2(map_cta(at_ml + 8 * r, k)), m1 = ld_cta2(map_cta(at_ml + 8 * r, k + 1));
                    const float x0 = ld_cta(map_cta(at_o + 4 * i, k)), x1 = ld_cta(map_cta(at_o + 4 * i, k + 1));
                    const float mn = fmaxf(M, fmaxf(m0.x, m1.x)), base = mn == -CUDART_INF_F ? 0.f : mn, f = pow2(M - base), f0 = pow2(m0.x - base), f1 = pow2(m1.x - base);
                    L = fmaf(L, f, fmaf(f0, m0.y, f1 * m1.y));
                    y = fmaf(y, f, fmaf(f0, x0, f1 * x1));
                    M = mn;
                }
                a.out[number_of(u, h, r0 + r) * dh + (i - r * dh)] = L == 0.f ? 0.f : y / L;
            }
            cluster_sync();                                 // nobody leaves while its shared memory is read
            return;
        }
        turn ^= 1u;
        todo -= t1 - t0;
        if (!todo) return;
        t = 0;
        if (++h == KVH) {
            h = 0;
            u.tiles = 0;
            while (u.tiles == 0 && ++b < a.c.B) u = unit_of<kTile>(a, b, 0);
            if (b >= a.c.B) return;
        }
    }
}

// One CTA per stretch that begins inside a unit, of which the first of a unit merges all of its parts: the last of the CTA before, and the
// first of its own and of those behind it. Rows over blockIdx.y; four threads per dim take every fourth part, a thread per part its
// weight. Bound by its trips to L2: the first 32 parts are on their way while the weights are worked out.
constexpr uint32_t kMergeGroups = 4;
__global__ void __launch_bounds__(kMergeGroups * 128) attn_few_merge_kernel(const __grid_constant__ AttnCall a, const float* part, const float2* stat, const Part* meta, uint32_t slot_rows) {
    constexpr uint32_t BATCH = 8, G = kMergeGroups, NT = G * 128;
    static_assert(NT >= kFewCtas + 1, "a thread per part");
    __shared__ float so[G][128], weight[NT];
    __shared__ float2 sml[NT / 32];
    pdl_enter();
    const uint32_t c = blockIdx.x + 1, r = blockIdx.y, d = threadIdx.x, grp = threadIdx.y, tid = grp * 128 + d, dh = a.c.dh;
    const Part p = meta[c];
    if (p.b < 0 || !p.first) return;
    const KvSeq s = kv_seq(a.c, (uint32_t)p.b);
    if (r >= s.n * a.rep) return;
    const uint32_t parts = (uint32_t)p.last - c + 2;
    float* const to = a.out + ((size_t)(s.q0 + r / a.rep) * a.H + p.h * a.rep + r % a.rep) * dh + d;
    auto row_of = [&](uint32_t i) { return (size_t)(2 * (c + i) - (i ? 2 : 1)) * slot_rows + r; };      // i = 0: slot 1 of CTA c - 1; else slot 0 of CTA c + i - 1
    if (parts <= BATCH) {                                   // a unit that two or three stretches share: a thread per dim, no waiting for others
        if (grp || d >= dh) return;
        float2 ml[BATCH];
        float x[BATCH], M = -CUDART_INF_F, L = 0.f, o = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < BATCH; ++i)
            if (i < parts) { ml[i] = __ldcg(stat + row_of(i)); x[i] = __ldcg(part + row_of(i) * dh + d); }
#pragma unroll
        for (uint32_t i = 0; i < BATCH; ++i)
            if (i < parts) M = fmaxf(M, ml[i].x);
#pragma unroll
        for (uint32_t i = 0; i < BATCH; ++i)
            if (i < parts) {
                const float w = ml[i].x == -CUDART_INF_F ? 0.f : pow2(ml[i].x - M);
                o = fmaf(w, x[i], o); L = fmaf(w, ml[i].y, L);
            }
        *to = L == 0.f ? 0.f : o / L;
        return;
    }
    float v[BATCH];
    auto request = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k)
            if (i0 + G * k + grp < parts && d < dh) v[k] = __ldcg(part + row_of(i0 + G * k + grp) * dh + d);
    };
    request(0);
    float2 ml = make_float2(-CUDART_INF_F, 0.f);
    if (tid < parts) ml = __ldcg(stat + row_of(tid));
    float M = ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (tid % 32 == 0) sml[tid / 32].x = M;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < NT / 32; ++i) M = fmaxf(M, sml[i].x);
    const float w = ml.x == -CUDART_INF_F ? 0.f : pow2(ml.x - M);
    weight[tid] = w;
    float L = w * ml.y;
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (tid % 32 == 0) sml[tid / 32].y = L;
    __syncthreads();
    float o = 0.f;
    for (uint32_t i0 = 0; i0 < parts; i0 += G * BATCH) {
        if (i0) request(i0);
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k)
            if (i0 + G * k + grp < parts) o = fmaf(weight[i0 + G * k + grp], v[k], o);
    }
    so[grp][d] = o;
    __syncthreads();
    if (grp || d >= dh) return;
    L = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < NT / 32; ++i) L += sml[i].y;
    o = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < G; ++i) o += so[i][d];
    *to = L == 0.f ? 0.f : o / L;
}

// How many clusters of 1, 2, 4, 8, 16 CTAs run at a time on the current device; nullptr (and the reason recorded) where that cannot be found out.
struct Fits { int clusters[5]; };
template <typename T, int DHP, bool PAIR>
const Fits* prepare() {
    using F = Few<T, DHP, PAIR>;
    static PerDevice<Fits> device;
    int dev = -1;
    const Fits* fits = cudaGetDevice(&dev) != cudaSuccess ? nullptr : device.get(dev, [](Fits& f) {
        auto* unit = attn_few_kernel<T, DHP, PAIR, false>;
        auto* list = attn_few_kernel<T, DHP, PAIR, true>;
        if (cudaFuncSetAttribute(unit, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::Smem) != cudaSuccess ||
            cudaFuncSetAttribute(list, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::Smem) != cudaSuccess ||
            cudaFuncSetAttribute(unit, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
        for (int i = 0; i < 5; ++i) {
            cudaLaunchConfig_t c = {};
            c.gridDim = dim3(1u << i); c.blockDim = dim3(32 * kWarps); c.dynamicSmemBytes = F::Smem;
            cudaLaunchAttribute at;
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = 1u << i; at.val.clusterDim.y = at.val.clusterDim.z = 1;
            c.attrs = &at; c.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&f.clusters[i], unit, &c) != cudaSuccess) { cudaGetLastError(); f.clusters[i] = 0; }
        }
        return true;
    });
    if (!fits) fail("attention: kernel attributes: %s", cudaGetErrorString(cudaGetLastError()));
    return fits;
}

template <typename T, int DHP, bool PAIR>
bool go(const AttnCall& a, float* scratch, cudaStream_t st) {
    using F = Few<T, DHP, PAIR>;
    const Fits* fits = prepare<T, DHP, PAIR>();
    if (!fits) return false;
    const unsigned most = std::min(kFewCtas, (unsigned)device_sm_count() * F::PerSm);
    // the keys that a sequence can have in reach, as far as the host knows
    const unsigned long long keys = a.c.table ? a.c.cap : a.c.total, seen = (unsigned long long)a.mask.window + a.mask.sinks + a.max_q;
    const unsigned long long each = ((a.mask.window && seen < keys ? seen : keys) + F::Tile - 1) / F::Tile, units = (unsigned long long)a.c.B * a.c.KVH, tiles = units * each;
    int cs = 4;
    while (cs && ((units << cs) > most || fits->clusters[cs] < (int)units || (1ull << cs) >= 2 * each)) --cs;
    // of several sequences some may be short, which evens out over a list and not over clusters
    const unsigned long long listed = a.c.B == 1 ? (tiles + most - 1) / most : 1;
    if ((units << cs) <= most && (each + (1u << cs) - 1) / (1u << cs) <= listed + kClusterTiles) {
        if (!launch_units(attn_few_kernel<T, DHP, PAIR, false>, (unsigned)units, 1u << cs, 32 * kWarps, F::Smem, st, a, (float*)nullptr, (float2*)nullptr, (Part*)nullptr, 1u << cs)) return false;
        note_launch();
        return check_launch("attn_few");
    }
    const unsigned grid = tiles < most ? (unsigned)std::max(tiles, 1ull) : most;
    Part* meta = reinterpret_cast<Part*>(scratch);
    float2* stat = reinterpret_cast<float2*>(meta + kFewCtas);
    float* part = reinterpret_cast<float*>(stat + 2 * kFewCtas * F::Rows);
    launch_overlapped(attn_few_kernel<T, DHP, PAIR, true>, dim3(grid), dim3(32 * kWarps), F::Smem, st, a, part, stat, meta, 1u);
    note_launch();
    if (!check_launch("attn_few")) return false;
    if (grid == 1) return true;
    const unsigned rows = a.max_q >= F::Rows ? F::Rows : std::min(F::Rows, a.max_q * a.rep);
    launch_overlapped(attn_few_merge_kernel, dim3(grid - 1, rows), dim3(128, kMergeGroups), 0, st, a, part, stat, meta, F::Rows);
    note_launch();
    return check_launch("attn_few_merge");
}

template <int DHP>
bool go_tiled(const AttnCall& a, const ChunkPlan& pl, cudaStream_t st) {
    const Fits* fits = prepare<float, DHP, false>();
    if (!fits) return false;
    const unsigned long long units = (unsigned long long)a.c.KVH * pl.slots;
    if (units * pl.splits > 0x7fffffffull) return fail("attention: %llu tiles of query rows", units);
    if (!launch_units(attn_few_kernel<float, DHP, false, false>, (unsigned)units, pl.splits, 32 * kWarps, Few<float, DHP, false>::Smem, st, a, (float*)nullptr, (float2*)nullptr,
                      (Part*)nullptr, pl.splits)) return false;
    note_launch();
    return check_launch("attn_tiled");
}

}  // namespace

bool launch_attn_tiled(AttnCall a, const ChunkPlan& pl, cudaStream_t st) {
    a.tiled = true;
    return a.c.dh <= 64 ? go_tiled<64>(a, pl, st) : go_tiled<128>(a, pl, st);
}

size_t attn_few_scratch(uint32_t rows, uint32_t dh) {
    const size_t slots = 2 * (size_t)kFewCtas * (rows <= 8 ? 8 : kFewRows);
    return kFewCtas * sizeof(Part) + slots * sizeof(float2) + slots * dh * sizeof(float);
}

// a.few says how many rows a sequence has at most: up to 8 the kernel with both parts in one product
bool launch_attn_few(const AttnCall& a, bool half, float* scratch, cudaStream_t st) {
    const bool pair = a.few <= 8;
    if (a.c.dh <= 64) {
        if (half) return pair ? go<__half, 64, true>(a, scratch, st) : go<__half, 64, false>(a, scratch, st);
        return pair ? go<float, 64, true>(a, scratch, st) : go<float, 64, false>(a, scratch, st);
    }
    if (half) return pair ? go<__half, 128, true>(a, scratch, st) : go<__half, 128, false>(a, scratch, st);
    return pair ? go<float, 128, true>(a, scratch, st) : go<float, 128, false>(a, scratch, st);
}

}  // namespace tmc
