// attn_rows.cuh — what the two kernels behind the attention over pages share: the tiles of keys that a set of rows sees, and a row
// computed key by key.
#pragma once

#include "attn_pages.h"

#include <math_constants.h>

namespace tmc {

// Partial results of a range of keys, for the merge of several: scores are kept in powers of two, and weights are 2^(s - m + kUp). Against fp16
// caches, whose weights are split into fp16 halves, the lift keeps the high half a normal number down to 2^-28 of the largest weight and
// the low one down to 2^-17; from there on a weight is off by up to 2^-25, 2^-39 of the largest. tf32 has fp32's exponents and needs none.
template <typename T> constexpr float kUp = sizeof(T) == 2 ? 14.f : 0.f;
// Sums of an fp32 cache's values beyond kFar are computed again by row_again, whose weights are 2^-kDown of the others', so that what 2^24
// keys add up to is finite if the values are. Parts that stay below do not make the merge of 600 infinite.
constexpr float kFar = 1.2676506e30f /* 2^100 */, kDown = 24.f;
template <typename T> __device__ __forceinline__ bool in_reach(float x) { return fabsf(x) < (sizeof(T) == 2 ? CUDART_INF_F : kFar); }

__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {   // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Where the window of a row at p begins
__device__ __forceinline__ int window_from(const KvMask& m, int p) { return m.window && p >= (int)m.window ? p - (int)m.window + 1 : 0; }

// The parts of a row that the CTAs of a cluster hold lie at the same place in the shared memory of each.
__device__ __forceinline__ uint32_t map_cta(uint32_t at, uint32_t rank) {
    uint32_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(v) : "r"(at), "r"(rank));
    return v;
}
__device__ __forceinline__ float2 ld_cta2(uint32_t at) {
    float2 f;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(at) : "memory");
    return f;
}
__device__ __forceinline__ float ld_cta(uint32_t at) {
    float f;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at) : "memory");
    return f;
}
__device__ __forceinline__ float4 ld_cta4(uint32_t at) {
    float4 f;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at) : "memory");
    return f;
}
__device__ __forceinline__ void cluster_sync() {            // by whole warps
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The keys [0, a) and [b, e) that a set of rows sees, one behind the other, in tiles of N places: a window's keys follow the first ones in
// the same tile. At least one tile, so that rows that see nothing are visited.
template <uint32_t N> struct KeyTiles {
    uint32_t tiles, count, a, skip;                         // places; the first that lies `skip` keys further on
    uint32_t end;                                           // no row is at a position from here on
    __device__ __forceinline__ void set(const KvSpan& sp, bool none) {
        a = sp.a; skip = sp.b - sp.a; end = none ? 0u : sp.e;
        count = none ? 0u : sp.e - min(sp.e, skip);
        tiles = max(1u, (count + N - 1) / N);
    }
    __device__ __forceinline__ uint32_t key(uint32_t place) const { return place + (place < a ? 0u : skip); }
    // Does a row at p_least or behind it, in a window that begins at `from` or before it, see all of the places [u, u + n)?
    __device__ __forceinline__ bool seen(uint32_t u, uint32_t n, int p_least, uint32_t from) const {
        return (int)key(u + n - 1) <= p_least && (u + n <= a || key(max(u, a)) >= from);
    }
};

// One row over tiles [t0, t1) by one warp, key by key in fp32: what a kernel whose products take masked values along computes again
// where a sum was not finite or beyond kFar. stat: the row stays unnormalised, with its maximum and sum there; nullptr: it is finished.
template <typename T, uint32_t N>
__device__ __noinline__ void row_again(const AttnCall& a, uint32_t b, uint32_t h, int p, KeyTiles<N> tiles, uint32_t t0, uint32_t t1, const float* q, float* to, float2* stat) {
    constexpr float down = sizeof(T) == 2 ? 0.f : kDown, lift = sizeof(T) == 2 ? 1.f : 1.f / (1u << (int)kDown);
    const uint32_t lane = threadIdx.x & 31u, dh = a.c.dh;
    const T* kb = (const T*)a.c.k + (size_t)h * a.c.page * dh;
    const T* vb = (const T*)a.c.v + (size_t)h * a.c.page * dh;
    float qr[4], acc[4] = {}, m = -CUDART_INF_F, l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) qr[k] = lane + 32u * k < dh ? q[lane + 32u * k] * (a.scale * kLog2e) : 0.f;
    for (uint32_t t = t0; t < t1; ++t) {
        for (uint32_t u = t * N; u < min((t + 1) * N, tiles.count); ++u) {
            const uint32_t j = tiles.key(u);
            size_t at;
            if (!kv_sees(a.mask, p, (int)j) || !kv_row(a.c, b, j, &at)) continue;
            float x = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (lane + 32u * k < dh) x = fmaf(qr[k], (float)kb[at + lane + 32u * k], x);
#pragma unroll
            for (int s = 16; s; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
            const float mn = fmaxf(m, x), corr = m == -CUDART_INF_F ? 0.f : exp2f(m - mn), w = x == -CUDART_INF_F ? 0.f : lift * exp2f(x - mn + kUp<T>);
            l = fmaf(l, corr, w);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (lane + 32u * k < dh) acc[k] = fmaf(acc[k], corr, w * (float)vb[at + lane + 32u * k]);
            m = mn;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (lane + 32u * k < dh) to[lane + 32u * k] = stat ? acc[k] : l == 0.f ? 0.f : acc[k] / l;
    if (stat && lane == 0) *stat = make_float2(m + down, l);
}

}  // namespace tmc
