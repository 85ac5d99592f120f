// kv_append.cu — the new tokens of a batch of sequences on their way into a paged K/V cache: rope(q), rope(k) -> pages, v -> pages.
//
// (a, b) = (x[j], x[j + dh/2]) of a head and (c, s) of its position: a c - b s and a s + b c, with the contractions written out
// as in the layer stack's append (llama_stack.cu), so that a row does not depend on which of the two wrote it.
//
// Bound: HBM, every value read once and written once: 2000 tokens of 32 / 4 heads of 64 to an fp32 cache, 31 MB, 6.2 us (5.0 TB/s, in part
// from L2). A decode batch is bound by its trips to memory, q_begin and the lengths, then the page: 48 tokens 2.4 us in a graph. A thread
// takes four pairs of a head (two 16-byte reads, two writes) or four values of v, and asks for them before its warp looks for the sequence.
// A token whose position is not known, or has no angles, is not stored and leaves NaN in its row of q: the attention that follows would
// find the length and the pages in order in the second case, and answer from what the buffers held before.
#include "cuda_shim.h"
#include "common.cuh"
#include "kv_pages.cuh"
#include "pdl.cuh"
#include "state.h"

#include <cuda_fp16.h>
#include <math_constants.h>

namespace tmc {
namespace {

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__half* p, float4 v) {
    const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ float turn_lo(float x, float y, float c, float s) { return fmaf(x, c, -__fmul_rn(y, s)); }
__device__ __forceinline__ float turn_hi(float x, float y, float c, float s) { return fmaf(x, s, __fmul_rn(y, c)); }

template <typename T>
__global__ void __launch_bounds__(512) kv_append_kernel(KvBatch c, const float* qkv, float* q, uint32_t H, const float2* rope, uint32_t rope_rows,
                                                        int* status) {
    const uint32_t t = blockIdx.x, dh = c.dh, KVH = c.KVH, half = dh / 2, per = dh / 8, turned = (H + KVH) * per;
    const uint32_t e = blockIdx.y * blockDim.x + threadIdx.x, i = 4 * (e - turned), h = e / per, j = 4 * (e % per);
    const float* row = qkv + (size_t)t * (H + 2 * KVH) * dh;
    const bool turns = e < turned, value = !turns && i < KVH * dh;
    pdl_enter();
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;          // on their way while the sequence is looked for
    if (turns) { u = *reinterpret_cast<const float4*>(row + (size_t)h * dh + j); w = *reinterpret_cast<const float4*>(row + (size_t)h * dh + j + half); }
    else if (value) u = *reinterpret_cast<const float4*>(row + (size_t)(H + KVH) * dh + i);
    if (t == 0 && blockIdx.y == 0) kv_note_lost(c, status);
    uint32_t b;
    KvSeq s;
    if (!kv_find_seq(c, t, &b, &s)) return;                     // behind the last sequence
    const int pos = s.first + (int)(t - s.q0);
    if (s.bad || (rope && pos >= (int)rope_rows)) {
        note_bad_batch(status);
        if (turns && h < H) {
            float* o = q + ((size_t)t * H + h) * dh + j;
            const float4 none = make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F);
            store4(o, none); store4(o + half, none);
        }
        return;
    }
    if (pos < 0) return;
    size_t at;
    const bool page = kv_row(c, b, (uint32_t)pos, &at);
    if (!page) note_bad_batch(status);
    if (turns) {
        float4 lo = u, hi = w;
        if (rope) {
            const float4* cs = reinterpret_cast<const float4*>(rope + (size_t)pos * half + j);
            const float4 p = cs[0], r = cs[1];
            lo = make_float4(turn_lo(u.x, w.x, p.x, p.y), turn_lo(u.y, w.y, p.z, p.w), turn_lo(u.z, w.z, r.x, r.y), turn_lo(u.w, w.w, r.z, r.w));
            hi = make_float4(turn_hi(u.x, w.x, p.x, p.y), turn_hi(u.y, w.y, p.z, p.w), turn_hi(u.z, w.z, r.x, r.y), turn_hi(u.w, w.w, r.z, r.w));
        }
        if (h < H) {
            float* o = q + ((size_t)t * H + h) * dh + j;
            store4(o, lo); store4(o + half, hi);
        } else if (page) {
            T* o = (T*)const_cast<void*>(c.k) + at + (size_t)(h - H) * c.page * dh + j;
            store4(o, lo); store4(o + half, hi);
        }
    } else if (value && page) {
        store4((T*)const_cast<void*>(c.v) + at + (size_t)(i / dh) * c.page * dh + i % dh, u);
    }
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" bool tm_cuda_kv_append_paged_dev(const tm_cuda_kv_pages* kv, const float* qkv, float* q, unsigned T, unsigned H, const float* rope,
                                            unsigned rope_rows, void* stream) {
    KvBatch c;
    if (!kv_batch_from(&c, kv, T, H, "kv_append_paged")) return false;
    if (!T) return true;
    if (!qkv || !q) return fail("kv_append_paged: null pointer");
    if ((uintptr_t)qkv % 16 || (uintptr_t)q % 16 || (uintptr_t)rope % 16) return fail("kv_append_paged: qkv, q and rope lie on 16-byte boundaries");
    if (rope && !rope_rows) return fail("kv_append_paged: an empty rope table");
    if (rope_rows > 0x7fffffffu) rope_rows = 0x7fffffffu;
    const bool half = kv->kv_half != 0;
    const size_t q_bytes = (size_t)T * H * c.dh * 4, qkv_bytes = (size_t)T * (H + 2 * (size_t)c.KVH) * c.dh * 4;
    if (overlap(q, q_bytes, qkv, qkv_bytes)) return fail("kv_append_paged: q overlaps qkv");
    if (overlaps_cache(c, half, q, q_bytes) || overlaps_cache(c, half, qkv, qkv_bytes)) return fail("kv_append_paged: q or qkv overlaps the cache");
    if (overlap(c.k, kv_bytes(c, half), c.v, kv_bytes(c, half))) return fail("kv_append_paged: the pages of keys overlap those of values");
    if (!on_library_device("kv_append_paged")) return false;
    // A token's items in as few blocks as hold them, and those no larger than they need be: a token's sequence is looked for once per warp.
    const unsigned items = (H + c.KVH) * (c.dh / 8) + c.KVH * c.dh / 4, blocks = (items + 511) / 512, threads = ((items + blocks - 1) / blocks + 31) / 32 * 32;
    const dim3 grid(T, blocks);
    launch_overlapped(half ? kv_append_kernel<__half> : kv_append_kernel<float>, grid, dim3(threads), 0, (cudaStream_t)stream, c, qkv, q, H, (const float2*)rope,
                      rope_rows, device_status_word());
    note_launch();
    return check_launch("kv_append_paged");
}
