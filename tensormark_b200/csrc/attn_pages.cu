// attn_pages.cu — attention of the new tokens of a batch of sequences over a paged K/V cache, and of a chunk of tokens over a
// contiguous one, with an optional sliding window and first tokens that stay visible. The simple form: a warp per query row.
#include "cuda_shim.h"
#include "attn_pages.h"
#include "common.cuh"
#include "state.h"

#include <algorithm>
#include <cmath>
#include <cuda_fp16.h>
#include <math_constants.h>

namespace tmc {

bool on_library_device(const char* who) {
    if (!ensure_init(-1)) return false;
    int dev = -1;
    if (cudaGetDevice(&dev) == cudaSuccess && dev == state().device) return true;
    cudaGetLastError();
    return fail("%s: the library's device %d is not the current one", who, state().device);
}

bool kv_batch_from(KvBatch* c, const tm_cuda_kv_pages* kv, unsigned T, unsigned H, const char* who) {
    if (!kv) return fail("%s: null pointer", who);
    if (!kv->k || !kv->v || !kv->table || !kv->q_begin || !kv->kv_len) return fail("%s: null pointer in the cache's description", who);
    if (!kv->B || !kv->KVH || !kv->page || !kv->npages || !kv->table_ld) return fail("%s: a zero in the cache's description", who);
    if (!H || H % kv->KVH || H / kv->KVH > 128) return fail("%s: %u query heads for %u K/V heads (a multiple, at most 128 each)", who, H, kv->KVH);
    if (!kv->dh || kv->dh % 8 || kv->dh > 128) return fail("%s: head dimension %u (multiples of 8 up to 128)", who, kv->dh);
    if ((uintptr_t)kv->k % 16 || (uintptr_t)kv->v % 16) return fail("%s: the pages lie on 16-byte boundaries", who);
    if ((unsigned long long)kv->table_ld * kv->page > 0x7fffff00ull || (unsigned long long)T * H > 0x7fffffffull || kv->B > 0x7ffffffu) return fail("%s: 2^31 positions or query rows", who);
    *c = KvBatch{kv->k, kv->v, kv->table, kv->q_begin, kv->kv_len, kv->B, kv->KVH, kv->dh, kv->page, kv->npages, kv->table_ld, T, kv->table_ld * kv->page, 0u, -1};
    if ((kv->page & (kv->page - 1u)) == 0)
        for (c->page_shift = 0; 1u << c->page_shift < kv->page;) ++c->page_shift;
    return true;
}

namespace {

template <typename T>
__global__ void __launch_bounds__(128) attn_rows_kernel(const __grid_constant__ AttnCall a) {
    const KvBatch& c = a.c;
    const uint32_t lane = threadIdx.x & 31u, id = blockIdx.x * 4u + (threadIdx.x >> 5), t = id / a.H, head = id % a.H;
    if (t >= c.T) return;
    const uint32_t b = kv_find_seq(c, t);
    if (b >= c.B) return;
    const KvSeq s = kv_seq(c, b);
    if (s.lost || t < s.q0 || t - s.q0 >= s.n) { note_bad_batch(a.status); return; }
    if (s.n * a.rep <= a.few) return;
    const uint32_t dh = c.dh;
    const int p = s.first + (int)(t - s.q0);
    const KvSpan span = kv_span(a.mask, p, p);
    const T* kb = (const T*)c.k + (size_t)(head / a.rep) * c.page * dh;
    const T* vb = (const T*)c.v + (size_t)(head / a.rep) * c.page * dh;
    float qr[4], acc[4] = {}, m = -CUDART_INF_F, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) qr[i] = lane + 32u * i < dh ? a.q[((size_t)t * a.H + head) * dh + lane + 32u * i] * (a.scale * kLog2e) : 0.f;
    bool bad = s.bad || s.n > a.max_q;
    for (uint32_t j = span.a ? 0u : span.b; j < span.e; j = j + 1 == span.a ? span.b : j + 1) {
        size_t at;
        if (!kv_row(c, b, j, &at)) { bad = true; continue; }
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32u * i < dh) x = fmaf(qr[i], (float)kb[at + lane + 32u * i], x);
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        const float mn = fmaxf(m, x), corr = m == -CUDART_INF_F ? 0.f : exp2f(m - mn), w = x == -CUDART_INF_F ? 0.f : exp2f(x - mn + kUp);
        l = fmaf(l, corr, w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32u * i < dh) acc[i] = fmaf(acc[i], corr, w * (float)vb[at + lane + 32u * i]);
        m = mn;
    }
    if (bad) { note_bad_batch(a.status); l = CUDART_NAN_F; }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 32u * i < dh) a.out[((size_t)t * a.H + head) * dh + lane + 32u * i] = l == 0.f ? 0.f : acc[i] / l;
}

// Which kernels serve a call: sequences with up to `few` rows per K/V head attn_few.cu, those with more (`others`: there may be some) this one.
struct Split { uint32_t few; bool others; };
Split split(unsigned B, unsigned long long rows, unsigned rep) {
    if (rows <= kFewRows) return Split{rows <= 8 ? 8u : kFewRows, false};
    return Split{B == 1 || rep > kFewRows ? 0u : rep <= 8 ? 8u : kFewRows, true};
}

size_t few_bytes(Split sp, unsigned dh) { return sp.few ? attn_few_scratch(sp.few, dh) : 0; }

bool launch(AttnCall a, bool half, float* scratch, cudaStream_t st) {
    const Split sp = split(a.c.B, (unsigned long long)a.max_q * a.rep, a.rep);
    a.few = sp.few; a.others = sp.others; a.status = device_status_word();
    if (sp.few && !launch_attn_few(a, half, scratch, st)) return false;
    if (!sp.others) return true;
    if (half) return launch_attn_chunk(a, plan_attn_chunk(a.c.T, a.c.B, a.c.KVH, a.rep, a.few), scratch + few_bytes(sp, a.c.dh) / sizeof(float), st);
    const unsigned grid = (unsigned)(((size_t)a.c.T * a.H + 3) / 4);
    attn_rows_kernel<float><<<grid, 128, 0, st>>>(a);
    note_launch();
    return check_launch("attention");
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" {

size_t tm_cuda_attn_paged_scratch(unsigned T, unsigned B, unsigned max_q, unsigned H, unsigned KVH, unsigned dh) {
    if (!KVH || !H || H % KVH || !dh || !T) return 16;
    const unsigned rep = H / KVH;
    const Split sp = split(B, (unsigned long long)(max_q && max_q < T ? max_q : T) * rep, rep);
    const size_t chunk = sp.others ? attn_chunk_scratch(plan_attn_chunk(T, B, KVH, rep, sp.few), T, H, dh) : 0;
    return std::max<size_t>(16, few_bytes(sp, dh) + chunk);
}
size_t tm_cuda_attn_window_scratch(unsigned T, unsigned H, unsigned KVH, unsigned dh) { return tm_cuda_attn_paged_scratch(T, 1, T, H, KVH, dh); }

bool tm_cuda_attn_paged_dev(const tm_cuda_kv_pages* kv, const float* q, float* scratch, size_t scratch_bytes, float* out, unsigned T, unsigned max_q,
                            unsigned H, unsigned window, unsigned sinks, float scale, void* stream) {
    KvBatch c;
    if (!kv_batch_from(&c, kv, T, H, "attn_paged")) return false;
    if (!q || !out || !scratch) return fail("attn_paged: null pointer");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)scratch % 16) return fail("attn_paged: q, out and scratch lie on 16-byte boundaries");
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail("attn_paged: the scale is not a positive number");
    const size_t need = tm_cuda_attn_paged_scratch(T, c.B, max_q, H, c.KVH, c.dh);
    if (scratch_bytes < need) return fail("attn_paged: %zu bytes of scratch, %zu are needed", scratch_bytes, need);
    if (!on_library_device("attn_paged")) return false;
    if (!T) return true;
    return launch(AttnCall{c, kv_mask(window, sinks), q, out, H, H / c.KVH, max_q && max_q < T ? max_q : T, 0, false, scale, nullptr}, kv->kv_half != 0, scratch, (cudaStream_t)stream);
}

bool tm_cuda_attn_window_dev(const float* q, const void* kc, const void* vc, float* scratch, size_t scratch_bytes, float* out, unsigned T,
                             unsigned pos0, unsigned H, unsigned KVH, unsigned dh, unsigned ctx, unsigned window, unsigned sinks, float scale,
                             int kv_half, void* stream) {
    if (!q || !kc || !vc || !scratch || !out) return fail("attn_window: null pointer");
    if (!KVH || !H || H % KVH || H / KVH > 128) return fail("attn_window: %u query heads for %u K/V heads (a multiple, at most 128 each)", H, KVH);
    if (!dh || dh % 8 || dh > 128) return fail("attn_window: head dimension %u (multiples of 8 up to 128)", dh);
    if (!ctx || ctx > 0x7fffff00u || pos0 > ctx || T > ctx - pos0) return fail("attn_window: positions %u to %llu of a cache of %u rows", pos0, (unsigned long long)pos0 + T, ctx);
    if ((unsigned long long)T * H > 0x7fffffffull) return fail("attn_window: 2^31 query rows");
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)scratch | (uintptr_t)out) % 16) return fail("attn_window: q, the caches, scratch and out lie on 16-byte boundaries");
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail("attn_window: the scale is not a positive number");
    const size_t need = tm_cuda_attn_window_scratch(T, H, KVH, dh);
    if (scratch_bytes < need) return fail("attn_window: %zu bytes of scratch, %zu are needed", scratch_bytes, need);
    if (!on_library_device("attn_window")) return false;
    if (!T) return true;
    const KvBatch c{kc, vc, nullptr, nullptr, nullptr, 1, KVH, dh, ctx, 1, 1, T, ctx, pos0 + T, -1};
    return launch(AttnCall{c, kv_mask(window, sinks), q, out, H, H / KVH, T, 0, false, scale, nullptr}, kv_half != 0, scratch, (cudaStream_t)stream);
}

}  // extern "C"
