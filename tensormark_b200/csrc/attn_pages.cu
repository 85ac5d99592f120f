// attn_pages.cu — attention of the new tokens of a batch of sequences over a paged K/V cache, and of a chunk of tokens over a
// contiguous one, with an optional sliding window and first tokens that stay visible: the entries, their checks, and which kernel serves what.
#include "cuda_shim.h"
#include "attn_pages.h"
#include "common.cuh"
#include "state.h"

#include <cmath>

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
    if (((uintptr_t)kv->table | (uintptr_t)kv->q_begin | (uintptr_t)kv->kv_len) % 4) return fail("%s: the table and the lengths lie on 4-byte boundaries", who);
    if ((uintptr_t)kv->k % 16 || (uintptr_t)kv->v % 16) return fail("%s: the pages lie on 16-byte boundaries", who);
    if ((unsigned long long)kv->table_ld * kv->page > 0x7fffff00ull || (unsigned long long)T * H > 0x7fffffffull || kv->B > 0x7ffffffu) return fail("%s: 2^31 positions or query rows", who);
    *c = KvBatch{kv->k, kv->v, kv->table, kv->q_begin, kv->kv_len, kv->B, kv->KVH, kv->dh, kv->page, kv->npages, kv->table_ld, T, kv->table_ld * kv->page, 0u, -1};
    if ((kv->page & (kv->page - 1u)) == 0)
        for (c->page_shift = 0; 1u << c->page_shift < kv->page;) ++c->page_shift;
    return true;
}

namespace {

// Which kernels serve a call: sequences with up to `few` rows per K/V head attn_few.cu, those with more (`others`: there may be some) attn_chunk.cu, or, over
// fp32 caches, attn_few.cu again with 16 rows at a time. One launch serves all up to 16 rows. Beside longer ones `few` is 8 for groups of
// up to 8 heads, whose single tokens then have the kernel that takes both parts in one product: 512 tokens + 16 x 1 of 32 / 8 heads of 128 in
// fp16 112 us, with 16 for `few` 118 (+ 48 x 1: 167 and 178; fp32 815 and 852); + 16 x 4 drafted tokens, which 8 sends to 256-row tiles,
// 157 and 126 (fp32 851 and 862). Groups of more than 16 heads have no other kernel than the tiles.
struct Split { uint32_t few; bool others; };
Split split(unsigned B, unsigned long long rows, unsigned rep) {
    if (rows <= kFewRows) return Split{rows <= 8 ? 8u : kFewRows, false};
    return Split{B == 1 || rep > kFewRows ? 0u : rep <= 8 ? 8u : kFewRows, true};
}

// What a call writes, against what it reads and against each other
bool apart(const KvBatch& c, bool half, const float* q, const float* scratch, size_t scratch_bytes, const float* out, size_t rows_bytes, const char* who) {
    if (overlap(q, rows_bytes, out, rows_bytes)) return fail("%s: out overlaps q", who);
    if (overlap(scratch, scratch_bytes, out, rows_bytes) || overlap(scratch, scratch_bytes, q, rows_bytes)) return fail("%s: scratch overlaps q or out", who);
    if (overlaps_cache(c, half, out, rows_bytes) || overlaps_cache(c, half, scratch, scratch_bytes)) return fail("%s: out or scratch overlaps the cache", who);
    return true;
}

bool launch(AttnCall a, bool half, float* scratch, cudaStream_t st) {
    const Split sp = split(a.c.B, (unsigned long long)a.max_q * a.rep, a.rep);
    a.few = sp.few; a.others = sp.others; a.status = device_status_word();
    if (sp.few && !launch_attn_few(a, half, scratch, st)) return false;
    if (!sp.others) return true;
    const ChunkPlan pl = plan_attn_chunk(a.c.T, a.c.B, a.c.KVH, a.rep, a.few, half ? kChunkRows : kFewRows);
    return half ? launch_attn_chunk(a, pl, st) : launch_attn_tiled(a, pl, st);
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" {

// What the call needs, or one with fewer tokens, sequences or new tokens of one: a prompt's call may need none, the decode step after it does.
size_t tm_cuda_attn_paged_scratch(unsigned T, unsigned, unsigned max_q, unsigned H, unsigned KVH, unsigned dh) {
    if (!KVH || !H || H % KVH || !dh || !T) return 16;
    const unsigned long long rows = (unsigned long long)(max_q && max_q < T ? max_q : T) * (H / KVH);
    return attn_few_scratch(rows <= 8 ? 8 : kFewRows, dh);
}
size_t tm_cuda_attn_window_scratch(unsigned T, unsigned H, unsigned KVH, unsigned dh) { return tm_cuda_attn_paged_scratch(T, 1, T, H, KVH, dh); }

bool tm_cuda_attn_paged_dev(const tm_cuda_kv_pages* kv, const float* q, float* scratch, size_t scratch_bytes, float* out, unsigned T, unsigned max_q,
                            unsigned H, unsigned window, unsigned sinks, float scale, void* stream) {
    KvBatch c;
    if (!kv_batch_from(&c, kv, T, H, "attn_paged")) return false;
    if (!T) return true;
    if (!q || !out || !scratch) return fail("attn_paged: null pointer");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)scratch % 16) return fail("attn_paged: q, out and scratch lie on 16-byte boundaries");
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail("attn_paged: the scale is not a positive number");
    const size_t need = tm_cuda_attn_paged_scratch(T, c.B, max_q, H, c.KVH, c.dh);
    if (scratch_bytes < need) return fail("attn_paged: %zu bytes of scratch, %zu are needed", scratch_bytes, need);
    if (!apart(c, kv->kv_half != 0, q, scratch, need, out, (size_t)T * H * c.dh * 4, "attn_paged")) return false;
    if (!on_library_device("attn_paged")) return false;
    return launch(AttnCall{c, kv_mask(window, sinks), q, out, H, H / c.KVH, max_q && max_q < T ? max_q : T, 0, false, scale, nullptr, false}, kv->kv_half != 0, scratch, (cudaStream_t)stream);
}

bool tm_cuda_attn_window_dev(const float* q, const void* kc, const void* vc, float* scratch, size_t scratch_bytes, float* out, unsigned T,
                             unsigned pos0, unsigned H, unsigned KVH, unsigned dh, unsigned ctx, unsigned window, unsigned sinks, float scale,
                             int kv_half, void* stream) {
    if (!KVH || !H || H % KVH || H / KVH > 128) return fail("attn_window: %u query heads for %u K/V heads (a multiple, at most 128 each)", H, KVH);
    if (!dh || dh % 8 || dh > 128) return fail("attn_window: head dimension %u (multiples of 8 up to 128)", dh);
    if (!ctx || ctx > 0x7fffff00u || pos0 > ctx || T > ctx - pos0) return fail("attn_window: positions %u to %llu of a cache of %u rows", pos0, (unsigned long long)pos0 + T, ctx);
    if (!T) return true;
    if (!q || !kc || !vc || !scratch || !out) return fail("attn_window: null pointer");
    if ((unsigned long long)T * H > 0x7fffffffull) return fail("attn_window: 2^31 query rows");
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)scratch | (uintptr_t)out) % 16) return fail("attn_window: q, the caches, scratch and out lie on 16-byte boundaries");
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail("attn_window: the scale is not a positive number");
    const size_t need = tm_cuda_attn_window_scratch(T, H, KVH, dh);
    if (scratch_bytes < need) return fail("attn_window: %zu bytes of scratch, %zu are needed", scratch_bytes, need);
    const KvBatch c{kc, vc, nullptr, nullptr, nullptr, 1, KVH, dh, ctx, 1, 1, T, ctx, pos0 + T, -1};
    if (!apart(c, kv_half != 0, q, scratch, need, out, (size_t)T * H * dh * 4, "attn_window")) return false;
    if (!on_library_device("attn_window")) return false;
    return launch(AttnCall{c, kv_mask(window, sinks), q, out, H, H / KVH, T, 0, false, scale, nullptr, false}, kv_half != 0, scratch, (cudaStream_t)stream);
}

}  // extern "C"
