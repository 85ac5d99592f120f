// kv_pages.cuh — what the kernels over a batch of sequences share: where a sequence's new tokens, positions and cache rows are,
// and which keys a position sees. A contiguous cache [KVH][ctx][dh] is the same thing with one sequence and one page of ctx rows.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#include <cuda_runtime.h>
#define TM_HD __host__ __device__ __forceinline__
#else
#define TM_HD inline                       // the index arithmetic is plain C++: a host test runs it against bad arrays
#endif

struct tm_cuda_kv_pages;

namespace tmc {

// A kernel argument. Every index that comes from device memory (table, q_begin, kv_len) is checked by the kernel that follows it:
// what is out of range is not read, makes the results that depend on it NaN and sets the status word to kStatusBatch.
struct KvBatch {
    const void* k;
    const void* v;
    const int* table;           // nullptr: one sequence on one page, `total` positions, all T tokens new
    const int* q_begin;
    const int* kv_len;
    uint32_t B, KVH, dh, page, npages, table_ld, T;
    uint32_t cap;               // positions that a sequence's row of the table can name
    uint32_t total;             // without a table: positions in the cache
    int page_shift;             // log2(page), or -1
};
constexpr int kStatusBatch = 64;                // waits that run out have 1 and 2

struct KvSeq {
    uint32_t q0, n;             // its rows of q and out; none where q_begin does not give a range of them
    int first;                  // position of the first new token (negative: more new tokens than positions)
    uint32_t len;               // positions in the cache, the new tokens among them
    bool lost, bad;             // no range of rows; no valid length (the rows are there, their results are NaN)
};
TM_HD KvSeq kv_seq(const KvBatch& c, uint32_t b) {
    KvSeq s;
    if (!c.table) {
        s.q0 = 0; s.n = c.T; s.len = c.total; s.lost = s.bad = false;
    } else {
        const int a = c.q_begin[b], e = c.q_begin[b + 1], len = c.kv_len[b];
        s.lost = a < 0 || e < a || (uint32_t)e > c.T;
        s.q0 = s.lost ? 0u : (uint32_t)a;
        s.n = s.lost ? 0u : (uint32_t)(e - a);
        s.bad = len < 0 || (uint32_t)len > c.cap;
        s.len = s.bad ? 0u : (uint32_t)len;
    }
    s.first = (int)s.len - (int)s.n;
    return s;
}
// Element offset of row `pos` (< cap) of K/V head 0; row r of head h of the same page lies h * page * dh elements further. false: no such page.
TM_HD bool kv_row(const KvBatch& c, uint32_t b, uint32_t pos, size_t* at) {
    if (!c.table) { *at = (size_t)pos * c.dh; return true; }
    uint32_t slot, row;
    if (c.page_shift >= 0) { slot = pos >> c.page_shift; row = pos & (c.page - 1u); }
    else { slot = pos / c.page; row = pos - slot * c.page; }
    const uint32_t pg = (uint32_t)c.table[(size_t)b * c.table_ld + slot];
    const bool ok = pg < c.npages;
    *at = ((size_t)(ok ? pg : 0u) * c.KVH * c.page + row) * c.dh;
    return ok;
}

#ifdef __CUDACC__
// The word is the library's one: what a wait that ran out has left there, and nobody has read yet, stays.
__device__ __forceinline__ void note_bad_batch(int* status) {
    if (status && *(volatile int*)status == 0) *(volatile int*)status = kStatusBatch;
}
// The sequence that token t belongs to, found by a whole warp: a lane reads all there is to know of a sequence, so that one trip to memory
// says which it is and what it is. false: none.
__device__ __forceinline__ bool kv_find_seq(const KvBatch& c, uint32_t t, uint32_t* b, KvSeq* s) {
    if (!c.table) { *b = 0; *s = kv_seq(c, 0); return true; }
    const uint32_t lane = threadIdx.x & 31u;
    for (uint32_t i0 = 0; i0 < c.B; i0 += 32) {
        KvSeq x{};
        if (i0 + lane < c.B) x = kv_seq(c, i0 + lane);
        const uint32_t here = __ballot_sync(0xffffffffu, t - x.q0 < x.n);
        if (!here) continue;
        const int at = __ffs((int)here) - 1;
        *b = i0 + (uint32_t)at;
        s->q0 = __shfl_sync(0xffffffffu, x.q0, at); s->n = __shfl_sync(0xffffffffu, x.n, at); s->len = __shfl_sync(0xffffffffu, x.len, at);
        s->first = (int)s->len - (int)s->n; s->lost = false; s->bad = __shfl_sync(0xffffffffu, (int)x.bad, at) != 0;
        return true;
    }
    return false;
}
// A range of rows that is none, noted by whoever walks all sequences anyway
__device__ __forceinline__ void kv_note_lost(const KvBatch& c, int* status) {
    if (!c.table) return;
    for (uint32_t i = threadIdx.x; i < c.B; i += blockDim.x)
        if (kv_seq(c, i).lost) note_bad_batch(status);
}
#endif

// Key j is seen from position p if it is not behind it and, with a window, less than `window` back or one of the first `sinks`.
// window 0: no window. Neither is more than 2^31 - 1 (kv_mask).
struct KvMask { uint32_t window, sinks; };
inline KvMask kv_mask(unsigned window, unsigned sinks) { return KvMask{window > 0x7fffffffu ? 0u : window, sinks > 0x7fffffffu ? 0x7fffffffu : sinks}; }
TM_HD bool kv_sees(const KvMask& m, int p, int j) {
    return (j <= p) & (!m.window | ((int)m.window > p - j) | (j < (int)m.sinks));     // without branches
}
// The keys that positions [p0, p1] see between them: [0, a) and [b, e), a <= b.
struct KvSpan { uint32_t a, b, e; };
TM_HD KvSpan kv_span(const KvMask& m, int p0, int p1) {
    KvSpan s;
    s.e = p1 < 0 ? 0u : (uint32_t)p1 + 1u;
    s.b = !m.window || p0 < (int)m.window ? 0u : (uint32_t)p0 - m.window + 1u;
    s.a = !m.window ? 0u : m.sinks < s.b ? m.sinks : s.b;
    return s;
}

constexpr float kLog2e = 1.4426950408889634f;

// host side (attn_pages.cu): the checks that every entry over such a batch makes; that the library is up on the current device
bool kv_batch_from(KvBatch* c, const tm_cuda_kv_pages* kv, unsigned T, unsigned H, const char* who);
bool on_library_device(const char* who);
inline bool overlap(const void* a, size_t na, const void* b, size_t nb) { return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; }
inline size_t kv_bytes(const KvBatch& c, bool half) { return (size_t)c.npages * c.KVH * c.page * c.dh * (half ? 2 : 4); }
// Does memory that a call writes overlap the cache or the arrays that describe it?
inline bool overlaps_cache(const KvBatch& c, bool half, const void* a, size_t n) {
    if (overlap(a, n, c.k, kv_bytes(c, half)) || overlap(a, n, c.v, kv_bytes(c, half))) return true;
    return c.table && (overlap(a, n, c.table, (size_t)c.B * c.table_ld * 4) || overlap(a, n, c.q_begin, ((size_t)c.B + 1) * 4) || overlap(a, n, c.kv_len, (size_t)c.B * 4));
}

}  // namespace tmc
