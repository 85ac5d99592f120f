"""CPU: refusals of the entries over a batch of sequences, and the index arithmetic of kv_pages.cuh against bad arrays."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tensormark_b200 import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20                      # an address that is on every boundary; no call gets as far as reading it


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        from tensormark_b200 import build
        build.build()
    return lib.load()


def pages(**kw):
    return lib.KvPages(**{**dict(k=A, v=A, table=A, q_begin=A, kv_len=A, B=3, KVH=2, dh=64, page=16, npages=9, table_ld=4, kv_half=1), **kw})


def refused(L, ok, *words):
    assert not ok
    for w in words:
        assert w in lib.last_error(), lib.last_error()


BAD_PAGES = [(dict(k=None), "null"), (dict(v=None), "null"), (dict(table=None), "null"), (dict(q_begin=None), "null"), (dict(kv_len=None), "null"),
             (dict(B=0), "zero"), (dict(KVH=0), "zero"), (dict(page=0), "zero"), (dict(npages=0), "zero"), (dict(table_ld=0), "zero"),
             (dict(KVH=3), "query heads"), (dict(KVH=16), "query heads"), (dict(dh=0), "head dimension"), (dict(dh=60), "head dimension"),
             (dict(dh=136), "head dimension"), (dict(k=A + 8), "16-byte"), (dict(v=A + 2), "16-byte"), (dict(page=1 << 20, table_ld=1 << 12), "2^31")]


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_cache_descriptions(L, kw, word):
    kv = pages(**kw)
    refused(L, L.tm_cuda_attn_paged_dev(C.byref(kv), A, A, 1 << 40, 2 * A, 5, 2, 8, 0, 0, 0.1, None), "attn_paged", word)
    refused(L, L.tm_cuda_kv_append_paged_dev(C.byref(kv), A, A, 5, 8, A, 100, None), "kv_append_paged", word)


def test_attention_arguments(L):
    kv, call = pages(), L.tm_cuda_attn_paged_dev
    need = L.tm_cuda_attn_paged_scratch(5, 3, 2, 8, 2, 64)
    for q, s, o, word in ((None, A, A, "null"), (A, None, A, "null"), (A, A, None, "null"), (A + 4, A, A, "16-byte"), (A, A + 8, A, "16-byte"), (A, A, A + 4, "16-byte")):
        refused(L, call(C.byref(kv), q, s, 1 << 40, o, 5, 2, 8, 0, 0, 0.1, None), "attn_paged", word)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(L, call(C.byref(kv), A, A, 1 << 40, A, 5, 2, 8, 0, 0, scale, None), "scale")
    refused(L, call(C.byref(kv), A, A, need - 1, A, 5, 2, 8, 0, 0, 0.1, None), "scratch")
    refused(L, call(C.byref(kv), A, A, 1 << 40, A, 1 << 31, 2, 8, 0, 0, 0.1, None), "2^31")
    refused(L, call(C.byref(kv), A, A, 1 << 40, A, 5, 2, 8, 0, 0, 0.1, None), "overlaps")
    refused(L, call(C.byref(kv), A + 5 * 8 * 64 * 4 - 16, A, 1 << 40, A, 5, 2, 8, 0, 0, 0.1, None), "overlaps")
    refused(L, call(None, A, A, 1 << 40, A, 5, 2, 8, 0, 0, 0.1, None), "null")
    refused(L, call(C.byref(kv), A, A, 1 << 40, A, 5, 2, 0, 0, 0, 0.1, None), "query heads")
    refused(L, call(C.byref(kv), A, A, 1 << 40, A, 5, 2, 2 * 129, 0, 0, 0.1, None), "query heads")


def test_window_arguments(L):
    need = L.tm_cuda_attn_window_scratch(5, 8, 2, 64)

    def call(q=A, k=A, v=A, s=A, n=1 << 40, o=A, T=5, pos0=0, H=8, KVH=2, dh=64, ctx=10, scale=0.1):
        return L.tm_cuda_attn_window_dev(q, k, v, s, n, o, T, pos0, H, KVH, dh, ctx, 0, 0, scale, 1, None)

    for kw, word in ((dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(s=None), "null"), (dict(o=None), "null"),
                     (dict(q=A + 4), "16-byte"), (dict(k=A + 8), "16-byte"), (dict(v=A + 2), "16-byte"), (dict(s=A + 4), "16-byte"), (dict(o=A + 12), "16-byte"),
                     (dict(T=11), "positions"), (dict(T=5, pos0=6), "positions"), (dict(pos0=11, T=0), "positions"), (dict(pos0=2 ** 32 - 1, T=2), "positions"),
                     (dict(ctx=0, T=0), "positions"), (dict(ctx=1 << 31), "positions"), (dict(H=7), "query heads"), (dict(H=0), "query heads"),
                     (dict(KVH=0), "query heads"), (dict(H=2 * 130), "query heads"), (dict(dh=0), "head dimension"), (dict(dh=4), "head dimension"),
                     (dict(dh=256), "head dimension"), (dict(n=need - 1), "scratch"), (dict(), "overlaps"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")):
        refused(L, call(**kw), "attn_window", word)


def test_append_arguments(L):
    kv, call = pages(), L.tm_cuda_kv_append_paged_dev
    refused(L, call(C.byref(kv), None, A, 5, 8, A, 9, None), "null")
    refused(L, call(C.byref(kv), A, None, 5, 8, A, 9, None), "null")
    for x, q, r in ((A + 4, A, A), (A, A + 8, A), (A, A, A + 8)):
        refused(L, call(C.byref(kv), x, q, 5, 8, r, 9, None), "16-byte")
    refused(L, call(C.byref(kv), A, A, 5, 8, A, 0, None), "rope")
    refused(L, call(C.byref(kv), A, A + 5 * 12 * 64 * 4 - 16, 5, 8, A, 9, None), "overlaps")


def test_rules_arguments(L):
    def call(x=A, ldx=100, o=A, ldo=100, B=2, V=100, **kw):
        r = lib.LogitRules(**{**dict(tokens=A, n_tokens=A, tokens_ld=5, repeat=A, bias_ids=A, bias=A, bias_ld=3, mask=A, mask_ld=4), **kw})
        return L.tm_cuda_logits_rules_dev(x, ldx, o, ldo, B, V, C.byref(r), None)

    for kw, word in ((dict(x=None), "null"), (dict(o=None), "null"), (dict(ldx=99), "strides"), (dict(ldo=99), "strides"), (dict(V=0), "rows"),
                     (dict(B=65536), "rows"), (dict(V=1 << 31, ldx=1 << 31, ldo=1 << 31), "rows"), (dict(n_tokens=None), "token list"), (dict(tokens_ld=0), "token list"),
                     (dict(tokens=None), "token list"), (dict(bias_ids=None), "biases"), (dict(bias_ld=0), "biases"), (dict(mask_ld=3), "mask")):
        refused(L, call(**kw), "logits_rules", word)
    refused(L, L.tm_cuda_logits_rules_dev(A, 9, A, 9, 1, 9, None, None), "null")


M = 1 << 24                      # buffers that are apart lie this far apart
ROWS, POOL = 5 * 8 * 64 * 4, 9 * 2 * 16 * 64 * 2                           # bytes of q and out; of the pages that pages() describes


@pytest.mark.parametrize("what,at", [("q", 3 * M - ROWS + 16), ("q", 3 * M + ROWS - 16), ("s", 3 * M - 16), ("s", 3 * M + ROWS - 16), ("s", M + ROWS - 16), ("o", M),
                                     ("o", 4 * M + POOL - 16), ("o", 5 * M - ROWS + 16), ("s", 4 * M + 16), ("s", 5 * M), ("o", 6 * M + 32), ("o", 7 * M), ("s", 8 * M)])
def test_attention_where_buffers_overlap(L, what, at):
    """What the call writes against q, the pages, the table and the lengths."""
    kv = pages(k=4 * M, v=5 * M, table=6 * M, q_begin=7 * M, kv_len=8 * M)
    where = {"q": M, "s": 2 * M, "o": 3 * M, what: at}
    need = L.tm_cuda_attn_paged_scratch(5, 3, 2, 8, 2, 64)
    assert need > 64
    refused(L, L.tm_cuda_attn_paged_dev(C.byref(kv), where["q"], where["s"], need, where["o"], 5, 2, 8, 0, 0, 0.1, None), "attn_paged", "overlaps")
    if at < 6 * M and (what != "s" or at % M < 64):
        refused(L, L.tm_cuda_attn_window_dev(where["q"], 4 * M, 5 * M, where["s"], 1 << 30, where["o"], 5, 0, 8, 2, 64, 9 * 16, 0, 0, 0.1, 1, None), "attn_window", "overlaps")


@pytest.mark.parametrize("what,at", [("q", 4 * M + POOL - 16), ("q", 5 * M), ("x", 4 * M), ("x", 5 * M + POOL - 16), ("q", 6 * M), ("q", 7 * M), ("q", 8 * M), ("v", 4 * M + POOL - 16),
                                     ("v", 4 * M)])
def test_append_where_buffers_overlap(L, what, at):
    where = {"x": M, "q": 2 * M, "v": 5 * M, what: at}
    kv = pages(k=4 * M, v=where["v"], table=6 * M, q_begin=7 * M, kv_len=8 * M)
    refused(L, L.tm_cuda_kv_append_paged_dev(C.byref(kv), where["x"], where["q"], 5, 8, 3 * M, 9, None), "kv_append_paged", "overlap")


@pytest.mark.parametrize("x,ldx,o,ldo,B", [
    (A, 100, A + 400, 100, 2), (A + 400, 100, A, 100, 2), (A, 100, A + 4, 100, 1), (A + 4, 100, A, 100, 1), (A, 100, A, 101, 2), (A, 200, A, 100, 2),
    (A, 200, A + 396, 200, 3), (A, 200, A + 404, 200, 3), (A, 300, A + 400 + 4 * 250 * 9, 250, 40), (A + 4 * 99 + 2, 100, A, 100, 1),
    (A, 1000, A + 4 * 1000 * 65534 + 396, 1000, 65535), (A + 4 * 1000 * 65534, 100, A, 1000, 65535)])
def test_rules_where_rows_overlap(L, x, ldx, o, ldo, B):
    """x one row behind out, another stride, a shift by less than a row: CTAs would read what others have written."""
    r = lib.LogitRules(mask=A, mask_ld=4)
    refused(L, L.tm_cuda_logits_rules_dev(x, ldx, o, ldo, B, 100, C.byref(r), None), "logits_rules", "overlaps")


@pytest.mark.parametrize("name", ["table", "q_begin", "kv_len"])
def test_batch_arrays_between_words(L, name):
    """An address that no load of four bytes may have ends the context, so it does not get as far as a kernel."""
    for by in (1, 2, 3):
        kv = pages(**{name: 9 * M + by})
        refused(L, L.tm_cuda_attn_paged_dev(C.byref(kv), 2 * M, 3 * M, 1 << 30, 4 * M, 5, 2, 8, 0, 0, 0.1, None), "attn_paged", "4-byte")
        refused(L, L.tm_cuda_kv_append_paged_dev(C.byref(kv), 2 * M, 3 * M, 5, 8, 4 * M, 9, None), "kv_append_paged", "4-byte")


@pytest.mark.parametrize("name", ["x", "out", "tokens", "n_tokens", "n_prompt", "repeat", "presence", "frequency", "bias_ids", "bias", "n_bias", "mask"])
def test_rules_arrays_between_words(L, name):
    for by in (1, 2, 3):
        a = {n: M * (i + 1) for i, n in enumerate(["x", "out", "tokens", "n_tokens", "n_prompt", "repeat", "presence", "frequency", "bias_ids", "bias", "n_bias", "mask"])}
        a[name] += by
        x, out = a.pop("x"), a.pop("out")
        r = lib.LogitRules(tokens_ld=5, bias_ld=3, mask_ld=4, **a)
        refused(L, L.tm_cuda_logits_rules_dev(x, 100, out, 100, 2, 100, C.byref(r), None), "logits_rules", "4-byte")


def test_scratch_of_the_largest_call_is_enough(L):
    """A workspace made for a server's largest step serves every smaller one."""
    sizes, out = (0, 1, 2, 3, 4, 5, 8, 9, 16, 17, 64, 1024, 1 << 20), {}
    for H, KVH, dh in ((32, 8, 128), (8, 8, 64), (9, 3, 80), (16, 1, 128), (20, 1, 40), (128, 1, 64)):
        for T in sizes:
            assert L.tm_cuda_attn_window_scratch(T, H, KVH, dh) == L.tm_cuda_attn_paged_scratch(T, 1, T, H, KVH, dh)
            for B in (1, 2, 7, 300):
                for max_q in sizes:
                    out[T, B, max_q] = L.tm_cuda_attn_paged_scratch(T, B, max_q, H, KVH, dh)
                    assert out[T, B, max_q] >= 16 and out[T, B, max_q] % 16 == 0
        for T, B, max_q in out:
            most = max_q or T                                              # 0: not known, as many as T
            for t in sizes:
                for m in sizes:
                    if t <= T and (m or t) <= most:
                        assert all(out[t, b, m] <= out[T, B, max_q] for b in (1, 2, 7, 300) if b <= B), (T, B, max_q, t, m)


def test_nothing_to_do(L):
    """No tokens, no rows: a call that does nothing, with the null pointers that empty tensors have."""
    kv = pages()
    assert L.tm_cuda_attn_paged_dev(C.byref(kv), None, None, 0, None, 0, 0, 8, 0, 0, 0.1, None)
    assert L.tm_cuda_kv_append_paged_dev(C.byref(kv), None, None, 0, 8, None, 0, None)
    assert L.tm_cuda_attn_window_dev(None, None, None, None, 0, None, 0, 10, 8, 2, 64, 10, 0, 0, 0.1, 1, None)
    assert L.tm_cuda_logits_rules_dev(None, 100, None, 100, 0, 100, None, None)


SRC = r"""
#include "kv_pages.cuh"
using namespace tmc;
extern "C" {
// out: q0, n, first, len, lost, bad
void seq(const int* q_begin, const int* kv_len, const int* table, unsigned T, unsigned cap, unsigned b, long long* out) {
    KvBatch c{}; c.q_begin = q_begin; c.kv_len = kv_len; c.table = table; c.T = T; c.cap = cap;
    const KvSeq s = kv_seq(c, b);
    out[0] = s.q0; out[1] = s.n; out[2] = s.first; out[3] = s.len; out[4] = s.lost; out[5] = s.bad;
}
int row(const int* table, unsigned ld, unsigned KVH, unsigned dh, unsigned page, int shift, unsigned npages, unsigned b, unsigned pos, unsigned long long* at) {
    KvBatch c{}; c.table = table; c.table_ld = ld; c.KVH = KVH; c.dh = dh; c.page = page; c.page_shift = shift; c.npages = npages;
    size_t a; const int ok = kv_row(c, b, pos, &a); *at = a; return ok;
}
int sees(unsigned window, unsigned sinks, int p, int j) { return kv_sees(kv_mask(window, sinks), p, j); }
void span(unsigned window, unsigned sinks, int p0, int p1, unsigned* out) { const KvSpan s = kv_span(kv_mask(window, sinks), p0, p1); out[0] = s.a; out[1] = s.b; out[2] = s.e; }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    src = d / "kv.cpp"
    src.write_text(SRC)
    subprocess.run(["g++", "-std=c++20", "-O1", "-fPIC", "-shared", "-I" + os.path.join(ROOT, "tensormark_b200", "csrc"), "-o", str(d / "kv.so"), str(src)], check=True)
    return C.CDLL(str(d / "kv.so"))


def test_sequences_from_bad_arrays(host):
    lo, hi = -2 ** 31, 2 ** 31 - 1
    T, cap = 10, 64
    for a in (lo, -1, 0, 3, 10, 11, hi):
        for e in (lo, -1, 0, 3, 10, 11, hi):
            for n in (lo, -1, 0, 1, 64, 65, hi):
                out = (C.c_longlong * 6)()
                host.seq(np.array([a, e], np.int32).ctypes.data_as(C.c_void_p), np.array([n], np.int32).ctypes.data_as(C.c_void_p), C.c_void_p(1), T, cap, 0, out)
                q0, rows, first, length, lost, bad = out
                assert lost == (not 0 <= a <= e <= T) and bad == (not 0 <= n <= cap)
                assert 0 <= q0 <= q0 + rows <= T and 0 <= length <= cap and first == length - rows
                if not lost and not bad:
                    assert (q0, rows, length) == (a, e - a, n)


def test_rows_of_bad_pages_stay_inside(host):
    ld, KVH, dh, npages = 5, 3, 8, 7
    for page, shift in ((16, 4), (1, 0), (24, -1), (7, -1)):
        rng = np.random.default_rng(page)
        table = rng.choice([-2 ** 31, -1, 0, 3, 6, 7, 2 ** 31 - 1], (4, ld)).astype(np.int32)
        for b in range(4):
            for pos in range(ld * page):
                at = C.c_ulonglong()
                ok = host.row(table.ctypes.data_as(C.c_void_p), ld, KVH, dh, page, shift, npages, b, pos, C.byref(at))
                pg = int(table[b, pos // page])
                assert bool(ok) == (0 <= pg < npages)
                assert at.value == ((pg if ok else 0) * KVH * page + pos % page) * dh
                assert at.value + ((KVH - 1) * page + 1) * dh <= npages * KVH * page * dh


def test_spans_cover_what_is_seen(host):
    out = (C.c_uint * 3)()
    for window in (0, 1, 5, 16, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1):
        for sinks in (0, 1, 4, 30, 2 ** 31, 2 ** 32 - 1):
            for p0 in (-3, 0, 2, 20):
                for p1 in (p0, p0 + 1, p0 + 9):
                    host.span(window, sinks, p0, p1, out)
                    a, b, e = out
                    assert a <= b
                    for j in range(0, 40):
                        seen = any(p >= 0 and j <= p and (not window or window > 2 ** 31 - 1 or j > p - window or j < sinks) for p in range(p0, p1 + 1))
                        assert seen == any(p >= 0 and bool(host.sees(window, sinks, p, j)) for p in range(p0, p1 + 1))
                        if seen:
                            assert j < a or b <= j < e


@pytest.mark.parametrize("dh,keys", [(64, 77), (64, 2000), (128, 200), (128, 333), (128, 2000)])
def test_what_the_precision_bound_breaks_on(dh, keys):
    """The bound on a whole output's error against the same attention with one operand rounded to 11 bits, in 64 bits otherwise."""
    from tests.test_gpu_kv_pages import RMS, reference, rms_error
    rng = np.random.default_rng(keys)
    q, k, v = rng.standard_normal((4, 1, dh)) * 2, rng.standard_normal((keys, 1, dh)), rng.standard_normal((keys, 1, dh))
    want, _ = reference(q, k, v, keys - 4, 0, 0, 1 / np.sqrt(dh))
    eleven = lambda x: np.ldexp(np.round(np.ldexp(np.frexp(x)[0], 11)), np.frexp(x)[1] - 11)  # noqa: E731
    for a in ((eleven(q), k, v), (q, eleven(k), v), (q, k, eleven(v))):
        assert rms_error(reference(*a, keys - 4, 0, 0, 1 / np.sqrt(dh))[0], want) > 8 * RMS
    lost = np.zeros_like(want)
    for i in range(4):
        s = k[:keys - 3 + i, 0] @ q[i, 0] / np.sqrt(dh)
        w = np.exp(s - s.max())
        lost[i, 0] = eleven(w) @ v[:keys - 3 + i, 0] / w.sum()
    assert rms_error(lost, want) > 8 * RMS
