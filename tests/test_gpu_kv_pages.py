"""A batch of sequences over a paged K/V cache: append, attention of new tokens (one or many), windows and sinks, against plain
implementations in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tensormark_b200 import lib, synth
from tests.gpu_util import ptr, stream_ptr

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Batch:
    """Random pages, lengths and queries; the pages that a sequence does not own hold NaN."""

    def __init__(self, torch, new, total, H, KVH, dh, page, half, seed=0, extra_rows=0):
        rng = np.random.default_rng(seed)
        self.torch, self.new, self.total, self.H, self.KVH, self.dh, self.page, self.half = torch, new, list(total), H, KVH, dh, page, half
        self.B, self.T = len(new), sum(new) + extra_rows
        need = [-(-t // page) for t in total]
        self.npages, self.ld = sum(need) + 2, max(need + [0]) + 1
        order = rng.permutation(self.npages).astype(np.int32)
        self.table = np.full((self.B, self.ld), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        kind = np.float16 if half else np.float32
        self.k = rng.standard_normal((self.npages, KVH, page, dh)).astype(kind)
        self.v = rng.standard_normal((self.npages, KVH, page, dh)).astype(kind)
        for a in (self.k, self.v):
            a[order[at:]] = np.nan
            for b, t in enumerate(total):                                  # rows behind the last position, too
                if t % page:
                    a[self.table[b, t // page], :, t % page:] = np.nan
        self.begin = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.q = (rng.standard_normal((self.T, H * dh)) * 2).astype(np.float32)
        self.upload()

    def upload(self):
        t = self.torch
        up = lambda a: t.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.d = {n: up(getattr(self, n)) for n in ("k", "v", "table", "q")}
        self.d["q_begin"], self.d["kv_len"] = up(self.begin), up(np.asarray(self.total, np.int32))
        self.desc = lib.KvPages(B=self.B, KVH=self.KVH, dh=self.dh, page=self.page, npages=self.npages, table_ld=self.ld, kv_half=int(self.half),
                                **{n: self.d[n].data_ptr() for n in ("k", "v", "table", "q_begin", "kv_len")})

    def rows(self, b):
        j = np.arange(self.total[b])
        pg = self.table[b, j // self.page]
        return self.k[pg, :, j % self.page], self.v[pg, :, j % self.page]          # [len, KVH, dh]

    def attend(self, cuda, window=0, sinks=0, max_q=None, scale=None, stream=None, want_ok=True):
        t = self.torch
        scale = 1 / np.sqrt(self.dh) if scale is None else scale
        max_q = max(self.new) if max_q is None else max_q
        need = cuda.tm_cuda_attn_paged_scratch(self.T, self.B, max_q, self.H, self.KVH, self.dh)
        scratch = t.full((need // 4 + 1,), float("nan"), device="cuda")
        out = t.full((self.T, self.H * self.dh), 7.0, device="cuda")
        lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(self.desc), ptr(self.d["q"]), ptr(scratch), need, ptr(out), self.T, max_q, self.H, window, sinks,
                                              scale, stream_ptr(t)), "attn_paged")
        t.cuda.synchronize()
        assert cuda.tm_cuda_tok_flush() == want_ok, lib.last_error()
        return out.cpu().numpy()

    def check(self, cuda, window=0, sinks=0, **kw):
        got = self.attend(cuda, window, sinks, **kw)
        self.verify(got, window, sinks, kw.get("scale"))
        assert np.all(got[self.begin[-1]:] == 7.0)                          # rows behind the last sequence
        return got

    def verify(self, got, window=0, sinks=0, scale=None, skip=()):
        for b in set(range(self.B)) - set(skip):
            q = self.q[self.begin[b]:self.begin[b + 1]].reshape(-1, self.H, self.dh)
            k, v = self.rows(b)
            want, tol = reference(q, k, v, self.total[b] - self.new[b], window, sinks, scale or 1 / np.sqrt(self.dh))
            mine = got[self.begin[b]:self.begin[b + 1]].reshape(-1, self.H, self.dh)
            assert np.array_equal(np.isnan(mine), np.isnan(want)), (b, "NaN in other places")
            fine = np.isfinite(want)
            assert np.array_equal(mine[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
            off = np.where(fine, np.abs(mine - np.where(fine, want, 0)), 0)
            assert np.all(off[fine] <= tol[fine]), (b, float((off / np.where(tol > 0, tol, 1)).max()), float(off.max()))


# Root mean square of an output's error over that of the output, for values drawn independently. With relative errors e_j of the weights
# the output is off by sum w_j e_j v_j, and sum w_j v_j is what it is, so this is the e_j's root mean square. An e_j is a score's error (in
# powers of two, times ln 2): the dominant scores of queries of standard deviation 2 lie below 16, where a step is 2^-20. A tensor core
# cuts its sum at dh / 16 steps (fp16; dh / 8 over fp32 caches), 0.3 of a step each at random and up to half a step alike for all large
# scores but not for small ones, at most 8 steps of 2^-20 for 16 of them; the sums of low parts, the maximum's subtraction and ex2 add one
# more. 9 ln 2 2^-20 < 2^-17. Weights, queries, keys or values without their low parts are off by half a step of 11 bits: 2^-11 / sqrt(3) x
# 0.72 = 2^-12.3 (queries and keys: twice that, a score's deviation being 2), 26 times as much.
RMS = 2.0 ** -17


def rms_error(got, want):
    return float(np.sqrt(np.mean((got - want) ** 2)) / np.sqrt(np.mean(want ** 2)))


def reference(q, k, v, first, window, sinks, scale):
    """q [n, H, dh], k and v [len, KVH, dh] -> out [n, H, dh] in 64 bits, and how far an fp32-grade kernel may be from it: a score is off by its
    products' rounding (two halves of q: 2^-22, accumulation of dh products and their halves in any order: (dh + 8) roundings), at most
    A (dh + 12) u with A the sum of their magnitudes; a weight by that (in powers of two: x log2 e, which the sums do not see, and a
    rounding of the argument) + 2^-21; the sums of weights and products by as many roundings as there are additions in a chain, of
    which a kernel that sums 16 keys at a time has len / 16 + 64. Numerator and denominator: twice."""
    n, H, dh = q.shape
    L, KVH = k.shape[0], k.shape[1]
    out, tol = np.zeros((n, H, dh)), np.zeros((n, H, dh))
    p, j = first + np.arange(n)[:, None], np.arange(L)[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    with np.errstate(all="ignore"):
        for h in range(H):
            kk, vv = k[:, h // (H // KVH)].astype(np.float64), v[:, h // (H // KVH)].astype(np.float64)
            for i in range(n):
                vis = seen[i]
                if not vis.any():
                    continue
                x, K, V = q[i, h].astype(np.float64), kk[vis], vv[vis]
                s = K @ x * scale
                A = np.abs(K) @ np.abs(x) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h] = w @ V
                size = w @ np.abs(V)
                tol[i, h] = 2 * size * ((A.max() if np.isfinite(A).all() else 0) * (dh + 13) * U + 2.0 ** -21 + (vis.sum() / 16 + 64) * U)
    return out, tol


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("rep", [1, 2, 3, 4, 5, 8, 16])
def test_single_tokens(cuda, torch_mod, rep, dh, half):
    Batch(torch_mod, [1] * 5, [1, 16, 17, 333, 64], 2 * rep, 2, dh, 16, half, seed=rep).check(cuda)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rep,dh,page", [(4, 128, 16), (1, 64, 1), (3, 64, 24), (8, 128, 64), (7, 8, 5), (4, 80, 256), (20, 40, 16), (128, 64, 16), (5, 120, 48)])
def test_chunks(cuda, torch_mod, rep, dh, page, half):
    """Ragged chunks: one token to some hundred, chunks that are the whole sequence, sequences without new tokens, an empty cache."""
    Batch(torch_mod, [1, 33, 0, 7, 130], [200, 33, 50, 8, 391], 2 * rep, 2, dh, page, half, seed=page).check(cuda)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rep,dh,new,total", [(4, 128, [1, 1, 1], [200, 333, 2000]), (4, 64, [1, 1, 1], [77, 333, 2000]), (4, 128, [4, 3], [200, 1500]), (8, 64, [2, 2], [200, 1500]),
                                              (16, 128, [1, 1], [333, 2000]), (4, 128, [150, 1, 70], [200, 333, 700]), (8, 64, [90, 200], [600, 200]), (1, 128, [300], [2000]),
                                              (4, 128, [1], [5000])])
def test_low_parts_count(cuda, torch_mod, rep, dh, new, total, half):
    """Results as good as fp32's over a whole output: each kernel, with its low parts."""
    b = Batch(torch_mod, new, total, 2 * rep, 2, dh, 16, half, seed=dh + rep)
    got = b.check(cuda)
    for s in range(b.B):
        r = slice(b.begin[s], b.begin[s + 1])
        want, _ = reference(b.q[r].reshape(-1, b.H, dh), *b.rows(s), total[s] - new[s], 0, 0, 1 / np.sqrt(dh))
        assert rms_error(got[r].reshape(want.shape), want) <= RMS, (s, rms_error(got[r].reshape(want.shape), want))


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (63, 4), (64, 64), (100, 70), (130, 200), (5000, 4), (2 ** 31, 2 ** 32 - 1), (40, 2 ** 31)])
def test_windows(cuda, torch_mod, window, sinks, half):
    Batch(torch_mod, [1, 1, 70, 3], [1, 300, 333, 129], 8, 2, 64, 16, half, seed=window % 97).check(cuda, window, sinks)
    Batch(torch_mod, [1, 2], [517, 90], 4, 1, 128, 7, half, seed=sinks % 89).check(cuda, window, sinks)


@pytest.mark.parametrize("half", [True, False])
def test_long_and_ragged(cuda, torch_mod, half):
    Batch(torch_mod, [1] * 9, [4000, 1, 2, 700, 65, 64, 63, 5000, 128], 8, 2, 128, 16, half, seed=3).check(cuda)
    Batch(torch_mod, [2, 300], [2500, 2000], 8, 2, 128, 32, half, seed=4).check(cuda)
    Batch(torch_mod, [1] * 300, list(range(1, 301)), 4, 2, 64, 8, half, seed=5).check(cuda)


@pytest.mark.parametrize("B,KVH,rep,dh,longest,window", [
    (1, 8, 4, 128, 20000, 0), (1, 8, 4, 128, 3000, 0), (1, 1, 8, 64, 9000, 0), (1, 149, 1, 64, 130, 0), (2, 8, 4, 128, 400, 0), (5, 8, 2, 64, 900, 100),
    (9, 8, 4, 128, 450, 0), (18, 8, 1, 64, 300, 0), (19, 8, 4, 128, 700, 60), (37, 8, 4, 64, 450, 0), (38, 8, 4, 64, 450, 0), (36, 8, 16, 128, 200, 0),
])
def test_around_one_launch_and_two(cuda, torch_mod, B, KVH, rep, dh, longest, window):
    """Clusters of 16 CTAs down to one, and the list of tiles: a sequence of the longest length, others anywhere below it."""
    rng = np.random.default_rng(B)
    total = [longest] + rng.integers(1, longest + 1, B - 1).tolist()
    for half in (True, False):
        Batch(torch_mod, [1] * B, total, KVH * rep, KVH, dh, 16, half, seed=B).check(cuda, window, 3)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,total,H,KVH,dh,window", [([5], [3000], 8, 2, 128, 0), ([9], [700], 4, 1, 64, 0), ([20], [1500], 4, 1, 128, 130), ([130], [900], 4, 1, 64, 0),
                                                       ([66], [66], 8, 8, 128, 0), ([257, 64], [300, 1000], 4, 4, 64, 40), ([40, 1, 33, 1], [900, 200, 33, 1], 8, 2, 128, 500)])
def test_shared_keys_of_a_chunk(cuda, torch_mod, new, total, H, KVH, dh, window, half):
    """Tiles of rows whose keys one to eight CTAs share, some of them without a key."""
    Batch(torch_mod, new, total, H, KVH, dh, 16, half, seed=new[0]).check(cuda, window, 5)


@pytest.mark.parametrize("half", [True, False])
def test_many_sequences_beside_chunks(cuda, torch_mod, half):
    """A batch of which most decode: the CTAs for chunks that might have been there find none."""
    new = [1] * 150 + [70] + [0] * 40 + [300] + [2] * 120
    total = [n + (37 * i) % 200 for i, n in enumerate(new)]
    Batch(torch_mod, new, total, 8, 2, 64, 16, half, seed=21).check(cuda, 90, 4)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,total,window", [([1] * 60, None, 0), ([1], [5000], 0), ([5, 1], [3000, 40], 700), ([300, 1], [900, 77], 0)])
def test_scratch_is_enough(cuda, torch_mod, new, total, window, half):
    """Nothing is written behind the scratch that was asked for, nor behind out or before it."""
    t = torch_mod
    total = total or [100 + 53 * i for i in range(len(new))]
    b = Batch(t, new, total, 8, 2, 128, 16, half, seed=31)
    need = cuda.tm_cuda_attn_paged_scratch(b.T, b.B, max(new), b.H, b.KVH, b.dh)
    assert need % 16 == 0
    scratch, out = t.full((need // 4 + 64,), 3.0, device="cuda"), t.full((b.T + 2, b.H * b.dh), 7.0, device="cuda")
    lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(out[1:]), b.T, max(new), b.H, window, 2, 1 / np.sqrt(128),
                                          stream_ptr(t)), "attn_paged")
    t.cuda.synchronize()
    assert bool((scratch[need // 4:] == 3.0).all()) and bool((out[0] == 7.0).all()) and bool((out[-1] == 7.0).all())
    b.verify(out[1:-1].cpu().numpy(), window, 2)


@pytest.mark.parametrize("half", [True, False])
def test_one_scratch_for_a_server(cuda, torch_mod, half):
    """Scratch for the prompts' step, then the same for chunks, drafts and single tokens of fewer sequences."""
    t = torch_mod
    H, KVH, dh = 8, 2, 128
    for T, B, max_q in ((700, 1, 700), (700, 5, 600), (900, 5, 0)):
        need = cuda.tm_cuda_attn_paged_scratch(T, B, max_q, H, KVH, dh)
        scratch = t.full((need // 4 + 16,), 3.0, device="cuda")
        for new, total in (([1], [4000]), ([4], [3000]), ([300], [500]), ([1] * 5, [900, 2000, 5, 77, 3100]), ([200, 1, 3], [200, 2500, 900]), ([5, 5, 4], [1800, 30, 700])):
            if len(new) > B:
                continue
            b = Batch(t, new, total, H, KVH, dh, 16, half, seed=len(new))
            out = t.full((b.T, H * dh), 7.0, device="cuda")
            lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(out), b.T, max(new), H, 0, 0, 1 / np.sqrt(dh), stream_ptr(t)), "attn_paged")
            t.cuda.synchronize()
            b.verify(out.cpu().numpy())
        assert bool((scratch[need // 4:] == 3.0).all())


@pytest.mark.parametrize("half", [True, False])
def test_offsets_past_32_bits(cuda, torch_mod, half):
    """A cache of more than 2^32 elements: pages at both of its ends, written by append and read by attention, single tokens and a chunk."""
    t, rng = torch_mod, np.random.default_rng(6)
    H, KVH, dh, page = 8, 2, 128, 16
    npages = 2 ** 32 // (KVH * page * dh) + 40
    kind = t.float16 if half else t.float32
    k, v = (t.empty(npages, KVH, page, dh, dtype=kind, device="cuda") for _ in range(2))
    total, new = [90, 60, 33], [90, 60, 33]
    table = np.full((3, 7), -1, np.int32)
    table[0, :6] = npages - 1 - np.arange(6)
    table[1, :4] = [0, npages - 30, 1, npages - 20]
    table[2, :3] = [npages - 10, npages // 2 + 1, 5]
    begin = np.array([0, 90, 150, 183], np.int32)
    qkv = rng.standard_normal((183, (H + 2 * KVH) * dh)).astype(np.float32)
    d = {"table": t.from_numpy(table).cuda(), "q_begin": t.from_numpy(begin).cuda(), "kv_len": t.tensor(total, dtype=t.int32, device="cuda")}
    desc = lib.KvPages(k=k.data_ptr(), v=v.data_ptr(), B=3, KVH=KVH, dh=dh, page=page, npages=npages, table_ld=7, kv_half=int(half), **{n: x.data_ptr() for n, x in d.items()})
    dq, q, out = t.from_numpy(qkv).cuda(), t.empty(183, H * dh, device="cuda"), t.empty(183, H * dh, device="cuda")
    lib.check(cuda.tm_cuda_kv_append_paged_dev(C.byref(desc), ptr(dq), ptr(q), 183, H, None, 0, stream_ptr(t)), "append")

    def attend(T, max_q, rows):
        need = cuda.tm_cuda_attn_paged_scratch(T, 3, max_q, H, KVH, dh)
        scratch = t.empty(need // 4 + 1, device="cuda")
        lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(desc), ptr(rows), ptr(scratch), need, ptr(out), T, max_q, H, 0, 0, 1 / np.sqrt(dh), stream_ptr(t)), "attention")
        t.cuda.synchronize()
        assert cuda.tm_cuda_tok_flush()
        return out.cpu().numpy()

    got = attend(183, 90, q)
    x = qkv.reshape(-1, H + 2 * KVH, dh)
    held = lambda a: a.astype(np.float16).astype(np.float32) if half else a  # noqa: E731
    for b in range(3):
        r = slice(begin[b], begin[b + 1])
        want, tol = reference(x[r, :H], held(x[r, H:H + KVH]), held(x[r, H + KVH:]), 0, 0, 0, 1 / np.sqrt(dh))
        assert np.all(np.abs(got[r].reshape(-1, H, dh) - want) <= tol)
    d["q_begin"].copy_(t.arange(4, dtype=t.int32))                          # the last token of each again, as a decode step
    got = attend(3, 1, q[t.from_numpy(begin[1:] - 1).long().cuda()].contiguous())
    for b in range(3):
        r = slice(begin[b], begin[b + 1])
        want, tol = reference(x[r, :H][-1:], held(x[r, H:H + KVH]), held(x[r, H + KVH:]), total[b] - 1, 0, 0, 1 / np.sqrt(dh))
        assert np.all(np.abs(got[b].reshape(1, H, dh) - want) <= tol)
    del k, v
    t.cuda.empty_cache()


@pytest.mark.parametrize("T", [1, 40])
def test_far_into_a_long_contiguous_cache(cuda, torch_mod, T):
    t, rng = torch_mod, np.random.default_rng(7)
    KVH, H, dh, ctx = 8, 16, 64, 4_300_000                                   # 2.2e9 elements
    first = ctx - 60
    k, v = (t.empty(KVH, ctx, dh, dtype=t.float16, device="cuda") for _ in range(2))
    near = {n: rng.standard_normal((KVH, 300, dh)).astype(np.float16) for n in "kv"}
    sink = {n: rng.standard_normal((KVH, 3, dh)).astype(np.float16) for n in "kv"}
    for n, c in (("k", k), ("v", v)):
        c[:, ctx - 300:] = t.from_numpy(near[n]).cuda()
        c[:, :3] = t.from_numpy(sink[n]).cuda()
    q = rng.standard_normal((T, H * dh)).astype(np.float32)
    dq, out = t.from_numpy(q).cuda(), t.empty(T, H * dh, device="cuda")
    need = cuda.tm_cuda_attn_window_scratch(T, H, KVH, dh)
    scratch = t.empty(need // 4 + 1, device="cuda")
    lib.check(cuda.tm_cuda_attn_window_dev(ptr(dq), ptr(k), ptr(v), ptr(scratch), need, ptr(out), T, first, H, KVH, dh, ctx, 200, 3, 0.125, 1, stream_ptr(t)), "window")
    t.cuda.synchronize()
    got = out.cpu().numpy().reshape(T, H, dh)
    for i in range(T):                                                      # the keys that token i sees, at positions of their own
        p = first + i
        lo = p - 199 - (ctx - 300)
        kk, vv = (np.concatenate((sink[n], near[n][:, lo:p + 1 - (ctx - 300)]), 1).transpose(1, 0, 2) for n in "kv")
        want, tol = reference(q[i].reshape(1, H, dh), kk, vv, len(kk) - 1, 0, 0, 0.125)
        assert np.all(np.abs(got[i:i + 1] - want) <= tol)
    del k, v, c
    t.cuda.empty_cache()


def test_graphs_that_share_scratch(cuda, torch_mod):
    """Two captured graphs with one scratch, replayed in turn, while lengths and ranges of rows change between replays: sequences come and go."""
    t = torch_mod
    b = Batch(t, [1] * 40, [200 + 9 * i for i in range(40)], 8, 2, 128, 16, True, seed=41)
    need = cuda.tm_cuda_attn_paged_scratch(b.T, b.B, 1, b.H, b.KVH, b.dh)
    scratch, outs, graphs = t.empty(need // 4 + 1, device="cuda"), [], []
    side = t.cuda.Stream()

    def call(out, window, s):
        lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(out), b.T, 1, b.H, window, 2, 1 / np.sqrt(128), s), "attention")

    for window in (0, 90):
        out = t.full((b.T, b.H * b.dh), 7.0, device="cuda")
        with t.cuda.stream(side):
            call(out, window, stream_ptr(t))
        side.synchronize()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            call(out, window, stream_ptr(t))
        outs.append(out); graphs.append(g)
    lengths = list(b.total)
    for turn in range(4):
        here = [int((i + turn) % 3 != 0) for i in range(40)]                # one new token, or none
        b.new, b.total = here, [n - 30 * turn for n in lengths]
        b.begin = np.concatenate([[0], np.cumsum(here)]).astype(np.int32)
        b.d["q_begin"].copy_(t.from_numpy(b.begin)); b.d["kv_len"].copy_(t.tensor(b.total, dtype=t.int32))
        for out in outs:
            out.fill_(7.0)
        for g in graphs + graphs[::-1]:
            g.replay()
        t.cuda.synchronize()
        for out, window in zip(outs, (0, 90)):
            got = out.cpu().numpy()
            b.verify(got, window, 2)
            assert np.all(got[b.begin[-1]:] == 7.0)


def test_two_calls_at_once(cuda, torch_mod):
    """Two batches on two streams at a time, each with scratch of its own."""
    t = torch_mod
    batches = [Batch(t, [1] * 30, list(range(100, 1600, 50)), 32, 8, 128, 16, True, seed=1), Batch(t, [200, 1], [900, 300], 8, 2, 64, 16, True, seed=2)]
    streams, outs, keep = [t.cuda.Stream() for _ in batches], [], []
    t.cuda.synchronize()
    for b in batches:
        need = cuda.tm_cuda_attn_paged_scratch(b.T, b.B, max(b.new), b.H, b.KVH, b.dh)
        keep.append((t.empty(need // 4 + 1, device="cuda"), need))
        outs.append(t.full((b.T, b.H * b.dh), 7.0, device="cuda"))
    t.cuda.synchronize()
    for _ in range(10):
        for b, s, o, (scratch, need) in zip(batches, streams, outs, keep):
            lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(o), b.T, max(b.new), b.H, 0, 0, 1 / np.sqrt(b.dh),
                                                  C.c_void_p(s.cuda_stream)), "attn_paged")
    t.cuda.synchronize()
    for b, o in zip(batches, outs):
        b.verify(o.cpu().numpy())


@pytest.mark.parametrize("half", [True, False])
def test_rows_that_see_nothing(cuda, torch_mod, half):
    """More new tokens than positions: those before position 0 give zeros. Rows of q and out behind the last sequence stay."""
    Batch(torch_mod, [3, 40, 5], [1, 0, 5], 4, 2, 64, 16, half, seed=1, extra_rows=4).check(cuda)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,total", [([1, 1], [100, 40]), ([50, 100], [120, 100])])
def test_nan_and_infinity_in_masked_places(cuda, torch_mod, new, total, half):
    """Keys and values that only later tokens see, or that the window hides, hold NaN and infinity."""
    b = Batch(torch_mod, new, total, 8, 2, 64, 16, half, seed=9)
    for s, t in enumerate(total):
        for pos, bad in ((t - 1, np.inf), (t - 2, np.nan), (20, -np.inf), (10, np.nan)):
            pg = b.table[s, pos // 16]
            b.v[pg, 1, pos % 16, ::3] = bad
            b.k[pg, 0, pos % 16, 5] = np.nan
    b.upload()
    b.check(cuda, window=18, sinks=2)
    b.check(cuda)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,total,window", [([1, 3], [100, 700], 0), ([1], [4000], 0), ([50, 100, 1], [120, 100, 90], 60), ([1] * 70, [60 + 20 * i for i in range(70)], 0)])
def test_infinity_in_keys_that_are_seen(cuda, torch_mod, new, total, window, half):
    """A key of minus infinity against positive queries has no weight, whatever its value; of plus infinity, or against a query of zero, the row is NaN."""
    b = Batch(torch_mod, new, total, 8, 2, 64, 16, half, seed=19)
    b.q.reshape(b.T, 8, 64)[:, :, 5] = np.abs(b.q.reshape(b.T, 8, 64)[:, :, 5]) + np.float32(0.1)
    for s, t in enumerate(total):
        for pos in (t - 1 - (s % 7), t - 9, 3):
            b.k[b.table[s, pos // 16], :, pos % 16, 5] = -np.inf
    b.upload()
    got = b.check(cuda, window, 2)
    assert np.isfinite(got).all()
    q, pos = b.q.reshape(b.T, 8, 64), total[-1] - 9
    q[b.begin[1] if b.B > 1 else 0:, 2:4, 5] = 0                           # some rows of every later sequence
    b.k[b.table[-1, pos // 16], 1, pos % 16, 9] = np.inf                   # and of the last one by the query's sign
    b.upload()
    b.check(cuda, window, 2)


@pytest.mark.parametrize("half", [True, False])
def test_many_short_sequences(cuda, torch_mod, half):
    """More sequences than a CTA has threads, many times over: append and attention; single tokens and, beside a chunk, several launches."""
    t, rng = torch_mod, np.random.default_rng(23)
    for B, first in ((3000, 1), (2500, 90)):
        new = [first] + [int(x) for x in rng.integers(0, 3, B - 1)]
        total = [n + int(x) for n, x in zip(new, rng.integers(0, 20, B))]
        b = Batch(t, new, total, 4, 2, 8, 4, half, seed=B, extra_rows=1)
        b.check(cuda)
        qkv = rng.standard_normal((b.T, (4 + 4) * 8)).astype(np.float32)
        q, k, v = append(cuda, b, None, qkv)
        assert np.array_equal(q[:-1], qkv[:-1, :32]) and np.all(q[-1] == 7.0)
        kind = np.float16 if half else np.float32
        x = qkv.reshape(b.T, 8, 8)
        for s in range(B):
            for i in range(new[s]):
                pos, row = total[s] - new[s] + i, b.begin[s] + i
                at = b.table[s, pos // 4], slice(None), pos % 4
                assert np.array_equal(k[at], x[row, 4:6].astype(kind)) and np.array_equal(v[at], x[row, 6:].astype(kind))


@pytest.mark.parametrize("half", [True, False])
def test_values_over_the_range(cuda, torch_mod, half):
    """Large and small queries, keys near fp16's ends, weights that vanish: the scores decide, not the number format of the products."""
    for gain in (1e-6, 1e-2, 30.0, 1e4):
        b = Batch(torch_mod, [1, 40], [150, 200], 8, 2, 64, 16, half, seed=11)
        b.q = (b.q * np.float32(gain)).astype(np.float32)
        b.k = np.where(np.isnan(b.k), b.k, b.k * b.k.dtype.type(min(1.0, 10 / gain))).astype(b.k.dtype)
        b.upload()
        b.check(cuda)
    b = Batch(torch_mod, [1, 40], [150, 200], 8, 2, 64, 16, half, seed=12)
    b.k, b.v = (b.k * b.k.dtype.type(8000)).astype(b.k.dtype), (b.v * b.v.dtype.type(8000)).astype(b.v.dtype)
    b.q[:, ::7] = 0
    b.upload()
    b.check(cuda, scale=1e-5)


@pytest.mark.parametrize("gain,share", [(1e-25, 1.0), (1e31, 1.0), (1e35, 1.0), (1e37, 0.02), (3.3e38, 1.0), (3.3e38, 0.02)])
@pytest.mark.parametrize("new,total,window", [([1] * 60, [90 + 31 * i for i in range(60)], 0), ([1], [5000], 0), ([4, 4], [3000, 40], 700), ([40, 1, 33, 1], [900, 200, 33, 1], 0),
                                              ([1, 20], [300, 1500], 130)])
def test_values_near_the_ends_of_fp32(cuda, torch_mod, new, total, window, gain, share):
    """An fp32 cache's values up to fp32's largest (all of them, or some keys'): a mean of them is finite, whatever the sum of so many is. Small
    ones: products of 2^-83 and their low parts, 2^-12 and 2^-24 of that, are far from fp32's smallest normal number."""
    b = Batch(torch_mod, new, total, 8, 2, 64, 16, False, seed=13)
    rng = np.random.default_rng(14)
    big = (rng.choice([-1.0, 1.0], b.v.shape) * rng.uniform(0.25, 1, b.v.shape) * gain).astype(np.float32)
    some = rng.random(b.v.shape[:3])[..., None] < share
    b.v = np.where(np.isnan(b.v) | ~some, b.v, big)
    b.v[..., 7] = np.where(np.isnan(b.v[..., 7]), b.v[..., 7], np.float32(gain))       # one dim has the same value everywhere: so has its mean
    b.upload()
    got = b.check(cuda, window, 2)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("rep,new", [(4, [1, 1, 1]), (4, [60, 1, 3])])
def test_bad_arrays_are_reported(cuda, torch_mod, rep, new):
    """A page, a length and a range of rows that are not there: NaN in the rows that need them, the others right, and an error."""
    total = [max(t, n) for t, n in zip([40, 300, 77], new)]
    make = lambda: Batch(torch_mod, new, total, 2 * rep, 2, 64, 16, True, seed=2)  # noqa: E731
    for page in (-1, make().npages, 2 ** 31 - 1, -2 ** 31):
        b = make()
        b.table[1, 2] = page
        b.upload()
        got = b.attend(cuda, want_ok=False)
        assert "out of range" in lib.last_error()
        assert np.isnan(got[b.begin[1]:b.begin[2]]).all()
        b.verify(got, skip=[1])
    for length in (-1, make().ld * 16 + 1, 2 ** 31 - 1):
        b = make()
        b.total[1] = length
        b.upload()
        got = b.attend(cuda, want_ok=False)
        assert np.isnan(got[b.begin[1]:b.begin[2]]).all()
        b.verify(got, skip=[1])
    for spoil, skip in ({2: b.T + 5, 3: b.T + 5}, [1, 2]), ({0: -3}, [0]), ({3: 2 ** 31 - 1}, [2]):
        b = make()
        good = b.begin.copy()
        for i, v in spoil.items():
            b.begin[i] = v
        b.upload()
        b.begin = good
        got = b.attend(cuda, want_ok=False)
        b.verify(got, skip=skip)
        for i in skip:
            assert np.all(got[good[i]:good[i + 1]] == 7.0)
    b = make()
    b.begin[2] = 0                                                         # not ascending: which rows are left is not said, only that it is noticed
    b.upload()
    b.attend(cuda, want_ok=False)


def test_a_wait_that_ran_out_is_reported_first(cuda, torch_mod):
    """A batch's bad page behind a lane's wait for a rank that is not there: the next synchronising entry names the wait, whose results are lost too."""
    t, L = torch_mod, cuda
    n, k, dt, xs, ys, zs, st = 64, 256, synth.Q4_0, 60, 61, 62, 63
    W, x = synth.make_weights(dt, n, k, seed=1), synth.make_activations(k, seed=2)
    b = Batch(t, [1, 1], [40, 30], 8, 2, 64, 16, True, seed=2)
    b.table[1, 1] = b.npages
    b.upload()
    need = L.tm_cuda_attn_paged_scratch(2, 2, 1, 8, 2, 64)
    scratch, out = t.empty(need // 4 + 1, device="cuda"), t.empty(2, 8 * 64, device="cuda")
    t.cuda.synchronize()
    handle = (C.c_ubyte * int(L.tm_cuda_peer_handle_bytes()))()
    assert L.tm_cuda_peer_arena(1 << 20, handle), lib.last_error()
    prev = L.tm_cuda_set_wait_limit_ms(100)
    try:
        assert L.tm_cuda_peer_open_loopback(0, 2), lib.last_error()
        assert L.tm_cuda_tok_reserve(xs, 4 * k) and L.tm_cuda_tok_reserve(zs, 4 * n) and L.tm_cuda_tok_reserve(st, 64) and L.tm_cuda_tok_reserve_shared(ys, 4 * n)
        state, woff = np.zeros(4, np.int32), C.c_uint64(0)
        assert L.tm_cuda_tok_upload(st, 0, state.ctypes.data, 16) and L.tm_cuda_tok_upload(xs, 0, x.ctypes.data, x.nbytes)
        wid = L.tm_cuda_tok_wbuf(W.ctypes.data, W.nbytes, None, 0, 0, C.byref(woff))
        assert wid >= 1000, lib.last_error()

        def gemv(to, wait_site, push_site):
            L.tm_cuda_tok_gemv_xchg(xs, 0, 0, 0, 0, None, 0.0, wid, to, (C.c_size_t * 1)(0), n, k, dt, (C.c_uint64 * 1)(woff.value), (C.c_uint * 1)(n), 1, 0,
                                    wait_site, push_site, st)

        assert L.tm_cuda_tok_begin()
        gemv(ys, -1, 5)
        assert L.tm_cuda_tok_flush(), lib.last_error()
        assert L.tm_cuda_tok_begin()
        gemv(zs, 5, -1)                                                    # for what the other rank has not pushed
        t.cuda.synchronize()
        lib.check(L.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(out), 2, 1, 8, 0, 0, 0.125, stream_ptr(t)), "attention")
        t.cuda.synchronize()
        assert not L.tm_cuda_tok_flush()
        assert "bounded wait" in lib.last_error() and "status 2" in lib.last_error(), lib.last_error()
        assert bool(t.isnan(out[1]).all()) and not bool(t.isnan(out[0]).any())
        assert L.tm_cuda_tok_flush(), lib.last_error()
    finally:
        L.tm_cuda_set_wait_limit_ms(prev)
        L.tm_cuda_peer_unmap()
        L.tm_cuda_peer_close()
    b.attend(cuda, want_ok=False)                                          # by itself it is what is reported
    assert "out of range" in lib.last_error()


def test_more_new_tokens_than_said(cuda, torch_mod):
    """max_q is a promise: a sequence that breaks it gets NaN or its right rows, an error in the first case, and the others are right."""
    b = Batch(torch_mod, [1, 40, 1], [100, 200, 30], 8, 2, 64, 16, True, seed=6)
    want = b.check(cuda)
    b.torch.cuda.synchronize()
    need = cuda.tm_cuda_attn_paged_scratch(b.T, b.B, 1, b.H, b.KVH, b.dh)
    scratch = torch_mod.empty(need // 4 + 1, device="cuda")
    out = torch_mod.full((b.T, b.H * b.dh), 7.0, device="cuda")
    assert cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(b.d["q"]), ptr(scratch), need, ptr(out), b.T, 1, b.H, 0, 0, 0.125, stream_ptr(torch_mod))
    torch_mod.cuda.synchronize()
    assert not cuda.tm_cuda_tok_flush()
    got = out.cpu().numpy()
    assert np.isnan(got[1:41]).all() and np.array_equal(got[0], want[0]) and np.array_equal(got[41], want[41])


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rep,new,total", [(4, [1, 1, 1], [40, 300, 77]), (4, [60, 2, 3], [60, 300, 77]), (2, [3, 90, 70], [40, 300, 77]), (4, [40], [900]), (4, [1], [3000]), (20, [1, 33], [90, 400])])
def test_bad_arrays_by_each_kernel(cuda, torch_mod, rep, new, total, half):
    """A page, a length and a range of rows that are not there, in each sequence's turn: single tokens, chunks beside them, keys that a cluster shares."""
    make = lambda: Batch(torch_mod, new, total, 2 * rep, 2, 64, 16, half, seed=2)  # noqa: E731
    good = make()
    for s in range(good.B):
        rows = slice(good.begin[s], good.begin[s + 1])
        for slot in (0, (total[s] - new[s]) // 16):                        # pages that all of the sequence's new tokens see
            for page in (-1, good.npages, 2 ** 31 - 1, -2 ** 31):
                b = make()
                b.table[s, slot] = page
                b.upload()
                got = b.attend(cuda, want_ok=False)
                assert "out of range" in lib.last_error() and np.isnan(got[rows]).all()
                b.verify(got, skip=[s])
        for length in (-1, good.ld * 16 + 1, 2 ** 31 - 1, -2 ** 31):
            b = make()
            b.total[s] = length
            b.upload()
            got = b.attend(cuda, want_ok=False)
            assert np.isnan(got[rows]).all()
            b.verify(got, skip=[s])
        for begin in (-1, -2 ** 31, 2 ** 31 - 1, good.T + 1):              # of this sequence, and the end of the one before it
            b = make()
            b.begin[s] = begin
            b.upload()
            b.begin = good.begin
            got = b.attend(cuda, want_ok=False)
            b.verify(got, skip=[s, s - 1] if s else [s])
            for i in {s, max(s - 1, 0)}:
                assert np.all(got[good.begin[i]:good.begin[i + 1]] == 7.0)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rep,new,max_q", [(4, [1, 40, 1, 2], 10), (4, [1, 300, 10, 1], 10), (1, [17, 2, 18], 17), (2, [3, 1, 16, 8], 8), (16, [1, 2], 1), (20, [1, 5, 2], 2)])
def test_a_broken_promise_by_each_kernel(cuda, torch_mod, rep, new, max_q, half):
    """Sequences with more new tokens than max_q are NaN whichever kernel they would go to, all others right."""
    total = [n + 50 + 97 * i for i, n in enumerate(new)]
    b = Batch(torch_mod, new, total, 2 * rep, 2, 64, 16, half, seed=6, extra_rows=3)
    long = [s for s, n in enumerate(new) if n > max_q]
    got = b.attend(cuda, max_q=max_q, want_ok=False)
    assert "out of range" in lib.last_error()
    b.verify(got, skip=long)
    for s in long:
        assert np.isnan(got[b.begin[s]:b.begin[s + 1]]).all(), s
    assert np.all(got[b.begin[-1]:] == 7.0)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,total", [([1] * 6, [40, 300, 1, 77, 16, 2000]), ([1], [700]), ([9], [700]), ([3, 90, 1], [500, 90, 1200])])
def test_max_q_that_is_not_known(cuda, torch_mod, new, total, half):
    """max_q = 0: as many as T."""
    b = Batch(torch_mod, new, total, 8, 2, 128, 16, half, seed=16, extra_rows=5)
    b.check(cuda, max_q=0)
    b.check(cuda, window=100, sinks=3, max_q=0)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("H,KVH,dh,T,pos0,ctx,window,sinks", [
    (8, 2, 128, 1, 0, 1, 0, 0), (8, 2, 128, 1, 999, 1000, 100, 4), (32, 8, 64, 1, 4000, 4100, 1000, 4), (4, 1, 64, 200, 0, 200, 0, 0),
    (6, 2, 80, 77, 130, 300, 50, 3), (8, 2, 128, 257, 300, 600, 64, 1), (16, 1, 128, 9, 77, 100, 0, 0), (5, 5, 64, 130, 1, 200, 200, 2),
])
def test_contiguous(cuda, torch_mod, H, KVH, dh, T, pos0, ctx, window, sinks, half):
    t, rng = torch_mod, np.random.default_rng(pos0)
    kind = np.float16 if half else np.float32
    k, v = (rng.standard_normal((KVH, ctx, dh)).astype(kind) for _ in range(2))
    k[:, pos0 + T:], v[:, pos0 + T:] = np.nan, np.nan
    q = (rng.standard_normal((T, H * dh)) * 2).astype(np.float32)
    kd, vd, qd = (t.from_numpy(a).cuda() for a in (k, v, q))
    need = cuda.tm_cuda_attn_window_scratch(T, H, KVH, dh)
    scratch, out = t.full((need // 4 + 1,), float("nan"), device="cuda"), t.full((T + 1, H * dh), 7.0, device="cuda")
    lib.check(cuda.tm_cuda_attn_window_dev(ptr(qd), ptr(kd), ptr(vd), ptr(scratch), need, ptr(out), T, pos0, H, KVH, dh, ctx, window, sinks,
                                           1 / np.sqrt(dh), int(half), stream_ptr(t)), "attn_window")
    t.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.all(got[T] == 7.0)
    want, tol = reference(q.reshape(T, H, dh), k[:, :pos0 + T].transpose(1, 0, 2), v[:, :pos0 + T].transpose(1, 0, 2), pos0, window, sinks, 1 / np.sqrt(dh))
    off = np.abs(got[:T].reshape(T, H, dh) - want)
    assert np.all(off <= tol), float((off / tol).max())


# ---- append --------------------------------------------------------------------------------------------------------------

def append(cuda, b, rope, qkv, want_ok=True):
    t = b.torch
    q = t.full((b.T, b.H * b.dh), 7.0, device="cuda")
    dq = t.from_numpy(qkv).cuda()
    dr = t.from_numpy(rope).cuda() if rope is not None else None
    lib.check(cuda.tm_cuda_kv_append_paged_dev(C.byref(b.desc), ptr(dq), ptr(q), b.T, b.H, ptr(dr) if rope is not None else None,
                                               len(rope) if rope is not None else 0, stream_ptr(t)), "append")
    t.cuda.synchronize()
    assert cuda.tm_cuda_tok_flush() == want_ok
    return q.cpu().numpy(), b.d["k"].cpu().numpy(), b.d["v"].cpu().numpy()


def rope_table(n, dh, theta=10000.0):
    a = np.arange(n)[:, None] * theta ** (-2.0 * np.arange(dh // 2) / dh)
    return np.ascontiguousarray(np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32))


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("H,KVH,dh,page,turned", [(8, 2, 128, 16, True), (4, 4, 64, 1, True), (6, 2, 80, 24, True), (5, 5, 8, 64, True), (8, 2, 64, 7, False)])
def test_append(cuda, torch_mod, H, KVH, dh, page, turned, half):
    new, total = [1, 70, 0, 3, 5], [100, 70, 9, 3, 4]                      # the last one: a token before position 0
    b = Batch(torch_mod, new, total, H, KVH, dh, page, half, seed=dh, extra_rows=2)
    rng = np.random.default_rng(1)
    qkv = rng.standard_normal((b.T, (H + 2 * KVH) * dh)).astype(np.float32)
    rope = rope_table(100, dh) if turned else None
    q, k, v = append(cuda, b, rope, qkv)
    wk, wv, wq = b.k.copy(), b.v.copy(), np.full((b.T, H, dh), 7.0)
    touched = np.zeros(b.k.shape, bool)
    tol = np.zeros((b.T, H, dh))
    ktol = np.zeros(b.k.shape)
    half_step = 2.0 ** -11 if half else 0.0
    for s in range(b.B):
        for i in range(new[s]):
            p, t = total[s] - new[s] + i, b.begin[s] + i
            if p < 0:
                continue
            x = qkv[t].reshape(-1, dh).astype(np.float64)
            y, size = x.copy(), np.abs(x)
            if turned:
                c, sn = rope[p, :, 0].astype(np.float64), rope[p, :, 1].astype(np.float64)
                lo, hi = x[:, :dh // 2], x[:, dh // 2:]
                y = np.concatenate((lo * c - hi * sn, lo * sn + hi * c), 1)
                size = np.concatenate((np.abs(lo * c) + np.abs(hi * sn), np.abs(lo * sn) + np.abs(hi * c)), 1)
            wq[t], tol[t] = y[:H], 2 * U * size[:H]                        # a product's rounding and the sum's
            pg, r = b.table[s, p // page], p % page
            touched[pg, :, r] = True
            wk[pg, :, r], wv[pg, :, r] = y[H:H + KVH], x[H + KVH:].astype(b.v.dtype)
            ktol[pg, :, r] = 2 * U * size[H:H + KVH] + half_step * (np.abs(y[H:H + KVH]) * (1 + 2 * U)) * 2 + 2.0 ** -24 * half
    assert np.all(np.abs(q.reshape(wq.shape) - wq) <= tol)
    assert np.array_equal(v, wv, equal_nan=True)
    assert np.array_equal(k[~touched], b.k[~touched], equal_nan=True)
    assert np.all(np.abs(k[touched].astype(np.float64) - wk[touched]) <= ktol[touched])


def test_append_checks_its_arrays(cuda, torch_mod):
    H, KVH, dh, page = 4, 2, 64, 16
    qkv = np.ones((4, (H + 2 * KVH) * dh), np.float32)
    for spoil in ("page", "length", "range", "rope"):
        b = Batch(torch_mod, [1, 2, 1], [40, 50, 20], H, KVH, dh, page, True, seed=3)
        rope = rope_table(49 if spoil == "rope" else 64, dh)
        if spoil == "page":
            b.table[1, 3] = b.npages                                       # positions 48 and 49
        if spoil == "length":
            b.total = [40, b.ld * page + 1, 20]
        if spoil == "range":
            b.begin = np.array([0, 1, -1, 4], np.int32)
        b.upload()
        q, k, v = append(cuda, b, rope, qkv, want_ok=False)
        changed = ~((v == b.v) | (np.isnan(v) & np.isnan(b.v)))
        allowed = np.zeros_like(changed)
        for s, p in ((0, 39), (2, 19)) + (((1, 48),) if spoil == "rope" else ()):
            if spoil == "range" and s == 2:
                continue
            allowed[b.table[s, p // page], :, p % page] = True
        assert not (changed & ~allowed).any(), spoil
        assert changed[b.table[0, 2], :, 7].any() or spoil == "range"


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("spoil", ["page", "length", "range", "rope"])
def test_tokens_without_a_position_leave_nan(cuda, torch_mod, spoil, half):
    """A token whose length or angles are out of range: its row of q is NaN and the attention that follows is NaN there, not what the buffers held;
    the other rows are as without it."""
    H, KVH, dh, page = 4, 2, 64, 16
    make = lambda: Batch(torch_mod, [1, 3, 1], [40, 50, 20], H, KVH, dh, page, half, seed=3, extra_rows=2)  # noqa: E731
    qkv = np.random.default_rng(2).standard_normal((7, (H + 2 * KVH) * dh)).astype(np.float32)
    good = make()
    want, want_k, want_v = append(cuda, good, rope_table(64, dh), qkv)
    good.d["q"].copy_(torch_mod.from_numpy(want))
    right = good.attend(cuda)
    b, lost, nan, stored = make(), [], [], {0, 1, 2, 3, 4}
    if spoil == "page":
        b.table[1, 3] = b.npages                                           # positions 48 and 49: their queries are known, their rows are not
        stored -= {2, 3}
    elif spoil == "length":
        b.total = [40, b.ld * page + 1, 20]
        nan = [1, 2, 3]
    elif spoil == "range":
        b.begin = np.array([0, 1, 8, 5], np.int32)                         # the second sequence's end, the third one's begin
        lost = [1, 2, 3, 4]
    else:
        nan = [2, 3]                                                       # the table ends behind position 47
    stored -= set(nan) | set(lost)
    b.upload()
    q, k, v = append(cuda, b, rope_table(48 if spoil == "rope" else 64, dh), qkv, want_ok=False)
    for t in range(7):
        if t in nan:
            assert np.isnan(q[t]).all(), t
        elif t in lost or t > 4:
            assert np.all(q[t] == 7.0), t
        else:
            assert np.array_equal(q[t], want[t]), t
    for t, (s, p) in enumerate([(0, 39), (1, 47), (1, 48), (1, 49), (2, 19)]):
        at = good.table[s, p // page], slice(None), p % page
        for mine, new, old in ((k, want_k, b.k), (v, want_v, b.v)):
            assert np.array_equal(mine[at], (new if t in stored else old)[at]), t
    b.d["q"].copy_(torch_mod.from_numpy(q))
    got = b.attend(cuda, want_ok=spoil == "rope")
    for t in range(5):
        if t in nan or (spoil == "page" and t in (2, 3)):
            assert np.isnan(got[t]).all(), t
        elif t in lost:
            assert np.all(got[t] == 7.0), t
        elif t in (0, 4):
            assert np.array_equal(got[t], right[t]), t
    if spoil == "rope":                                                    # beside rows that are NaN a row is computed key by key
        b.k, b.v = k, v
        kk, vv = b.rows(1)
        ref, tol = reference(q[1].reshape(1, H, dh), kk[:48], vv[:48], 47, 0, 0, 1 / np.sqrt(dh))
        assert np.all(np.abs(got[1].reshape(1, H, dh) - ref) <= tol)


def test_append_then_attend_captured(cuda, torch_mod):
    """A graph of append and attention, captured once, replayed for token after token with lengths that grow on the device."""
    t = torch_mod
    H, KVH, dh, page, steps = 8, 2, 64, 16, 20
    start = [30, 1, 47]
    b = Batch(t, [1, 1, 1], [s + steps for s in start], H, KVH, dh, page, True, seed=8)
    rng = np.random.default_rng(5)
    qkv = rng.standard_normal((steps, 3, (H + 2 * KVH) * dh)).astype(np.float32)
    rope = rope_table(128, dh)
    dr, dqkv, src = t.from_numpy(rope).cuda(), t.zeros(3, (H + 2 * KVH) * dh, device="cuda"), t.from_numpy(qkv).cuda()
    q, out = t.zeros(3, H * dh, device="cuda"), t.zeros(3, H * dh, device="cuda")
    need = cuda.tm_cuda_attn_paged_scratch(3, 3, 1, H, KVH, dh)
    scratch = t.empty(need // 4 + 1, device="cuda")
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())

    def step(s):
        lib.check(cuda.tm_cuda_kv_append_paged_dev(C.byref(b.desc), ptr(dqkv), ptr(q), 3, H, ptr(dr), 128, s), "append")
        lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(b.desc), ptr(q), ptr(scratch), need, ptr(out), 3, 1, H, 25, 2, 0.125, s), "attend")

    with t.cuda.stream(side):
        b.d["kv_len"].copy_(t.tensor(start, dtype=t.int32))
        step(stream_ptr(t))
    side.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        step(stream_ptr(t))
    for i in range(steps):
        dqkv.copy_(src[i])
        b.d["kv_len"].copy_(t.tensor([s + i + 1 for s in start], dtype=t.int32))
        graph.replay()
        t.cuda.synchronize()
        b.k, b.v = b.d["k"].cpu().numpy(), b.d["v"].cpu().numpy()
        b.total = [s + i + 1 for s in start]
        got, qs = out.cpu().numpy(), q.cpu().numpy()
        for s in range(3):
            want, tol = reference(qs[s].reshape(1, H, dh), *b.rows(s), b.total[s] - 1, 25, 2, 0.125)
            assert np.all(np.abs(got[s].reshape(1, H, dh) - want) <= tol)


@pytest.mark.parametrize("half", [True, False])
def test_serving_loop(cuda, torch_mod, half):
    """Prompts in one chunk, then token by token: append, attention, logits, rules, choice, against the same in 64 bits on the tokens
    that the GPU chose. The choice is checked where the two largest logits are further apart than the logits' tolerance."""
    t, rng = torch_mod, np.random.default_rng(4)
    H, KVH, dh, page, V, steps = 4, 2, 64, 16, 600, 12
    W = (H + 2 * KVH) * dh
    table_e = rng.standard_normal((V, W)).astype(np.float32)
    head = (rng.standard_normal((H * dh, V)) / 16).astype(np.float32)
    prompts = [rng.integers(0, V, n).tolist() for n in (37, 1, 90)]
    B, cap = 3, 128
    npages, ld = B * cap // page, cap // page
    table = rng.permutation(npages).astype(np.int32).reshape(B, ld)
    kind = t.float16 if half else t.float32
    d = {"k": t.zeros(npages, KVH, page, dh, dtype=kind, device="cuda"), "v": t.zeros(npages, KVH, page, dh, dtype=kind, device="cuda"),
         "table": t.from_numpy(table).cuda(), "q_begin": t.zeros(B + 1, dtype=t.int32, device="cuda"), "kv_len": t.zeros(B, dtype=t.int32, device="cuda")}
    desc = lib.KvPages(B=B, KVH=KVH, dh=dh, page=page, npages=npages, table_ld=ld, kv_half=int(half), **{n: x.data_ptr() for n, x in d.items()})
    rope = rope_table(cap, dh)
    dr, dw, de = (t.from_numpy(x).cuda() for x in (rope, head, table_e))
    lists = t.full((B, cap), -1, dtype=t.int32, device="cuda")
    counts, prompt_n = t.zeros(B, dtype=t.int32, device="cuda"), t.tensor([len(p) for p in prompts], dtype=t.int32, device="cuda")
    rep, pres, freq = (t.tensor(x, dtype=t.float32, device="cuda") for x in ([1.2, 1.5, 1.0], [0.1, 0.0, 0.3], [0.05, 0.2, 0.0]))
    mask = rng.integers(0, 2 ** 32, (B, (V + 31) // 32), dtype=np.uint32)
    dm = t.from_numpy(mask.view(np.int32)).cuda()
    rules = lib.LogitRules(tokens=lists.data_ptr(), n_tokens=counts.data_ptr(), n_prompt=prompt_n.data_ptr(), tokens_ld=cap, repeat=rep.data_ptr(),
                           presence=pres.data_ptr(), frequency=freq.data_ptr(), mask=dm.data_ptr(), mask_ld=mask.shape[1])
    seqs, new = [list(p) for p in prompts], [list(p) for p in prompts]
    bits = (mask[:, :, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(B, -1)[:, :V].astype(bool)
    sure = 0
    for step in range(steps):
        begin = np.concatenate([[0], np.cumsum([len(n) for n in new])]).astype(np.int32)
        T, max_q = int(begin[-1]), max(len(n) for n in new)
        d["q_begin"].copy_(t.from_numpy(begin)); d["kv_len"].copy_(t.tensor([len(s) for s in seqs], dtype=t.int32))
        for b in range(B):
            lists[b, :len(seqs[b])] = t.tensor(seqs[b], dtype=t.int32)
        counts.copy_(d["kv_len"])
        qkv = de[t.tensor(sum(new, []), device="cuda")].contiguous()
        q, out = t.empty(T, H * dh, device="cuda"), t.empty(T, H * dh, device="cuda")
        need = cuda.tm_cuda_attn_paged_scratch(T, B, max_q, H, KVH, dh)
        scratch = t.empty(need // 4 + 1, device="cuda")
        lib.check(cuda.tm_cuda_kv_append_paged_dev(C.byref(desc), ptr(qkv), ptr(q), T, H, ptr(dr), cap, stream_ptr(t)), "append")
        lib.check(cuda.tm_cuda_attn_paged_dev(C.byref(desc), ptr(q), ptr(scratch), need, ptr(out), T, max_q, H, 48, 2, 0.125, stream_ptr(t)), "attention")
        logits = (out[t.from_numpy(begin[1:] - 1).long().cuda()].double() @ dw.double()).float()
        ruled, token = t.empty_like(logits), t.zeros(B, dtype=t.int32, device="cuda")
        lib.check(cuda.tm_cuda_logits_rules_dev(ptr(logits), V, ptr(ruled), V, B, V, C.byref(rules), stream_ptr(t)), "rules")
        for b in range(B):
            lib.check(cuda.tm_cuda_argmax_dev(ptr(ruled[b]), ptr(token[b:]), V, stream_ptr(t)), "argmax")
        t.cuda.synchronize()
        assert cuda.tm_cuda_tok_flush()
        got, chosen = ruled.cpu().numpy(), token.cpu().tolist()
        for b in range(B):
            x = table_e[seqs[b]].astype(np.float64).reshape(-1, H + 2 * KVH, dh)
            c, sn = rope[:len(x), None, :, 0].astype(np.float64), rope[:len(x), None, :, 1].astype(np.float64)
            lo, hi = x[:, :H + KVH, :dh // 2], x[:, :H + KVH, dh // 2:]
            y = np.concatenate((lo * c - hi * sn, lo * sn + hi * c), 2)
            kk, vv = y[:, H:], x[:, H + KVH:]
            want, tol = reference(y[-1:, :H], kk, vv, len(x) - 1, 48, 2, 0.125)
            # the caches' rounding: a key's half step moves a score by at most A 2^-11, a value's the result by size 2^-11; both through softmax
            if half:
                A = max(np.abs(kk[:, h // 2] @ y[-1, h]).max() + np.linalg.norm(y[-1, h]) * np.linalg.norm(kk[:, h // 2], axis=1).max() for h in range(H)) * 0.125
                tol = tol + (2 * A + 1) * 2.0 ** -11 * np.abs(vv).max()
            z = want.reshape(-1) @ head
            ztol = tol.reshape(-1) @ np.abs(head) + np.abs(want.reshape(-1)) @ np.abs(head) * 2.0 ** -22
            n, first = len(seqs[b]), len(prompts[b])
            r, p, f = float(rep[b]), float(pres[b]), float(freq[b])
            for tok in set(seqs[b]):
                made = seqs[b][first:].count(tok)
                z[tok] = (z[tok] / r if z[tok] > 0 else z[tok] * r) - f * made - p * (made > 0)
                ztol[tok] *= max(1.0, r)
            ztol = ztol + (np.abs(z) + 4) * 2.0 ** -22
            assert np.isneginf(got[b][~bits[b]]).all()
            assert np.all(np.abs(got[b] - z)[bits[b]] <= ztol[bits[b]]), (step, b)
            z[~bits[b]] = -np.inf
            best = int(np.argmax(z))
            second = np.max(np.delete(z, best))
            if z[best] - second > 2 * ztol.max():
                assert chosen[b] == best
                sure += 1
            assert bits[b][chosen[b]]
        new = [[c] for c in chosen]
        seqs = [s + n for s, n in zip(seqs, new)]
    assert half or sure > 25
