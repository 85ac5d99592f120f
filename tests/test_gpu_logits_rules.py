"""Rules on logits against a plain implementation in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tensormark_b200 import lib
from tests.gpu_util import ptr, stream_ptr

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def plain(x, V, tokens, n_tokens, n_prompt, repeat, presence, frequency, bias_ids, bias, n_bias, mask):
    y = x[:, :V].astype(np.float64)
    tol = np.zeros_like(y)
    for b in range(len(y)):
        if tokens is not None:
            n = min(max(int(n_tokens[b]), 0), tokens.shape[1])
            first = 0 if n_prompt is None else int(n_prompt[b])
            past, made = {}, {}
            for i, t in enumerate(tokens[b, :n].tolist()):
                if 0 <= t < V:
                    past[t] = 1
                    if i >= first:
                        made[t] = made.get(t, 0) + 1
            for t in past:
                r = float(repeat[b]) if repeat is not None else 1.0
                y[b, t] = y[b, t] / r if y[b, t] > 0 else y[b, t] * r
                tol[b, t] += abs(y[b, t]) * U
                if t in made:
                    take = (float(frequency[b]) if frequency is not None else 0.0) * made[t] + (float(presence[b]) if presence is not None else 0.0)
                    y[b, t] -= take
                    tol[b, t] += (abs(take) * 2 + abs(y[b, t])) * U
        if bias is not None:
            m = bias.shape[1] if n_bias is None else min(max(int(n_bias[b]), 0), bias.shape[1])
            for t, w in dict(zip(bias_ids[b, :m].tolist(), bias[b, :m].tolist())).items():
                if 0 <= t < V:
                    y[b, t] += w
                    tol[b, t] += (abs(y[b, t]) + tol[b, t]) * U
        if mask is not None:
            bits = (mask[b][:, None] >> np.arange(32, dtype=np.uint32)) & 1
            y[b, bits.reshape(-1)[:V] == 0] = -np.inf
    return y, tol * 1.01 + 2.0 ** -149                                       # and a step of fp32's smallest numbers


def case(rng, B, V, n, k, masked, ld):
    x = (rng.standard_normal((B, ld)) * 3).astype(np.float32)
    pool = rng.integers(0, V, max(1, n // 3))
    a = dict(tokens=rng.choice(pool, (B, n)).astype(np.int32) if n else None, n_tokens=rng.integers(0, n + 1, B).astype(np.int32) if n else None,
             n_prompt=rng.integers(0, n + 1, B).astype(np.int32) if n else None, repeat=(1 + rng.random(B)).astype(np.float32) if n else None,
             presence=rng.random(B).astype(np.float32) if n else None, frequency=rng.random(B).astype(np.float32) if n else None,
             bias_ids=rng.integers(0, V, (B, k)).astype(np.int32) if k else None, bias=rng.standard_normal((B, k)).astype(np.float32) if k else None,
             n_bias=rng.integers(0, k + 1, B).astype(np.int32) if k else None,
             mask=rng.integers(0, 2 ** 32, (B, (V + 31) // 32 + 1), dtype=np.uint32) if masked else None)
    return x, a


def run(cuda, t, x, V, a, ldo=None, in_place=False, shift=0):
    B, ld = x.shape
    ldo = ld if in_place else ldo or V
    flat = t.full((B * ld + shift,), 7.0, device="cuda")
    flat[shift:] = t.from_numpy(x.reshape(-1)).cuda()
    out = flat if in_place else t.full((B * ldo + shift,), 7.0, device="cuda")
    d = {n: t.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for n, v in a.items() if v is not None}
    width = lambda n: d[n].shape[1] if n in d else 0  # noqa: E731
    r = lib.LogitRules(tokens_ld=width("tokens"), bias_ld=width("bias"), mask_ld=width("mask"), **{n: v.data_ptr() for n, v in d.items()})
    lib.check(cuda.tm_cuda_logits_rules_dev(C.c_void_p(flat.data_ptr() + 4 * shift), ld, C.c_void_p(out.data_ptr() + 4 * shift), ldo, B, V, C.byref(r),
                                            stream_ptr(t)), "logits_rules")
    t.cuda.synchronize()
    got = out.cpu().numpy()[shift:].reshape(B, ldo)
    want, tol = plain(x, V, **a)
    mine = got[:, :V].astype(np.float64)
    assert np.array_equal(np.isnan(mine), np.isnan(want))
    same = ~np.isfinite(want)
    assert np.array_equal(mine[same], want[same], equal_nan=True)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(mine - want) <= tol) | same), float(np.nanmax(np.where(same, 0, np.abs(mine - want) - tol)))
    assert np.array_equal(got[:, V:], x[:, V:] if in_place else np.full((B, ldo - V), 7.0, np.float32))   # the strides' rest
    return got


@pytest.mark.parametrize("B,V,n,k,masked", [(1, 1, 1, 1, True), (1, 33, 5, 3, True), (3, 4096, 100, 0, False), (2, 4097, 0, 7, False), (5, 12289, 900, 64, True),
                                            (2, 32000, 300, 8, True), (1, 128256, 2500, 500, True), (4, 31, 200, 0, True), (70, 1000, 20, 2, True)])
def test_rules(cuda, torch_mod, B, V, n, k, masked):
    rng = np.random.default_rng(V)
    x, a = case(rng, B, V, n, k, masked, V)
    run(cuda, torch_mod, x, V, a)
    x, a = case(rng, B, V, n, k, masked, V + 5)
    run(cuda, torch_mod, x, V, a, ldo=V + 3)
    run(cuda, torch_mod, x, V, a, in_place=True)
    run(cuda, torch_mod, x, V, a, in_place=True, shift=3)


@pytest.mark.parametrize("V", list(range(1018, 1030)) + [4094, 4095, 8190, 8191])
def test_slices_that_end_anywhere(cuda, torch_mod, V):
    """Every alignment of rows against slices: last slices of one logit, and ones that the row does not reach."""
    rng = np.random.default_rng(V)
    for B in (1, 200 if V < 2000 else 160):
        for shift in (0, 1, 2, 3):
            x, a = case(rng, B, V, 40, 6, True, V + shift)
            a["tokens"][:, :4] = V - 1 - np.arange(4)
            a["bias_ids"][:, 0] = V - 1
            a["n_tokens"][:], a["n_bias"][:] = 40, 6
            run(cuda, torch_mod, x, V, a, in_place=True, shift=shift)


def test_each_rule_alone(cuda, torch_mod):
    rng = np.random.default_rng(0)
    x, a = case(rng, 3, 5000, 64, 9, True, 5000)
    for keep in (("repeat",), ("presence",), ("frequency",), ("bias",), ("mask",), ("repeat", "mask"), ()):
        b = dict(a)
        for n in ("repeat", "presence", "frequency", "mask"):
            if n not in keep:
                b[n] = None
        if "bias" not in keep:
            b["bias_ids"] = b["bias"] = b["n_bias"] = None
        if not set(keep) & {"repeat", "presence", "frequency"}:
            b["tokens"] = b["n_tokens"] = b["n_prompt"] = None
        run(cuda, torch_mod, x, 5000, b)
    a["n_prompt"] = a["n_bias"] = None
    run(cuda, torch_mod, x, 5000, a)


def test_ids_and_lengths_out_of_range(cuda, torch_mod):
    rng = np.random.default_rng(1)
    x, a = case(rng, 4, 9000, 50, 12, True, 9000)
    a["tokens"][:, ::3] = rng.choice([-1, 9000, 2 ** 31 - 1, -2 ** 31], a["tokens"][:, ::3].shape)
    a["bias_ids"][:, ::2] = rng.choice([-1, 9000, 2 ** 31 - 1, -2 ** 31], a["bias_ids"][:, ::2].shape)
    a["n_tokens"][:] = [-5, 51, 2 ** 31 - 1, 50]
    a["n_prompt"][:] = [-2 ** 31, 2 ** 31 - 1, 0, 25]
    a["n_bias"][:] = [2 ** 31 - 1, -7, 12, 13]
    run(cuda, torch_mod, x, 9000, a)


def test_same_id_twice_and_special_values(cuda, torch_mod):
    rng = np.random.default_rng(2)
    x, a = case(rng, 3, 300, 40, 30, True, 300)
    a["bias_ids"][:] = rng.integers(0, 6, a["bias_ids"].shape)              # of an id that is listed twice the last one counts
    a["n_bias"][:] = [30, 7, 1]
    x[:, :8] = [np.inf, -np.inf, np.nan, 0.0, -0.0, 1e38, -1e38, 1e-40]
    a["tokens"][:, :8] = np.arange(8)
    a["n_tokens"][:] = 40
    run(cuda, torch_mod, x, 300, a)
    a["mask"][:] = 0                                                       # a grammar that lets nothing through
    assert np.isneginf(run(cuda, torch_mod, x, 300, a)).all()


def test_rows_far_apart(cuda, torch_mod):
    """Strides whose products pass 32 bits."""
    t, rng = torch_mod, np.random.default_rng(9)
    V, ld = 5001, 1_500_000_003
    x, a = case(rng, 3, V, 30, 4, True, V)
    far = t.empty(2 * ld + V, dtype=t.float32, device="cuda")
    for b in range(3):
        far[b * ld:b * ld + V] = t.from_numpy(x[b]).cuda()
    d = {n: t.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for n, v in a.items()}
    r = lib.LogitRules(tokens_ld=30, bias_ld=4, mask_ld=a["mask"].shape[1], **{n: v.data_ptr() for n, v in d.items()})
    lib.check(cuda.tm_cuda_logits_rules_dev(ptr(far), ld, ptr(far), ld, 3, V, C.byref(r), stream_ptr(t)), "logits_rules")
    t.cuda.synchronize()
    want, tol = plain(x, V, **a)
    for b in range(3):
        got = far[b * ld:b * ld + V].cpu().numpy().astype(np.float64)
        same = ~np.isfinite(want[b])
        with np.errstate(invalid="ignore"):
            assert np.array_equal(got[same], want[b][same]) and np.all((np.abs(got - want[b]) <= tol[b]) | same)
    del far
    t.cuda.empty_cache()


@pytest.mark.parametrize("B,V,n_x,n_out,shift", [(3, 1000, 2000, 2000, 1000), (3, 1001, 2002, 2002, 1001), (2, 500, 1500, 500, 500), (1, 700, 700, 9000, 0), (4, 300, 300, 300, 1200)])
def test_rows_between_rows(cuda, torch_mod, B, V, n_x, n_out, shift):
    """out between the rows of x, behind them, or x itself with a stride that a single row does not use: taken, and right."""
    t, rng = torch_mod, np.random.default_rng(V)
    x, a = case(rng, B, V, 40, 6, True, V)
    d = {n: t.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for n, v in a.items()}
    r = lib.LogitRules(tokens_ld=40, bias_ld=6, mask_ld=a["mask"].shape[1], **{n: v.data_ptr() for n, v in d.items()})
    flat = t.full((max((B - 1) * n_x, shift + (B - 1) * n_out) + V,), 7.0, device="cuda")
    for b in range(B):
        flat[b * n_x:b * n_x + V] = t.from_numpy(x[b]).cuda()
    lib.check(cuda.tm_cuda_logits_rules_dev(ptr(flat), n_x, ptr(flat[shift:]), n_out, B, V, C.byref(r), stream_ptr(t)), "logits_rules")
    t.cuda.synchronize()
    got = flat.cpu().numpy()
    want, tol = plain(x, V, **a)
    for b in range(B):
        mine = got[shift + b * n_out:shift + b * n_out + V].astype(np.float64)
        same = ~np.isfinite(want[b])
        with np.errstate(invalid="ignore"):
            assert np.array_equal(mine[same], want[b][same]) and np.all((np.abs(mine - want[b]) <= tol[b]) | same)
        if shift:
            assert np.array_equal(got[b * n_x:b * n_x + V], x[b])


def test_a_step_to_the_token(cuda, torch_mod):
    """Rules, then the framework's choice: the token that the plain rules' largest logit has, lowest index on ties."""
    t, rng = torch_mod, np.random.default_rng(3)
    x, a = case(rng, 4, 32000, 200, 5, True, 32000)
    got = run(cuda, t, x, 32000, a)
    logits, token = t.from_numpy(got).cuda(), t.zeros(4, dtype=t.int32, device="cuda")
    for b in range(4):
        lib.check(cuda.tm_cuda_argmax_dev(ptr(logits[b]), ptr(token[b:]), 32000, stream_ptr(t)), "argmax")
    t.cuda.synchronize()
    assert token.cpu().tolist() == [int(np.argmax(row)) for row in got]
