"""The operators of a serving step over a batch of sequences, as measurable cases.

  append   rope of the new tokens' queries and keys, keys and values into the pages of the cache
  paged    attention of each sequence's new tokens (one or many) over its pages
  window   attention of a chunk of tokens over one contiguous cache, with a sliding window and first tokens that stay visible
  rules    penalties for repeated tokens, biases and grammar masks on a batch of logits

`run` computes the plain form in elementary torch operations; with `own` set it makes the C ABI calls of
include/cuda_shim.h through tensormark_b200.lib.
"""
from __future__ import annotations

import ctypes as C
import math
import random

import torch

own = False

# Two model geometries: 32 / 8 heads of 128 (8B shapes) and 32 / 4 heads of 64 (a small model).


def listed():
    return [
        # one decode step of 48 conversations: a token each, the smallest append there is in a serving loop
        {"name": "append_f16_48x1_8b", "op": "append", "heads": 32, "kv_heads": 8, "dh": 128, "page": 16, "half": True,
         "batch": 48, "q_min": 1, "q_max": 1, "old_min": 20, "old_max": 900, "lens": 1},
        # the prompts of five requests on the fp32 cache of a small model, odd lengths, odd page size
        {"name": "append_f32_5x400_small", "op": "append", "heads": 32, "kv_heads": 4, "dh": 64, "page": 24, "half": False,
         "batch": 5, "q_min": 150, "q_max": 700, "old_min": 0, "old_max": 333, "lens": 2},
        # a single conversation's decode step: latency
        {"name": "paged_f16_1x1_600", "op": "paged", "heads": 32, "kv_heads": 8, "dh": 128, "page": 16, "half": True,
         "batch": 1, "q_min": 1, "q_max": 1, "old_min": 600, "old_max": 600, "window": 0, "sinks": 0, "lens": 3},
        # a full decode batch, conversations of very different lengths: streaming
        {"name": "paged_f16_64x1_ragged", "op": "paged", "heads": 32, "kv_heads": 8, "dh": 128, "page": 16, "half": True,
         "batch": 64, "q_min": 1, "q_max": 1, "old_min": 150, "old_max": 8100, "window": 0, "sinks": 0, "lens": 4},
        # a continuous batch: one prompt's chunk next to decoding sequences, a windowed model with sinks
        {"name": "paged_f16_mixed_window", "op": "paged", "heads": 32, "kv_heads": 4, "dh": 64, "page": 32, "half": True,
         "batch": 17, "q_min": 1, "q_max": 1, "q_first": 512, "old_min": 40, "old_max": 3500, "window": 1000, "sinks": 4, "lens": 5},
        # long documents read in chunks: the largest contraction
        {"name": "paged_f16_2x1024_15k", "op": "paged", "heads": 32, "kv_heads": 8, "dh": 128, "page": 64, "half": True,
         "batch": 2, "q_min": 1000, "q_max": 1024, "old_min": 14000, "old_max": 15000, "window": 0, "sinks": 0, "lens": 6},
        # decode far into a long stream
        {"name": "window_f16_1_at_32k", "op": "window", "heads": 32, "kv_heads": 8, "dh": 128, "half": True,
         "tokens": 1, "pos0": 32700, "ctx": 32768, "window": 4096, "sinks": 4},
        # a chunk of a stream
        {"name": "window_f16_1000_at_7k", "op": "window", "heads": 32, "kv_heads": 8, "dh": 128, "half": True,
         "tokens": 1000, "pos0": 7001, "ctx": 8192, "window": 1024, "sinks": 4},
        # a prompt on the fp32 cache of a small model
        {"name": "window_f32_700_small", "op": "window", "heads": 32, "kv_heads": 4, "dh": 64, "half": False,
         "tokens": 700, "pos0": 0, "ctx": 1024, "window": 255, "sinks": 1},
        # one conversation's sampling step, small vocabulary
        {"name": "rules_1x32000", "op": "rules", "batch": 1, "vocab": 32000, "history": 300, "biases": 8, "mask": True},
        # a full batch under grammars, large vocabulary, long histories: streaming
        {"name": "rules_64x128256", "op": "rules", "batch": 64, "vocab": 128256, "history": 2500, "biases": 64, "mask": True},
        # a small batch without grammars, a vocabulary that is no multiple of anything
        {"name": "rules_7x50257", "op": "rules", "batch": 7, "vocab": 50257, "history": 901, "biases": 0, "mask": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "window", "window", "rules"])
    if op == "rules":
        batch = _log_int(rng, 1, 64)
        return {"op": "rules", "batch": batch, "vocab": _log_int(rng, 20000, 128256), "history": _log_int(rng, 1, 2500),
                "biases": rng.choice([0, 1, 13, 64]), "mask": rng.random() < 0.7}
    dh = rng.choice([64, 128, 128, 128, 80])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    half = rng.random() < 0.75
    base = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dh": dh, "half": half}
    window = rng.choice([0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 70]) if window else 0
    if op == "append":
        return {**base, "page": rng.choice([1, 16, 24, 64, 128]), "batch": _log_int(rng, 1, 48), "q_min": 1,
                "q_max": _log_int(rng, 1, 60), "old_min": 0, "old_max": _log_int(rng, 1, 900), "lens": rng.randrange(1 << 20)}
    if op == "window":
        tokens = rng.choice([1, _log_int(rng, 1, 2000)])
        pos0 = _log_int(rng, 1, 30000 if tokens * kv_heads * group < 1000 else 5000) - 1
        return {**base, "tokens": tokens, "pos0": pos0, "ctx": pos0 + tokens + rng.randrange(0, 200), "window": window, "sinks": sinks}
    q_max = rng.choice([1, 1, 4, _log_int(rng, 2, 1000)])
    batch = _log_int(rng, 1, 64 if q_max <= 4 else 4)
    old = _log_int(rng, 2, 8000 if q_max <= 64 else 4000)
    return {**base, "page": rng.choice([1, 16, 16, 24, 64, 256]), "batch": batch, "q_min": 1, "q_max": q_max, "old_min": rng.randrange(0, old),
            "old_max": old, "window": window, "sinks": sinks, "lens": rng.randrange(1 << 20)}


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence"""
    r = random.Random(case["lens"])
    new = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["batch"])]
    if "q_first" in case:
        new[0] = case["q_first"]
    return new, [n + r.randint(case["old_min"], case["old_max"]) for n in new]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op = case["op"]
    if op == "rules":
        B, V, n = case["batch"], case["vocab"], case["history"]
        lengths = torch.randint(0, n + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = n
        # text repeats itself: tokens come from a small part of the vocabulary that differs from row to row
        tokens = (torch.randint(0, V, (B, 1), generator=g, device="cuda") + (normal(B, n) * 200).long() ** 2 // 64) % V
        st = {"x": normal(B, V) * 3, "tokens": tokens.int(), "n_tokens": lengths, "n_prompt": lengths // 3,
              "repeat": 1 + 0.3 * torch.rand(B, generator=g, device="cuda"), "presence": torch.rand(B, generator=g, device="cuda"),
              "frequency": 0.5 * torch.rand(B, generator=g, device="cuda"), "bias_ids": None, "mask": None}
        if k := case["biases"]:
            st["bias_ids"] = torch.rand(B, V, generator=g, device="cuda").topk(k, dim=1).indices.int()
            st["bias"] = normal(B, k) * 5
            st["n_bias"] = torch.randint(0, k + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        if case["mask"]:  # the tokens that a grammar's state lets through: few in some rows, nearly all in others
            words = (V + 31) // 32
            dense = torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g, device="cuda")
            sparse = dense & dense.roll(1, 1) & dense.roll(2, 1) & dense.roll(3, 1)
            st["mask"] = torch.where(torch.rand(B, 1, generator=g, device="cuda") < 0.5, sparse, ~sparse).int()
        return {"case": case, **st}
    H, KVH, dh = case["heads"], case["kv_heads"], case["dh"]
    kind = torch.float16 if case["half"] else torch.float32
    if op == "window":
        T, ctx = case["tokens"], case["ctx"]
        return {"case": case, "q": normal(T, H * dh) * 1.5, "k": normal(KVH, ctx, dh).to(kind), "v": normal(KVH, ctx, dh).to(kind)}
    new, total = _lengths(case)
    B, page = case["batch"], case["page"]
    need = [-(-n // page) for n in total]
    npages, width = sum(need) + 3, max(need) + 1
    order = torch.randperm(npages, generator=g, device="cuda").int()  # pages are handed out in any order
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    begin = [0]
    for n in new:
        begin.append(begin[-1] + n)
    T = begin[-1]
    st = {"case": case, "table": table, "q_begin": torch.tensor(begin, dtype=torch.int32, device="cuda"),
          "kv_len": torch.tensor(total, dtype=torch.int32, device="cuda"), "T": T, "max_q": max(new), "max_kv": max(total),
          "k": normal(npages, KVH, page, dh).to(kind), "v": normal(npages, KVH, page, dh).to(kind)}
    # the scheduler's own view of the batch: which sequence and which position each new token is
    st["seq"] = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
    st["pos"] = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(new, total)])
    if op == "append":
        st["qkv"] = normal(T, (H + 2 * KVH) * dh)
        inv = 500000.0 ** (-2.0 * torch.arange(dh // 2, device="cuda", dtype=torch.float64) / dh)
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * inv
        st["rope"] = torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()
    else:
        st["q"] = normal(T, H * dh) * 1.5
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _plain_append(s):
    c = s["case"]
    H, KVH, dh, T, page = c["heads"], c["kv_heads"], c["dh"], s["T"], c["page"]
    rows = s["qkv"].view(T, H + 2 * KVH, dh)
    cos, sin = s["rope"][s["pos"]].unbind(-1)
    a, b = rows[:, :H + KVH, :dh // 2], rows[:, :H + KVH, dh // 2:]
    cos, sin = cos[:, None], sin[:, None]
    turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    at = s["table"][s["seq"], s["pos"] // page].long()
    s["k"][at, :, s["pos"] % page] = turned[:, H:].to(s["k"].dtype)
    s["v"][at, :, s["pos"] % page] = rows[:, H + KVH:].to(s["v"].dtype)
    return {"q": turned[:, :H].reshape(T, H * dh), "k": s["k"], "v": s["v"]}


def _plain_attention(q, k, v, pos, length, c):
    """q [B, Q, H, dh], k and v [B, L, KVH, dh], pos [B, Q] (negative: no token), length [B]"""
    B, Q, H, dh = q.shape
    L, KVH = k.shape[1], k.shape[2]
    q = q.view(B, Q, KVH, H // KVH, dh).permute(0, 2, 3, 1, 4).reshape(B, KVH, -1, dh)
    score = q @ k.float().permute(0, 2, 3, 1) * (1 / math.sqrt(dh))
    key, p = torch.arange(L, device=q.device), pos[:, :, None]
    seen = (key <= p) & (key < length[:, None, None])
    if c["window"]:
        seen &= (key > p - c["window"]) | (key < c["sinks"])
    seen = seen[:, None, None]
    score = score.view(B, KVH, H // KVH, Q, L).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min_(-3e38)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    v = v.float().masked_fill(key[None, :, None, None] >= length[:, None, None, None], 0.0).permute(0, 2, 1, 3)
    out = weight.view(B, KVH, -1, L) @ v
    out = out.view(B, KVH, H // KVH, Q, dh) / total.clamp_min(1e-38)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Q, H * dh)


def _plain_paged(s):
    c = s["case"]
    H, KVH, dh, B, page = c["heads"], c["kv_heads"], c["dh"], c["batch"], c["page"]
    q = s["q"].new_zeros(B, s["max_q"], H, dh)
    pos = torch.full((B, s["max_q"]), -1, device="cuda")
    row = torch.arange(s["T"], device="cuda") - s["q_begin"].long()[s["seq"]]
    q[s["seq"], row] = s["q"].view(-1, H, dh)
    pos[s["seq"], row] = s["pos"]
    pages = s["table"].long().clamp_min(0)[:, :-(-s["max_kv"] // page)]
    k, v = (s[n][pages].permute(0, 1, 3, 2, 4).reshape(B, -1, KVH, dh) for n in ("k", "v"))
    return _plain_attention(q, k, v, pos, s["kv_len"].long(), c)[s["seq"], row]


def _plain_window(s):
    c = s["case"]
    T, end = c["tokens"], c["pos0"] + c["tokens"]
    k, v = (s[n][:, :end].transpose(0, 1)[None] for n in ("k", "v"))
    pos = torch.arange(c["pos0"], end, device="cuda")[None]
    return _plain_attention(s["q"].view(1, T, c["heads"], c["dh"]), k, v, pos, torch.tensor([end], device="cuda"), c)[0]


def _plain_rules(s):
    x, V = s["x"], s["case"]["vocab"]
    index = torch.arange(s["tokens"].shape[1], device="cuda")
    ids, there = s["tokens"].long(), index < s["n_tokens"][:, None]
    zero = torch.zeros_like(x)
    seen = zero.scatter_add(1, ids, there.float()) > 0
    count = zero.scatter_add(1, ids, (there & (index >= s["n_prompt"][:, None])).float())
    repeat = s["repeat"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / repeat, x * repeat), x)
    x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_ids"] is not None:
        there = torch.arange(s["bias"].shape[1], device="cuda") < s["n_bias"][:, None]
        x = x + zero.scatter_add(1, s["bias_ids"].long(), torch.where(there, s["bias"], 0.0))
    if s["mask"] is not None:
        token = torch.arange(V, device="cuda")
        x = torch.where((s["mask"][:, token // 32] >> (token % 32)) & 1 != 0, x, -math.inf)
    return x


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _address(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


def _own_setup(s):
    """What a program keeps from call to call: the cache's description, the output, the workspace."""
    from tensormark_b200 import lib
    L, c = lib.load(), s["case"]
    if not L.tm_cuda_init(-1):
        raise RuntimeError(lib.last_error())
    op = c["op"]
    if op == "rules":
        out = torch.empty_like(s["x"])
        words = s["mask"].shape[1] if s["mask"] is not None else 0
        some = s["bias_ids"] is not None
        rules = lib.LogitRules(
            tokens=s["tokens"].data_ptr(), n_tokens=s["n_tokens"].data_ptr(), n_prompt=s["n_prompt"].data_ptr(), tokens_ld=s["tokens"].shape[1],
            repeat=s["repeat"].data_ptr(), presence=s["presence"].data_ptr(), frequency=s["frequency"].data_ptr(),
            bias_ids=s["bias_ids"].data_ptr() if some else None, bias=s["bias"].data_ptr() if some else None,
            n_bias=s["n_bias"].data_ptr() if some else None, bias_ld=s["bias"].shape[1] if some else 0,
            mask=s["mask"].data_ptr() if words else None, mask_ld=words)
        return L.tm_cuda_logits_rules_dev, (_address(s["x"]), c["vocab"], _address(out), c["vocab"], c["batch"], c["vocab"], C.byref(rules)), out, rules
    H, KVH, dh, half = c["heads"], c["kv_heads"], c["dh"], int(c["half"])
    scale = C.c_float(1 / math.sqrt(dh))
    if op == "window":
        out = torch.empty_like(s["q"])
        need = L.tm_cuda_attn_window_scratch(c["tokens"], H, KVH, dh)
        scratch = torch.empty(need // 4 + 1, dtype=torch.float32, device="cuda")
        return L.tm_cuda_attn_window_dev, (_address(s["q"]), _address(s["k"]), _address(s["v"]), _address(scratch), need, _address(out), c["tokens"],
                                           c["pos0"], H, KVH, dh, c["ctx"], c["window"], c["sinks"], scale, half), out, scratch
    pages = lib.KvPages(k=s["k"].data_ptr(), v=s["v"].data_ptr(), table=s["table"].data_ptr(), q_begin=s["q_begin"].data_ptr(),
                        kv_len=s["kv_len"].data_ptr(), B=c["batch"], KVH=KVH, dh=dh, page=c["page"], npages=s["k"].shape[0],
                        table_ld=s["table"].shape[1], kv_half=half)
    if op == "append":
        q = torch.empty(s["T"], H * dh, device="cuda")
        return L.tm_cuda_kv_append_paged_dev, (C.byref(pages), _address(s["qkv"]), _address(q), s["T"], H, _address(s["rope"]), s["rope"].shape[0]), \
            {"q": q, "k": s["k"], "v": s["v"]}, pages
    out = torch.empty_like(s["q"])
    need = L.tm_cuda_attn_paged_scratch(s["T"], c["batch"], s["max_q"], H, KVH, dh)
    scratch = torch.empty(need // 4 + 1, dtype=torch.float32, device="cuda")
    return L.tm_cuda_attn_paged_dev, (C.byref(pages), _address(s["q"]), _address(scratch), need, _address(out), s["T"], s["max_q"], H,
                                      c["window"], c["sinks"], scale), out, (pages, scratch)


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _own_setup(state)
        entry, args, out, _ = state["call"]
        if not entry(*args, torch.cuda.current_stream().cuda_stream):
            from tensormark_b200 import lib
            raise RuntimeError(lib.last_error())
        return out
    return {"append": _plain_append, "paged": _plain_paged, "window": _plain_window, "rules": _plain_rules}[state["case"]["op"]](state)


# ---- what the path cannot do without -----------------------------------------------------------------------------------

def _visible(p, c):
    """keys that position p sees"""
    w, s = c.get("window", 0), c.get("sinks", 0)
    return p + 1 if not w or w >= p + 1 else w + min(s, p + 1 - w)


def work(case):
    op = case["op"]
    if op == "rules":
        B, V = case["batch"], case["vocab"]
        return {"bytes": B * (8 * V + 4 * case["history"] + 8 * case["biases"] + (V // 8 if case["mask"] else 0)), "flops": 8 * B * V}
    H, KVH, dh = case["heads"], case["kv_heads"], case["dh"]
    elem = 2 if case["half"] else 4
    if op == "append":
        T = sum(_lengths(case)[0])
        return {"bytes": T * dh * (4 * (H + 2 * KVH) + 4 * H + 2 * elem * KVH), "flops": 3 * T * dh * (H + KVH)}
    spans = [(case["tokens"], case["pos0"] + case["tokens"])] if op == "window" else list(zip(*_lengths(case)))
    pairs = sum(_visible(p, case) for n, t in spans for p in range(t - n, t))
    # rows of the cache that at least one new token sees: its window and the sinks before it
    rows = sum(min(t, n - 1 + _visible(t - 1, case)) if case["window"] else t for n, t in spans)
    T = sum(n for n, _ in spans)
    return {"bytes": 2 * elem * KVH * dh * rows + 8 * T * H * dh, "flops": 4 * H * dh * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _exact_head(q, k, v, first, c):
    """One query head of one sequence: q [n, dh] at positions first.., k and v [first + n, dh], all in 64 bits."""
    n, L = q.shape[0], k.shape[0]
    i = torch.arange(first, first + n, device="cuda").view(n, 1)
    j = torch.arange(L, device="cuda").view(1, L)
    hidden = j > i
    if c["window"]:
        hidden |= (j + c["window"] <= i) & (j >= c["sinks"])
    s = (q @ k.T / math.sqrt(q.shape[1])).masked_fill(hidden, -math.inf)
    return torch.softmax(s, 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rules":
        rows = []
        for b in range(case["batch"]):
            n, first = int(s["n_tokens"][b]), int(s["n_prompt"][b])
            x = s["x"][b].double()
            said = s["tokens"][b, :n].long()
            past = torch.bincount(said, minlength=case["vocab"])
            made = torch.bincount(said[first:], minlength=case["vocab"])
            r, pres, freq = (s[k][b].double() for k in ("repeat", "presence", "frequency"))
            old = past > 0
            x[old] = torch.where(x[old] > 0, x[old] / r, x[old] * r)
            x -= made * freq
            x[made > 0] -= pres
            if s["bias_ids"] is not None:
                m = int(s["n_bias"][b])
                x[s["bias_ids"][b, :m].long()] += s["bias"][b, :m].double()
            if s["mask"] is not None:
                bits = (s["mask"][b][:, None] >> torch.arange(32, device="cuda")) & 1
                x[bits.flatten()[:case["vocab"]] == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    H, KVH, dh = case["heads"], case["kv_heads"], case["dh"]
    group = H // KVH
    if op == "window":
        end = case["pos0"] + case["tokens"]
        q = s["q"].double().view(-1, H, dh)
        heads = [_exact_head(q[:, h], s["k"][h // group, :end].double(), s["v"][h // group, :end].double(), case["pos0"], case) for h in range(H)]
        return torch.stack(heads, 1).reshape(-1, H * dh)
    new, total = _lengths(case)
    page = case["page"]
    where = [(s["table"][b, torch.arange(t, device="cuda") // page].long(), torch.arange(t, device="cuda") % page) for b, t in enumerate(total)]
    first = 0
    if op == "append":
        qkv = s["qkv"].double().view(-1, H + 2 * KVH, dh)
        k, v, qs = s["k"].double(), s["v"].double(), []
        for n, t, (pg, row) in zip(new, total, where):
            x = qkv[first:first + n]
            first += n
            z = torch.view_as_complex(s["rope"][t - n:t].double())[:, None]
            y = torch.complex(x[:, :H + KVH, :dh // 2], x[:, :H + KVH, dh // 2:]) * z
            y = torch.cat((y.real, y.imag), -1)
            qs.append(y[:, :H].reshape(n, H * dh))
            k[pg[t - n:], :, row[t - n:]] = y[:, H:]
            v[pg[t - n:], :, row[t - n:]] = x[:, H + KVH:]
        return {"q": torch.cat(qs), "k": k, "v": v}
    q, outs = s["q"].double().view(-1, H, dh), []
    for n, t, (pg, row) in zip(new, total, where):
        k, v = s["k"][pg, :, row].double(), s["v"][pg, :, row].double()
        heads = [_exact_head(q[first:first + n, h], k[:, h // group], v[:, h // group], t - n, case) for h in range(H)]
        outs.append(torch.stack(heads, 1).reshape(n, H * dh))
        first += n
    return torch.cat(outs)
