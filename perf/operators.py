"""Cases, inputs and plain forms of the serving operators: page reservation, the writer of an 8-bit paged KV cache, the
attention that reads it, and token sampling.

``run`` computes an operator with elementary torch operations, or, where ``own`` is true, with this package's kernels.
Both forms take the same state and return the same outputs."""

from __future__ import annotations

import math
import random

import torch

own = False

_FLOATS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_MIN_SCALE, _MAX_SCALE = 2.0 ** -60, 2.0 ** 60


def _attention(name, requests, kv_heads, group, head_dim, page, dtype, cache, lens, q=(1, 1), long_share=0.0, window=0,
               layout="hnd", mix=1):
    return {"name": name, "op": "attention", "requests": requests, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "page": page, "dtype": dtype, "cache": cache, "len_lo": lens[0], "len_hi": lens[1],
            "q_lo": q[0], "q_hi": q[1], "long_share": long_share, "window": window, "layout": layout, "mix": mix}


def listed():
    return [
        # one decode step of a batch of 64: one slot each, a page for some
        {"name": "reserve_decode", "op": "reserve", "requests": 64, "page": 16, "max_pages": 512, "len_hi": 8100,
         "new_lo": 1, "new_hi": 1, "ended": 0.0, "mix": 1},
        # a busy scheduler: a thousand requests, prefill chunks among single tokens, some requests that end
        {"name": "reserve_mixed", "op": "reserve", "requests": 1001, "page": 16, "max_pages": 600, "len_hi": 8192,
         "new_lo": 0, "new_hi": 511, "ended": 0.05, "mix": 2},
        # the cache writes of one decode step
        {"name": "append_decode", "op": "append", "tokens": 64, "run": 1, "kv_heads": 8, "head_dim": 128, "page": 16,
         "dtype": "bf16", "cache": "e4m3", "layout": "hnd", "mix": 3},
        # the cache writes of prefill chunks: odd lengths that begin and end inside pages
        {"name": "append_prefill", "op": "append", "tokens": 16001, "run": 515, "kv_heads": 8, "head_dim": 128,
         "page": 64, "dtype": "f16", "cache": "int8", "layout": "nhd", "mix": 4},
        # one user, one token, a short history: latency alone
        _attention("attend_one_short", 1, 8, 4, 128, 16, "bf16", "e4m3", (777, 777)),
        # the framework's decode workload (64 requests of 512 to 8192 tokens, 8 KV heads, groups of 4) in 8 bits
        _attention("attend_decode", 64, 8, 4, 128, 16, "f16", "e4m3", (512, 8192), mix=4),
        # few requests with very long histories: the split over the tokens counts
        _attention("attend_long", 3, 4, 8, 128, 64, "bf16", "int8", (100_000, 200_000), layout="nhd", mix=5),
        # verification of drafted tokens under a sliding window
        _attention("attend_verify", 48, 4, 2, 64, 32, "f16", "e4m3", (1, 6000), q=(2, 7), long_share=0.5, window=1000,
                   mix=6),
        # prefill chunks next to decoding requests
        _attention("attend_prefill", 6, 8, 4, 128, 16, "bf16", "e4m3", (2048, 8192), q=(1, 2048), long_share=0.6, mix=7),
        # one user's next token over an odd vocabulary
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 50_021, "dtype": "f32", "filters": "top_p",
         "masked": 0.0},
        # a batch of users with their own settings
        {"name": "sample_batch", "op": "sample", "rows": 64, "vocab": 131_072, "dtype": "bf16",
         "filters": "top_k,top_p,min_p", "masked": 0.0},
        # rollouts of many sequences at temperature alone, a grammar's mask over half of the vocabulary
        {"name": "sample_rollout", "op": "sample", "rows": 509, "vocab": 32_000, "dtype": "f32", "filters": "",
         "masked": 0.5},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("reserve", "append", "attention", "attention", "sample"))
    mix = rng.randrange(1 << 20)
    if op == "reserve":
        page = rng.choice((16, 32, 64))
        hi = _spread(rng, 1, 512)
        len_hi = _spread(rng, 16, 8192)
        return {"op": op, "requests": _spread(rng, 1, 1001), "page": page, "max_pages": (len_hi + hi) // page + 2,
                "len_hi": len_hi, "new_lo": rng.choice((0, 1)), "new_hi": hi, "ended": rng.choice((0.0, 0.1)),
                "mix": mix}
    if op == "append":
        tokens = _spread(rng, 1, 16001)
        return {"op": op, "tokens": tokens, "run": _spread(rng, 1, min(tokens, 1000)), "kv_heads": rng.choice((1, 2, 4, 8)),
                "head_dim": rng.choice((64, 128)), "page": rng.choice((16, 32, 64)),
                "dtype": rng.choice(("f16", "bf16", "f32")), "cache": rng.choice(("e4m3", "int8")),
                "layout": rng.choice(("hnd", "nhd")), "mix": mix}
    if op == "sample":
        vocab = _spread(rng, 1000, 131_072)
        return {"op": op, "rows": _spread(rng, 1, max(1, min(509, 8_000_000 // vocab))), "vocab": vocab,
                "dtype": rng.choice(("f32", "bf16", "f16")),
                "filters": rng.choice(("", "top_k", "top_p", "min_p", "top_k,top_p", "top_k,top_p,min_p")),
                "masked": rng.choice((0.0, 0.3))}
    kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 6, 8, 16))
    head_dim, page = rng.choice((64, 128)), rng.choice((16, 32, 64))
    kind = rng.choice(("decode", "verify", "prefill"))
    q_hi = 1 if kind == "decode" else rng.randint(2, 8) if kind == "verify" else _spread(rng, 9, 2048)
    len_hi = _spread(rng, max(q_hi, 16), 16384 if kind == "prefill" else 65536)
    # what the plain form holds at once bounds the batch: gathered K, and the scores
    most = min(2 ** 29 // (len_hi * kv_heads * head_dim), 2 ** 30 // (len_hi * kv_heads * group * q_hi), 128)
    requests = _spread(rng, 1, max(1, most))
    return {"op": op, "requests": requests, "kv_heads": kv_heads, "group": group, "head_dim": head_dim, "page": page,
            "dtype": rng.choice(("f16", "bf16")), "cache": rng.choice(("e4m3", "int8")),
            "len_lo": rng.choice((1, max(1, len_hi // 2))), "len_hi": len_hi, "q_lo": 1, "q_hi": q_hi,
            "long_share": 0.0 if kind == "decode" else 0.7, "window": rng.choice((0, 0, 0, _spread(rng, 16, 4096))),
            "layout": rng.choice(("hnd", "nhd")), "mix": mix}


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone
# ---------------------------------------------------------------------------


def _attention_lens(case):
    rng = random.Random(case["mix"])
    lens, qs = [], []
    for _ in range(case["requests"]):
        many = rng.random() < case["long_share"]
        q = rng.randint(max(case["q_lo"], (case["q_hi"] + 1) // 2), case["q_hi"]) if many else case["q_lo"]
        qs.append(q)
        lens.append(max(q, rng.randint(case["len_lo"], case["len_hi"])))
    return lens, qs


def _reserve_lens(case):
    rng = random.Random(case["mix"])
    lens, new = [], []
    for _ in range(case["requests"]):
        lens.append(rng.randint(0, case["len_hi"]))
        few = rng.random() < 0.5
        new.append(-1 if rng.random() < case["ended"] else
                   case["new_lo"] if few else rng.randint(case["new_lo"], case["new_hi"]))
    return lens, new


def _visible(n, q, window):
    """(row, key) pairs that the mask leaves to q rows at the end of n tokens, and the first key that any row sees."""
    pairs = sum(min(n - q + j + 1, window) if window else n - q + j + 1 for j in range(q))
    return pairs, max(0, n - q + 1 - window) if window else 0


def work(case):
    if case["op"] == "reserve":
        lens, new = _reserve_lens(case)
        page, tokens = case["page"], sum(max(0, n) for n in new)
        pages = sum(-(-(a + max(0, b)) // page) - -(-a // page) if b >= 0 else -(-a // page) for a, b in zip(lens, new))
        touched = sum(-(-(a + b) // page) - a // page for a, b in zip(lens, new) if b > 0)
        return {"bytes": 17 * case["requests"] + 12 * tokens + 8 * pages + 4 * touched, "flops": 0}
    if case["op"] == "append":
        elem = 4 if case["dtype"] == "f32" else 2
        n = case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": 2 * n * (elem + 1) + 8 * case["tokens"], "flops": 4 * n}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2), "flops": 4 * n}
    lens, qs = _attention_lens(case)
    heads, dim, nbytes, flops = case["kv_heads"] * case["group"], case["head_dim"], 0, 0
    for n, q in zip(lens, qs):
        pairs, first = _visible(n, q, case["window"])
        pages = -(-n // case["page"]) - first // case["page"]
        nbytes += 2 * (n - first) * case["kv_heads"] * dim + 8 * pages * case["kv_heads"] + 4 * pages
        nbytes += q * heads * (4 * dim + 4)
        flops += 4 * pairs * heads * dim
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _cuda(values, dtype):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _page_rows(have, max_pages, perm):
    """A block table: `have[r]` pages of `perm` for request r, -1 behind them."""
    table = torch.full((have.numel(), max_pages), -1, dtype=torch.int32, device="cuda")
    mask = torch.arange(max_pages, device="cuda")[None, :] < have[:, None]
    table[mask] = perm[: int(have.sum())].to(torch.int32)
    return table


def _empty_cache(case, pages):
    size = (pages, case["kv_heads"], case["page"], case["head_dim"])
    if case["layout"] == "hnd":  # the tokens of one head of a page stand together
        return torch.empty(size, dtype=_CODES[case["cache"]], device="cuda").transpose(1, 2)
    return torch.empty((size[0], size[2], size[1], size[3]), dtype=_CODES[case["cache"]], device="cuda")


def _filled_cache(case, pages, gen):
    """Codes and scales as a writer leaves them: normal K and V, whose size differs from page to page and head to head."""
    cache, e4m3 = _empty_cache(case, pages), case["cache"] == "e4m3"
    step = max(1, 2 ** 25 // (case["page"] * case["kv_heads"] * case["head_dim"]))
    for a in range(0, pages, step):
        part = cache[a:a + step]
        x = torch.randn(part.shape, generator=gen, device="cuda") * (96.0 if e4m3 else 36.0)
        part.copy_(x.clamp_(-448, 448) if e4m3 else x.round_().clamp_(-127, 127))
    size = torch.exp(0.3 * torch.randn(pages, case["kv_heads"], generator=gen, device="cuda"))
    scale = torch.exp2(torch.round(torch.log2(size / 96.0))) if e4m3 else size / 36.0
    return cache, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *size: torch.randn(size, generator=gen, device="cuda")  # noqa: E731
    state = {"case": dict(case)}
    if case["op"] == "reserve":
        lens, new = _reserve_lens(case)
        page = case["page"]
        kv_len = _cuda(lens, torch.int32)
        have = torch.div(kv_len + page - 1, page, rounding_mode="floor")
        used = sum(-(-n // page) for n in lens)
        pages = used + sum(-(-max(0, n) // page) + 1 for n in new)
        perm = torch.randperm(pages, generator=gen, device="cuda")
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        head = seed % pages
        at = (head + torch.arange(pages - used, device="cuda")) % pages
        ring[at] = perm[used:].to(torch.int32)
        return state | {"table": _page_rows(have, case["max_pages"], perm), "kv_len": kv_len,
                        "new": _cuda(new, torch.int32), "ring": ring,
                        "free": _cuda([head, head + pages - used], torch.int64),
                        "tokens": sum(max(0, n) for n in new)}
    if case["op"] == "append":
        # runs of new tokens, each in pages of its own, beginning anywhere in a page that holds earlier tokens
        page, tokens, run = case["page"], case["tokens"], case["run"]
        rng = random.Random(case["mix"])
        runs = [min(run, tokens - a) for a in range(0, tokens, run)]
        starts = [rng.randrange(page) for _ in runs]
        spans = [-(-(s + n) // page) for s, n in zip(starts, runs)]
        pages = sum(spans) + 3
        perm = torch.randperm(pages, generator=gen, device="cuda")
        first = torch.cumsum(_cuda([0] + spans[:-1], torch.int64), 0)
        of = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), _cuda(runs, torch.int64))
        begin = torch.cumsum(_cuda([0] + runs[:-1], torch.int64), 0)
        at = _cuda(starts, torch.int64)[of] + torch.arange(tokens, device="cuda") - begin[of]
        slots = perm[first[of] + at // page] * page + at % page
        k_cache, k_scale = _filled_cache(case, pages, gen)
        v_cache, v_scale = _filled_cache(case, pages, gen)
        dtype, size = _FLOATS[case["dtype"]], (tokens, case["kv_heads"], case["head_dim"])
        return state | {"k": normal(*size).to(dtype), "v": normal(*size).to(dtype), "slots": slots,
                        "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a wide body of unlikely tokens and a few likely ones, as a model's last layer gives them
        x = 1.5 * normal(rows, vocab)
        at = torch.randint(vocab, (rows, 48), generator=gen, device="cuda")
        x.scatter_add_(1, at, 6.0 + 2.0 * normal(rows, 48))
        if case["masked"]:
            x.masked_fill_(torch.rand(rows, vocab, generator=gen, device="cuda") < case["masked"], -math.inf)
        u = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
        temperature = 0.6 + 0.6 * u()
        if rows > 8:
            temperature[::8] = 0.0  # users who want the likeliest token
        return state | {"logits": x.to(_FLOATS[case["dtype"]]), "u": u(), "temperature": temperature,
                        "top_k": torch.randint(1, 200, (rows,), generator=gen, device="cuda", dtype=torch.int32)
                        if "top_k" in case["filters"] else None,
                        "top_p": 0.5 + 0.49 * u() if "top_p" in case["filters"] else None,
                        "min_p": 0.1 * u() if "min_p" in case["filters"] else None}
    lens, qs = _attention_lens(case)
    page = case["page"]
    kv_len = _cuda(lens, torch.int32)
    have = torch.div(kv_len + page - 1, page, rounding_mode="floor")
    pages, max_pages = sum(-(-n // page) for n in lens), -(-max(lens) // page)
    k_cache, k_scale = _filled_cache(case, pages, gen)
    v_cache, v_scale = _filled_cache(case, pages, gen)
    q = 1.5 * normal(sum(qs), case["kv_heads"] * case["group"], case["head_dim"])
    start = [sum(qs[:i]) for i in range(len(qs) + 1)]
    return state | {"q": q.to(_FLOATS[case["dtype"]]), "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale,
                    "v_scale": v_scale, "kv_len": kv_len, "max_q": max(qs), "longest": max(lens),
                    "table": _page_rows(have, max_pages, torch.randperm(pages, generator=gen, device="cuda")),
                    "q_start": None if max(qs) == 1 else _cuda(start, torch.int32)}


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"reserve": _plain_reserve, "append": _plain_append, "attention": _plain_attention,
            "sample": _plain_sample}[op](state)


def _own(op, s):
    from pto_wsp_b200 import serving

    if op == "reserve":
        step = serving.reserve_pages(s["table"], s["kv_len"], s["new"], s["ring"], s["free"],
                                     page_size=s["case"]["page"], max_tokens=s["tokens"])
        return {"slots": step.slots, "positions": step.positions, "q_start": step.q_start, "kv_len": step.kv_len,
                "free": step.free_state, "granted": step.granted, "table": s["table"], "ring": s["ring"]}
    if op == "append":
        serving.append_kv8(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "sample":
        token, logprob = serving.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                               top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "logprob": logprob}
    out, lse = serving.attend_kv8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                  s["kv_len"], q_start=s["q_start"], max_q=s["max_q"], window=s["case"]["window"],
                                  return_lse=True)
    return {"out": out, "lse": lse}


def _plain_reserve(s):
    page, max_tokens, cap = s["case"]["page"], s["tokens"], s["ring"].numel()
    table, ring = s["table"], s["ring"]
    n, new, max_pages = s["kv_len"].long(), s["new"].long(), table.shape[1]
    want = new.clamp(min=0)
    q_end = torch.cumsum(want, 0)
    q_start = torch.cat([torch.zeros_like(q_end[:1]), q_end])
    have, after = (n + page - 1) // page, (n + want + page - 1) // page
    fits = (new >= 0) & (after <= max_pages) & (q_end <= max_tokens)
    need = torch.where(fits, after - have, 0)
    need_end = torch.cumsum(need, 0)
    head, tail = s["free"][0], s["free"][1]
    granted = fits & ((need == 0) | (need_end <= tail - head))
    back = torch.where(new < 0, have, 0)
    back_end = torch.cumsum(back, 0)
    j = torch.arange(max_pages, device=n.device)[None, :]
    # pages of requests that ended go behind the ring's tail, then new pages come from its head
    to = torch.where(j < back[:, None], (tail + (back_end - back)[:, None] + j) % cap, cap)
    grown = torch.cat([ring, ring[:1]])
    grown[to.reshape(-1)] = table.reshape(-1)
    old = ring.clone()
    ring.copy_(grown[:cap])
    gets = granted[:, None] & (j >= have[:, None]) & (j < after[:, None])
    taken = old[((head + (need_end - need)[:, None] + j - have[:, None]) % cap).reshape(-1)].reshape(table.shape)
    table.copy_(torch.where(gets, taken, table))
    i = torch.arange(max_tokens, device=n.device)
    of = torch.searchsorted(q_end, i, right=True).clamp(max=n.numel() - 1)
    at = n[of] + i - q_start[of]
    ok = (i < q_end[-1]) & granted[of]
    where = table[of, (at // page).clamp(max=max_pages - 1)].long() * page + at % page
    left = torch.stack([head + torch.where(granted, need, 0).sum(), tail + back.sum()])
    return {"slots": torch.where(ok, where, -1), "positions": torch.where(ok, at, -1).int(), "q_start": q_start.int(),
            "kv_len": torch.where(new < 0, 0, n + torch.where(granted, want, 0)).int(), "free": left,
            "granted": granted, "table": table, "ring": ring}


def _scale_of(amax, cache):
    if cache == "int8":
        return (amax / 127.0).clamp(_MIN_SCALE, _MAX_SCALE)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, 448 = 0.875 * 2^9
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    return torch.where(amax > 0, torch.exp2(exponent.float().clamp(-60, 60)), _MIN_SCALE)


def _quantised(x, cache):
    if cache == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _bytes(t):
    return t.view(torch.int8) if t.dtype != torch.int8 else t


def _plain_append(s):
    page, kind = s["case"]["page"], s["case"]["cache"]
    at, off = s["slots"] // page, s["slots"] % page
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf)
        size = torch.where(torch.isinf(x), 0.0, x.abs()).amax(-1)
        amax = torch.zeros_like(scale).index_reduce_(0, at, size, "amax")
        touched = torch.zeros_like(scale[:, 0]).index_fill_(0, at, 1.0).bool()
        fresh = torch.zeros_like(touched).index_fill_(0, at[off == 0], True)
        base = torch.where(fresh[:, None], 0.0, scale)
        grown = torch.where(touched[:, None], torch.maximum(base, _scale_of(amax, kind)), scale)
        redo = (touched & ~fresh & (grown > scale).any(1)).nonzero()[:, 0]
        codes = cache[redo].float() * scale[redo][:, None, :, None] / grown[redo][:, None, :, None]
        _bytes(cache)[redo] = _bytes(_quantised(codes, kind))
        _bytes(cache)[at, off] = _bytes(_quantised(x / grown[at][:, :, None], kind))
        scale.copy_(grown)
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attention(s):
    case, q, table = s["case"], s["q"], s["table"].long().clamp(min=0)
    requests, max_q, longest, dim = case["requests"], s["max_q"], s["longest"], case["head_dim"]
    start = torch.arange(requests + 1, device=q.device) if s["q_start"] is None else s["q_start"].long()
    nq, n = start[1:] - start[:-1], s["kv_len"].long()

    def rows(cache, scale):  # [R, T, heads, D] of real K or V
        x = _bytes(cache)[table].view(cache.dtype).float() * scale[table][:, :, None, :, None]
        return x.reshape(requests, -1, case["kv_heads"], dim)[:, :longest]

    j = torch.arange(max_q, device=q.device)
    at = (start[:-1, None] + j).clamp(max=q.shape[0] - 1)
    real = j < nq[:, None]
    padded = q.float()[at].reshape(requests, max_q, case["kv_heads"], case["group"], dim)
    scores = torch.einsum("rjhgd,rthd->rhgjt", padded, rows(s["k_cache"], s["k_scale"])) * dim ** -0.5
    last = (n - nq)[:, None] + j  # the last key that row j sees
    t = torch.arange(longest, device=q.device)
    seen = t <= last[:, :, None]
    if case["window"]:
        seen &= t > last[:, :, None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum("rhgjt,rthd->rjhgd", weights, rows(s["v_cache"], s["v_scale"]))
    out = out / torch.where(total > 0, total, 1.0).permute(0, 3, 1, 2, 4)
    lse = (torch.log(total) + top)[..., 0].permute(0, 3, 1, 2)
    heads = case["kv_heads"] * case["group"]
    return {"out": out.reshape(requests, max_q, heads, dim)[real].to(q.dtype),
            "lse": lse.reshape(requests, max_q, heads)[real]}


def _plain_sample(s):
    x = torch.nan_to_num(s["logits"].float(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    rows, vocab = x.shape
    column = lambda v, default: torch.full((rows, 1), default, device=x.device) if v is None else v[:, None]  # noqa: E731
    top = x.amax(-1, keepdim=True)
    greedy = ~(s["temperature"][:, None] > 0)
    w = torch.exp((x - top) / torch.where(greedy, 1.0, s["temperature"][:, None]))
    w = torch.where(x == top, 1.0, torch.nan_to_num(w, nan=0.0))
    w = torch.where(torch.isinf(x) & (x < 0), 0.0, w)
    whole = (w * 2.0 ** 40).long()  # sums of whole numbers are exact in any order
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws, wholes = w.gather(1, order), whole.gather(1, order)
    rank = torch.arange(vocab, device=x.device)[None, :]
    k = torch.where(greedy, 1, column(s["top_k"], 0))
    keep = ((k <= 0) | (rank < k)) & (ws >= column(s["min_p"], 0.0).clamp(max=1.0)) & (wholes > 0)
    wholes = wholes * keep
    before = torch.cumsum(wholes, 1) - wholes
    p = column(s["top_p"], 1.0).double()
    limit = torch.ceil(p * wholes.sum(1, keepdim=True).double()).long()
    wholes = wholes * ((p >= 1) | (rank == 0) | (before < limit))
    total = wholes.sum(1, keepdim=True)
    kept = torch.zeros_like(wholes).scatter_(1, order, wholes)
    pick = (s["u"][:, None].double() * total.double()).long().clamp(min=0)
    pick = torch.minimum(pick, (total - 1).clamp(min=0))
    token = (torch.cumsum(kept, 1) <= pick).sum(1, keepdim=True)
    some = total > 0
    chance = kept.gather(1, token.clamp(max=vocab - 1)).float() / total.clamp(min=1).float()
    return {"token": torch.where(some, token, -1)[:, 0].int(),
            "logprob": torch.where(some, torch.log(chance), -math.inf)[:, 0]}


# ---------------------------------------------------------------------------
# The operators' definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reserve":
        return None  # whole numbers only
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_attention(s)


def _exact_e4m3(x):
    """The nearest e4m3 value of each x, ties to the even one: three bits behind the leading one, exponents from -6."""
    x = x.clamp(-448.0, 448.0)
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    exponent = torch.where(torch.exp2(exponent) > x.abs().clamp(min=2.0 ** -6), exponent - 1, exponent)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    page, e4m3, got = s["case"]["page"], s["case"]["cache"] == "e4m3", {}
    pages, order = torch.unique(s["slots"] // page, return_inverse=True)
    off = s["slots"] % page
    begins = torch.zeros(pages.numel(), dtype=torch.bool, device="cuda")
    begins[order[off == 0]] = True
    for name in ("k", "v"):
        x, scale = s[name].double(), s[name + "_scale"].double()
        size = x.abs().amax(-1)
        most = torch.zeros(pages.numel(), size.shape[1], dtype=torch.float64, device="cuda")
        most.scatter_reduce_(0, order[:, None].expand_as(size), size, "amax")
        need = torch.exp2(torch.ceil(torch.log2(most / 448.0))) if e4m3 else most / 127.0
        need = torch.where(begins[:, None], need, torch.maximum(need, scale[pages]))
        codes = s[name + "_cache"].double()
        codes[pages] = codes[pages] * torch.where(begins[:, None], 1.0, scale[pages] / need)[:, None, :, None]
        codes[pages[order], off] = x / need[order][:, :, None]
        scale[pages] = need
        got[name] = _exact_e4m3(codes) if e4m3 else None
        got[name + "_scale"] = scale
    return got


def _exact_sample(s):
    x, token, logprob = s["logits"].double(), [], []
    for r in range(x.shape[0]):
        t = float(s["temperature"][r])
        if t == 0:
            logprob.append(0.0)
            continue
        z, order = torch.sort(x[r], descending=True, stable=True)
        w = torch.softmax(z / t, 0)
        if s["top_k"] is not None:
            w[int(s["top_k"][r]):] = 0
        if s["min_p"] is not None:
            w[w < float(s["min_p"][r]) * w[0]] = 0
        if s["top_p"] is not None:
            w[1:][torch.cumsum(w, 0)[:-1] >= float(s["top_p"][r]) * w.sum()] = 0
        w = torch.zeros_like(w).scatter_(0, order, w / w.sum())
        i = int(torch.searchsorted(torch.cumsum(w, 0), s["u"][r].double(), right=True).clamp(max=w.numel() - 1))
        logprob.append(math.log(float(w[i])) if float(w[i]) > 0 else -math.inf)
    return {"token": None, "logprob": torch.tensor(logprob, dtype=torch.float64, device="cuda")}


def _exact_attention(s):
    case, page = s["case"], s["case"]["page"]
    group, dim = case["group"], case["head_dim"]
    lens, qs = _attention_lens(case)
    out, lse, row = [], [], 0
    for r, (n, q) in enumerate(zip(lens, qs)):
        pages = s["table"][r, : -(-n // page)].long()
        last = torch.arange(n - q, n, device="cuda")[:, None]
        t = torch.arange(n, device="cuda")[None, :]
        hidden = t > last
        if case["window"]:
            hidden = hidden | (t <= last - case["window"])
        part, log = [], []
        for h in range(case["kv_heads"]):
            k, v = ((s[c + "_cache"][pages][:, :, h].double() * s[c + "_scale"][pages, h].double()[:, None, None])
                    .reshape(-1, dim)[:n] for c in "kv")
            for g in range(group):
                z = s["q"][row:row + q, h * group + g].double() @ k.T / math.sqrt(dim)
                z = z.masked_fill(hidden, -math.inf)
                part.append(torch.softmax(z, -1) @ v)
                log.append(torch.logsumexp(z, -1))
        out.append(torch.stack(part, 1))
        lse.append(torch.stack(log, 1))
        row += q
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
