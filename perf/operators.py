"""The operators of serving many sequences from one paged key-value cache, as cases of one pass each, in two forms: plain torch
operations (`own` false) and the framework's kernels (`own` true).

A cache is a pool of pages, (pages, KV heads, page size, head size); a sequence owns the pages that its row of the block table
names, in order.  One step of a serving loop is: pages and cache rows for the step's new tokens (ops.PagedAdvance), then in every
layer the queries and keys normed and rotated with keys and values written to their rows (ops.QKNormRoPE) and the attention of
each sequence's new token over its pages (ops.PagedDecodeAttention); ops.PagedRelease takes the pages of finished sequences back.

    attention   q (B, NH, D) over `lens` keys of each sequence
    rotate      q, k, v of T tokens out of one (T, (NH + 2 KH) D) projection
    advance     block table, slots and positions for new tokens
    release     the pages of finished sequences back to the pool
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST_KEYS = 64 * 8192 * 8 * 128        # elements of a drawn case's keys, every sequence as long as the longest
MOST_READ = 131072 * 8 * 128 * 4       # bytes of the keys that a drawn case reads


def listed():
    llama8b = {"heads": 32, "kv_heads": 8, "head_dim": 128}
    plain = {"window": 0, "softcap": 0.0, "layout": "heads"}
    return [
        # one chat session, 1024 tokens into the conversation: latency
        {"name": "attention_1x1024", "kind": "attention", "dtype": "bf16", "batch": 1, "longest": 1024, "lengths": "even", "page": 16, **llama8b, **plain},
        # a batch of sessions of every age, as a server has it
        {"name": "attention_64_ragged", "kind": "attention", "dtype": "bf16", "batch": 64, "longest": 8192, "lengths": "ragged", "page": 16, **llama8b, **plain},
        # one session over a very long document
        {"name": "attention_1x131072", "kind": "attention", "dtype": "bf16", "batch": 1, "longest": 131072, "lengths": "even", "page": 64, **llama8b, **plain},
        # the F32 activations and cache of a GGUF model, eight sessions deep into long conversations
        {"name": "attention_f32_8x8192", "kind": "attention", "dtype": "f32", "batch": 8, "longest": 8192, "lengths": "even", "page": 32, **llama8b, **plain},
        # a layer with a sliding window and capped scores, pages that end inside every tile, cache rows of one token side by side
        {"name": "attention_f16_window", "kind": "attention", "dtype": "f16", "batch": 33, "longest": 12001, "lengths": "ragged", "page": 48, "heads": 40, "kv_heads": 4,
         "head_dim": 64, "window": 4096, "softcap": 50.0, "layout": "tokens"},
        # a decode step of 64 sessions
        {"name": "rotate_64", "kind": "rotate", "dtype": "bf16", "tokens": 64, "padded": 0, "first": 5000, "page": 16, **llama8b, "rotary": 128, "interleaved": False,
         "norm": True, "stretch": 1.0},
        # prompts of 8192 tokens in all
        {"name": "rotate_8192", "kind": "rotate", "dtype": "bf16", "tokens": 8192, "padded": 0, "first": 0, "page": 16, **llama8b, "rotary": 128, "interleaved": False,
         "norm": True, "stretch": 1.0},
        # F32, neighbouring dims as pairs, half of the head rotated, stretched frequencies far into a context, a padded batch
        {"name": "rotate_f32_part", "kind": "rotate", "dtype": "f32", "tokens": 1037, "padded": 11, "first": 200000, "page": 32, **llama8b, "rotary": 64, "interleaved": True,
         "norm": False, "stretch": 8.0},
        # the pages of a decode step of 256 sessions
        {"name": "advance_256", "kind": "advance", "requests": 256, "longest": 8192, "new": 1, "padded": 0, "page": 16},
        # prompts of 48 requests
        {"name": "advance_prompts", "kind": "advance", "requests": 48, "longest": 1024, "new": 8192, "padded": 77, "page": 16},
        # some of 256 sessions end; a server of 1000 is emptied for the most part
        {"name": "release_256", "kind": "release", "requests": 256, "longest": 8192, "done": 0.05, "page": 16},
        {"name": "release_1000", "kind": "release", "requests": 1000, "longest": 16384, "done": 0.9, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["rotate"] * 3 + ["advance"] * 2 + ["release"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 48, 64, 100, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "attention":
        d, kh, g = rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8, 8, 10]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
        batch = _log(rng, 1, 200)
        size = 4 if dtype == "f32" else 2
        longest = _log(rng, 1, min(131072, MOST_KEYS // (batch * kh * d), MOST_READ // (2 * size * batch * kh * d)))
        return {"kind": kind, "dtype": dtype, "batch": batch, "longest": longest, "lengths": rng.choice(["even", "ragged", "ragged"]), "page": page, "heads": kh * g, "kv_heads": kh,
                "head_dim": d, "window": rng.choice([0, 0, _log(rng, 1, 8192)]), "softcap": rng.choice([0.0, 0.0, 30.0, 50.0]), "layout": rng.choice(["heads", "tokens"])}
    if kind == "rotate":
        d, kh, g = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 4, 5, 8])
        return {"kind": kind, "dtype": dtype, "tokens": _log(rng, 1, min(16384, MOST_KEYS // (8 * d * kh * (g + 2)))), "padded": rng.choice([0, 0, 5]), "first": rng.choice([0, _log(rng, 1, 1000000)]),
                "page": page, "heads": kh * g, "kv_heads": kh, "head_dim": d, "rotary": rng.choice([d, d, d // 2, d // 4]), "interleaved": rng.choice([False, True]),
                "norm": rng.choice([True, True, False]), "stretch": rng.choice([1.0, 4.0])}
    requests = _log(rng, 1, 2000)
    longest = _log(rng, 1, min(131072, (1 << 24) // requests))
    if kind == "advance":
        return {"kind": kind, "requests": requests, "longest": longest, "new": rng.choice([1, 1, _log(rng, 1, max(1, 131072 // requests))]), "padded": rng.choice([0, 9]), "page": page}
    return {"kind": kind, "requests": requests, "longest": longest, "done": rng.choice([0.02, 0.3, 1.0]), "page": page}


# ---------------------------------------------------------------- the inputs

def _lengths(n, longest, how, least=1):
    """n lengths up to `longest`: all alike, or spread over their logarithm; the same ones for every seed."""
    if how == "even":
        return [longest] * n
    r = random.Random(n * 1000003 + longest)
    some = [min(longest, max(least, _log(r, 1, longest))) for _ in range(n)]
    some[0] = longest
    if n > 8:
        some[3] = 0  # a row of the batch that no sequence has
    return some


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def _shuffled(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def _table(held, width, perm):
    """Row b: the next held[b] page numbers of perm, then -1."""
    held = torch.tensor(held, device=DEVICE)
    first = held.cumsum(0) - held
    w = torch.arange(width, device=DEVICE)
    return torch.where(w < held[:, None], perm[(first[:, None] + w).clamp(max=perm.numel() - 1)], -1).to(torch.int32)


def _new_tokens(case):
    return _lengths(case["requests"], case["new"], "even" if case["new"] == 1 else "ragged")


def _cache(pages, case, layout, g):
    """Keys or values of a pool of pages, as (pages, KH, page, D)."""
    kh, page, d = case["kv_heads"], case["page"], case["head_dim"]
    shape = (pages, kh, page, d) if layout == "heads" else (pages, page, kh, d)
    t = torch.randn(shape, generator=g, device=DEVICE).to(DTYPES[case["dtype"]])
    return t if layout == "heads" else t.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    i32 = {"dtype": torch.int32, "device": DEVICE}
    page = case["page"]
    s = {"case": case}
    if case["kind"] == "attention":
        lens = _shuffled(_lengths(case["batch"], case["longest"], case["lengths"]), seed)
        held = _pages(lens, page)
        pool = sum(held) + 3
        s["q"] = (2 * torch.randn((case["batch"], case["heads"], case["head_dim"]), generator=g, device=DEVICE)).to(DTYPES[case["dtype"]])
        s["k_cache"], s["v_cache"] = (_cache(pool, case, case["layout"], g) for _ in range(2))
        s["table"] = _table(held, max(max(held), 1), torch.randperm(pool, generator=g, device=DEVICE))
        s["lens"] = torch.tensor(lens, **i32)
        s["scale"] = case["head_dim"] ** -0.5
    elif case["kind"] == "rotate":
        T, NH, KH, D, R = (case[n] for n in ("tokens", "heads", "kv_heads", "head_dim", "rotary"))
        dt = DTYPES[case["dtype"]]
        qkv = torch.randn((T, (NH + 2 * KH) * D), generator=g, device=DEVICE).to(dt)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in qkv.split((NH * D, KH * D, KH * D), dim=1))
        s["q_weight"], s["k_weight"] = (((1 + 0.1 * torch.randn(D, generator=g, device=DEVICE)).to(dt) for _ in range(2)) if case["norm"] else (None, None))
        s["inv_freq"] = 500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEVICE) / R) / case["stretch"]
        s["positions"] = case["first"] + torch.randint(0, 8192, (T,), generator=g, device=DEVICE)
        pool = 2 * -(-T // page) + 64
        s["k_cache"], s["v_cache"] = (_cache(pool, case, "heads", g) for _ in range(2))
        s["slots"] = torch.randperm(pool * page, generator=g, device=DEVICE)[:T].contiguous()
        if case["padded"]:
            s["slots"][T - min(T - 1, case["padded"]):] = -1
    else:
        lens = _shuffled(_lengths(case["requests"], case["longest"], "ragged"), seed)
        held = _pages(lens, page)
        if case["kind"] == "advance":
            new = _shuffled(_new_tokens(case), seed)
            more = [-(-(n + m) // page) - h for n, m, h in zip(lens, new, held)]
            s["new_lens"] = torch.tensor(new, **i32)
            s["tokens"] = sum(new) + case["padded"]
            free = sum(more) + 5
            width = max(h + m for h, m in zip(held, more)) + 1
        else:
            done = _shuffled([i < max(1, round(case["done"] * len(lens))) for i in range(len(lens))], seed + 1)
            s["done"] = torch.tensor(done, device=DEVICE)
            free, width = 7, max(held) + 1
        pool = sum(held) + free
        perm = torch.randperm(pool, generator=g, device=DEVICE)
        s["table"] = _table(held, width, perm)
        s["lens"] = torch.tensor(lens, **i32)
        s["free_pages"] = torch.cat([perm[pool - free:], torch.zeros(pool - free, dtype=torch.int64, device=DEVICE)]).to(torch.int32)
        s["free_count"] = torch.tensor([free], **i32)
    return s


# ---------------------------------------------------------------- the plain forms

def _attention(s):
    q, k_cache, v_cache, lens, case = s["q"], s["k_cache"], s["v_cache"], s["lens"], s["case"]
    (B, NH, D), KH, W = q.shape, k_cache.shape[1], s["table"].shape[1]
    rows = s["table"].clamp(min=0).long()
    k = k_cache[rows].transpose(1, 2).reshape(B, KH, -1, D).float()     # (B, KH, W page, D)
    v = v_cache[rows].transpose(1, 2).reshape(B, KH, -1, D).float()
    scores = torch.matmul(q.float().view(B, KH, NH // KH, D), k.transpose(2, 3)) * s["scale"]
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    j = torch.arange(k.shape[2], device=q.device)
    n = lens[:, None]
    seen = j < n
    if case["window"]:
        seen = seen & (j >= n - case["window"])
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return torch.where(n[:, :, None] > 0, out.reshape(B, NH, D), 0.0).to(q.dtype)


def _rotate(s):
    R, between = s["case"]["rotary"], s["case"]["interleaved"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    c, n = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turned(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
        if between:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            turn = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            turn = torch.cat((a * c - b * n, a * n + b * c), -1)
        return torch.cat((turn, y[..., R:]), -1).to(x.dtype)

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    kept = s["slots"] >= 0
    slots, page = s["slots"][kept], s["k_cache"].shape[2]
    s["k_cache"][slots // page, :, slots % page] = k[kept]
    s["v_cache"][slots // page, :, slots % page] = s["v"][kept]
    return q, s["k_cache"], s["v_cache"]


def _advance(s):
    page, table, T = s["case"]["page"], s["table"], s["tokens"]
    lens, new = s["lens"].long(), s["new_lens"].long()
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    held = (lens + page - 1) // page
    more = (lens + new + page - 1) // page - held
    first = more.cumsum(0) - more
    granted = (more == 0) | (first + more <= s["free_count"])
    w = torch.arange(table.shape[1], device=table.device) - held[:, None]
    at = (s["free_count"].long() - 1 - first[:, None] - w).clamp(0, s["free_pages"].numel() - 1)
    table.copy_(torch.where((w >= 0) & (w < more[:, None]) & granted[:, None], s["free_pages"][at], table))
    i = torch.arange(T, device=table.device)
    b = torch.searchsorted(starts[1:], i, right=True).clamp(max=lens.numel() - 1)
    inside = i < starts[-1]
    position = torch.where(inside, lens[b] + i - starts[b], 0)
    slot = table[b, position // page].long() * page + position % page
    given = torch.where(granted, new, 0)
    left = s["free_count"] - torch.where(granted, more, 0).sum().to(torch.int32)
    return {"positions": position, "slots": torch.where(inside & granted[b], slot, -1), "starts": starts.to(torch.int32), "lens": (lens + given).to(torch.int32),
            "granted": given.to(torch.int32), "free_count": left, "block_table": table}


def _release(s):
    page, table, free = s["case"]["page"], s["table"], s["free_pages"]
    held = torch.where(s["done"], (s["lens"].long() + page - 1) // page, 0)
    first = held.cumsum(0) - held
    w = torch.arange(table.shape[1], device=table.device)
    gone = w < held[:, None]
    free[(s["free_count"].long() + first[:, None] + w)[gone]] = table[gone]
    return {"lens": torch.where(s["done"], 0, s["lens"]), "free_count": s["free_count"] + held.sum().to(torch.int32), "free_pages": free}


def _by_kernels(s):
    from light_b200 import ops

    case, kind = s["case"], s["case"]["kind"]
    if kind == "attention":
        return ops.PagedDecodeAttention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["scale"], window=case["window"], softcap=case["softcap"])
    if kind == "rotate":
        q, _ = ops.QKNormRoPE(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6, interleaved=case["interleaved"],
                              v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], slots=s["slots"])
        return q, s["k_cache"], s["v_cache"]
    if kind == "advance":
        r = ops.PagedAdvance(s["table"], s["lens"], s["new_lens"], s["free_pages"], s["free_count"], case["page"], s["tokens"])
        return {"positions": r.positions, "slots": r.slots, "starts": r.starts, "lens": r.lens, "granted": r.granted, "free_count": r.free_count, "block_table": s["table"]}
    lens, free_count = ops.PagedRelease(s["table"], s["lens"], s["done"], s["free_pages"], s["free_count"], case["page"])
    return {"lens": lens, "free_count": free_count, "free_pages": s["free_pages"]}


def run(state):
    if own:
        return _by_kernels(state)
    return {"attention": _attention, "rotate": _rotate, "advance": _advance, "release": _release}[state["case"]["kind"]](state)


def work(case):
    kind, page = case["kind"], case["page"]
    if kind in ("attention", "rotate"):
        size, D, NH, KH = 4 if case["dtype"] == "f32" else 2, case["head_dim"], case["heads"], case["kv_heads"]
    if kind == "attention":
        lens = _lengths(case["batch"], case["longest"], case["lengths"])
        keys = sum(min(n, case["window"] or n) for n in lens)
        named = sum(-(-n // page) - max(0, n - (case["window"] or n)) // page for n in lens)
        return {"bytes": 2 * keys * KH * D * size + 2 * case["batch"] * NH * D * size + 4 * named + 4 * len(lens), "flops": 4 * keys * NH * D}
    if kind == "rotate":
        T = case["tokens"]
        return {"bytes": 2 * T * (NH + 2 * KH) * D * size + 16 * T + 8 * case["rotary"] // 2, "flops": T * (NH + KH) * (3 * case["rotary"] + (4 * D if case["norm"] else 0))}
    n = case["requests"]
    lens = _lengths(n, case["longest"], "ragged")
    if kind == "advance":
        new = _new_tokens(case)
        most = sum(-(-m // page) for m in new)
        return {"bytes": 20 * n + 8 * most + 16 * (sum(new) + case["padded"]), "flops": 0}
    count = max(1, round(case["done"] * n))
    return {"bytes": 9 * n + 8 * sum(_pages(lens, page)) * count // n, "flops": 0}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        B, NH, D = s["q"].shape
        KH, page = s["k_cache"].shape[1:3]
        out = torch.zeros((B, NH, D), dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            j = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device=DEVICE)
            at = s["table"][b].long()[j // page]
            for h in range(KH):
                k, v = s["k_cache"][at, h, j % page].double(), s["v_cache"][at, h, j % page].double()
                group = slice(h * (NH // KH), (h + 1) * (NH // KH))
                x = s["q"][b, group].double() @ k.T * s["scale"]
                x = x if not case["softcap"] else torch.tanh(x / case["softcap"]) * case["softcap"]
                out[b, group] = torch.softmax(x, dim=-1) @ v
        return out
    if case["kind"] == "rotate":
        R, T = case["rotary"], case["tokens"]
        unit = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), s["positions"][:, None, None].double() * s["inv_freq"])

        def turned(x, weight):
            y = x.double()
            if weight is not None:
                y = y / ((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * weight.double()
            front = y[..., :R].unflatten(-1, (R // 2, 2) if case["interleaved"] else (2, R // 2))
            if not case["interleaved"]:
                front = front.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(front.contiguous()) * unit)
            return torch.cat(((z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2), y[..., R:]), -1)

        caches = []
        for name, rows in (("k_cache", turned(s["k"], s["k_weight"])), ("v_cache", s["v"].double())):
            flat = s[name].double().transpose(1, 2).flatten(0, 1).contiguous()  # (cache rows, KH, D)
            used = [t for t, x in enumerate(s["slots"].tolist()) if x >= 0]
            flat[s["slots"][used]] = rows[used]
            caches.append(flat.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous())
        return turned(s["q"], s["q_weight"]), caches[0], caches[1]
    return None
