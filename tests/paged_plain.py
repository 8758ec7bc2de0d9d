"""The paged operators from their definitions, in 64 bits and plain Python or torch, and how far a kernel may be from them."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
# ... and absolute, where results are subnormal: halves below 2^-14 lie 2^-24 apart (11 bits from 2^-14 on down to 2^-24), so a rounding moves
# one by up to 2^-25 whatever its size; of the other types the same is below 2^-133
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def advance(table, lens, new, free, count, page, tokens):
    """One request after the other.  Lists in, lists out; `table` is changed."""
    width, got_all, given, starts, pos, slot, avail = len(table[0]), True, [], [0], [0] * tokens, [-1] * tokens, min(max(count, 0), len(free))
    top, out = avail, []
    for b, (n, m) in enumerate(zip(lens, new)):
        n, m = max(n, 0), max(m, 0)
        starts.append(starts[-1] + m)
        held = -(-n // page)
        fits = n + m <= width * page and starts[-1] <= tokens
        more = -(-(n + m) // page) - held if fits else 0
        ok = fits and (more == 0 or (got_all and more <= top))
        if fits and not ok:
            got_all = False
        if ok:
            for w in range(held, held + more):
                top -= 1
                table[b][w] = free[top]
        for i in range(m):
            if starts[b] + i < tokens:
                pos[starts[b] + i] = n + i
                if ok and table[b][(n + i) // page] >= 0:
                    slot[starts[b] + i] = table[b][(n + i) // page] * page + (n + i) % page
        given.append(m if ok else 0)
        out.append(n + (m if ok else 0))
    return pos, slot, starts, out, given, top


def release(table, lens, done, free, count, page):
    avail = min(max(count, 0), len(free))
    out = list(lens)
    for b, d in enumerate(done):
        if d:
            for w in range(min(-(-max(lens[b], 0) // page), len(table[0]))):
                if avail < len(free):
                    free[avail] = table[b][w]
                    avail += 1
            out[b] = 0
    return out, avail


def rotated(x, weight, eps, positions, inv_freq, interleaved, factor):
    """x (T, heads, D) -> (the result in f64, the bound on |kernel - result|)."""
    T, _, D = x.shape
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    R = 2 * inv_freq.numel()
    t = positions.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(t) * factor, torch.sin(t) * factor
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    out, size = y.clone(), y.abs()
    first, second = a * c - b * s, a * s + b * c
    both = (a.abs() + b.abs()) * max(factor, 1.0)
    if interleaved:
        out[..., 0:R:2], out[..., 1:R:2], size[..., 0:R:2], size[..., 1:R:2] = first, second, both, both
    else:
        out[..., :R // 2], out[..., R // 2:R], size[..., :R // 2], size[..., R // 2:R] = first, second, both, both
    # in f32: the mean of D squares (relative error D / 2 steps in the root), root, quotient and two products; sine and cosine of an angle reduced
    # in 64 bits (argument rounded: up to pi 2^-24; the functions: two steps; times factor), two products, a sum
    return out, LEAST[x.dtype] + EPS[x.dtype] * out.abs() + (D / 2 + 24) * 2.0 ** -24 * size


def attention(q, k_cache, v_cache, table, lens, scale, window=0, softcap=0.0, rounded_p=True):
    """(the result in f64, the bound on |kernel - result|); pages outside the cache hold no keys."""
    B, NH, D = q.shape
    pages, KH, page, _ = k_cache.shape
    G, cap = NH // KH, table.shape[1] * page
    out = torch.zeros((B, NH, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    u, u_p = EPS[q.dtype], EPS[q.dtype] if rounded_p and q.dtype != torch.float32 else 0.0
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), cap)
        j = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        pg = table[b].long()[j // page]
        inside = (pg >= 0) & (pg < pages)
        j, pg = j[inside], pg[inside]
        if n == 0:
            continue
        for h in range(KH):
            k, v = k_cache[pg, h, j % page].double(), v_cache[pg, h, j % page].double()
            x = q[b, h * G:(h + 1) * G].double()
            s = x @ k.T * scale
            size = (x.abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True) if len(j) else torch.zeros((G, 1), device=q.device)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            p = torch.softmax(s, -1)
            out[b, h * G:(h + 1) * G] = p @ v
            spread = p @ v.abs()
            # a score: D products summed in f32 (tensor cores cut, they do not round: a whole step each), scaled, capped (a tanh right to 16 steps of its
            # value, and no larger than the score); its error is p's relative one, exp2 adds two steps, and rescaling at a new maximum one each time, 64 times at most; the sums over the keys: one step per key
            # in the worst order.  Numerator and denominator have them each.
            e = (D + 8 + (8 if softcap else 0)) * 2.0 ** -23 * size + 70 * 2.0 ** -23 + min(len(j), 4096) * 2.0 ** -24
            bound[b, h * G:(h + 1) * G] = u * p.matmul(v).abs() + 2 * (u_p + e) * spread + LEAST[q.dtype]
    return out, bound
