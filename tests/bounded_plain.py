"""The operators of bounded caches in 64 bits, straight from their definitions, one query and head
at a time; and the bounds that their 32-bit kernels keep to."""
import math

import torch

PAGE = 64
EPS32 = 2.0 ** -24


def visible(p, window, sinks):
    """Places that a query at place p sees."""
    lo = max(0, p - window + 1) if window else 0
    return list(range(min(sinks, lo))) + list(range(lo, p + 1))


def attention(q, nh, nkv, hd, k_pages, v_pages, table, cu, ctx, scale, window=None, sinks=0):
    """Returns float64 (out [T, nh * hd], the same of |v|, a bound of a score's 32-bit error in natural
    units, weights {(b, g): [ctx] sums}, largest number of weights in one sum)."""
    T = q.shape[0]
    q, k_pages, v_pages = q.double().cpu(), k_pages.double().cpu(), v_pages.double().cpu()
    table, cu, ctx = table.tolist(), cu.tolist(), ctx.tolist()
    out, mag = torch.zeros((T, nh, hd), dtype=torch.float64), torch.zeros((T, nh, hd), dtype=torch.float64)
    sums, worst, rep, most = {}, 0.0, nh // nkv, 1
    for b, length in enumerate(ctx):
        first = length - (cu[b + 1] - cu[b])
        for g in range(nkv):
            sums[b, g] = torch.zeros(length, dtype=torch.float64)
        most = max(most, (length - first) * rep)
        for t in range(cu[b], cu[b + 1]):
            at = visible(first + t - cu[b], window, sinks)
            pages = [table[b][p // PAGE] for p in at]
            assert min(pages) >= 0
            rows = [p % PAGE for p in at]
            for h in range(nh):
                k, v = k_pages[pages, h // rep, rows], v_pages[pages, h // rep, rows]
                x = q[t, h * hd:(h + 1) * hd]
                w = torch.softmax((k @ x) * scale, 0)
                worst = max(worst, float((k.abs() @ x.abs()).max()) * scale)
                out[t, h], mag[t, h] = w @ v, w @ v.abs()
                sums[b, h // rep][at] += w
    # products are exact or rounded once, sums of hd terms lose at most 2 units in the last place a step
    # (the matrix unit truncates); two more roundings scale and shift the score
    score_err = worst * (2 * hd + 4) * EPS32
    return out.reshape(T, -1), mag.reshape(T, -1), score_err, sums, most


def out_bound(want, mag, score_err, dtype, keys):
    """A weight is off by at most e^(2 score_err) - 1 and the exponential's 2^-21; in bfloat16 it is
    rounded once before it meets the values, and so is the output."""
    rel = 2 * score_err + 2.0 ** -21 + (keys + 8) * 2 * EPS32
    half = torch.finfo(dtype).eps / 2
    if dtype == torch.bfloat16:
        rel = rel + half * 1.01
    return rel * mag + half * want.abs() * 1.01 + 1e-30


def sum_bound(want, old, score_err, terms):
    return (want + old.abs()) * (2 * score_err + 2.0 ** -20 + (terms + 8) * 2 * EPS32) + 1e-30


def select(sums, stored, table, lens, after, keep, sinks, recent):
    """int64 [layers, B, nkv, keep] from float/int tensors [layers, n_pages, nkv, PAGE]."""
    L, _, nkv, _ = sums.shape
    sums, stored, table = sums.cpu().tolist(), stored.cpu().tolist(), table.tolist()
    out = torch.full((L, len(lens), nkv, keep), -1)
    for layer in range(L):
        for b, n in enumerate(lens):
            for g in range(nkv):
                def rank(i):
                    page, r = table[b][i // PAGE], i % PAGE
                    w, p = sums[layer][page][g][r], stored[layer][page][g][r]
                    safe = p < sinks or p >= after[b] - recent
                    return (0, 0.0, i) if safe else (1, math.inf if math.isnan(w) else -w, i)
                best = sorted(range(n), key=rank)[:keep]
                inside, movers = {i for i in best if i < keep}, iter(sorted(i for i in best if i >= keep))
                for i in range(min(n, keep)):
                    out[layer, b, g, i] = i if i in inside else next(movers)
    return out


def move(tensors, table, kept):
    """The tensors ([layers, n_pages, nkv, PAGE, ..]) after the moves that `kept` asks for."""
    new = [t.clone() for t in tensors]
    table = table.tolist()
    for layer in range(kept.shape[0]):
        for b in range(kept.shape[1]):
            for g in range(kept.shape[2]):
                for i, src in enumerate(kept[layer, b, g].tolist()):
                    if src >= 0 and src != i:
                        for o, n in zip(tensors, new):
                            n[layer, table[b][i // PAGE], g, i % PAGE] = o[layer, table[b][src // PAGE], g, src % PAGE]
    return new
