"""Oracle: statements in 64 bits, token by token or request by request, of what gsk.h's operators do over a paged cache (test
infrastructure, never product code).

  to_8        rows in 8 bits with a scale each (the scale in fp32, as it is stored)
  write       rows to their slots
  tokens      a request's cached rows, in order
  attend      softmax attention of new tokens over what they see, with what a computed result may be off by
  beams       the best continuations over beams and vocabulary
  reorder     cached rows moved between beams

Pinned in tests/test_kv_host.py: 8-bit rounding by a search over every value that 8 bits hold, attend by closed forms, beams by a
full sort.
"""
import math

import numpy as np
import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def to_8(x, dtype):
    """float64 rows [..., dim] -> (the values held, float64; the scales, float32). A row with a NaN or infinity: zeros, NaN."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    s = np.maximum(np.abs(x).max(-1).astype(np.float32) * np.float32(1 / MOST[dtype]), np.float32(2.0 ** -126))
    y = (x * (np.float32(1) / s).astype(np.float64)[..., None]).astype(np.float32).astype(np.float64)
    step = 1.0
    if dtype is torch.float8_e4m3fn:
        step = 2.0 ** (np.maximum(np.frexp(np.abs(y))[1] - 1, -6) - 3.0)
    return np.rint(y / step) * step, np.where(bad, np.float32("nan"), s)


def _np(t):
    return (t.float() if t.dtype is torch.float8_e4m3fn else t).double().cpu().numpy()


def write(slot, k, v, keys, values, scales, heads_first):
    """The cache's arrays after the call, float64 (and float32 scales), by slot, as ([keys, values], [scales])."""
    out, sc = [], []
    for i, (x, c) in enumerate(((k, keys), (v, values))):
        c8, x = c.dtype in MOST, _np(x)
        a = _np(c)
        s = scales[i].cpu().numpy().copy() if c8 else None
        page = a.shape[2 if heads_first else 1]
        if c8:
            x, xs = to_8(x, c.dtype)
        for t, z in enumerate(slot.tolist()):
            if 0 <= z < a.shape[0] * page:
                at = (z // page, slice(None), z % page) if heads_first else (z // page, z % page)
                a[at] = x[t]
                if c8:
                    s[at] = xs[t]
        out.append(a)
        sc.append(s)
    return out, sc


def tokens(cache, scale, ids, first, n, heads_first):
    """Tokens first .. first + n - 1 of a request that holds the pages ids: float64 [n, heads, dim] (a page out of range: None
    rows are NaN-free zeros, and False in the mask returned beside)."""
    page, pages = cache.shape[2 if heads_first else 1], cache.shape[0]
    heads, dim = cache.shape[1 if heads_first else 2], cache.shape[3]
    at = first + np.arange(n)
    held = np.concatenate([np.asarray(ids, np.int64), [-1]])
    page_of = held[np.clip(at // page, 0, len(ids))]
    there = (at >= 0) & (at // page < len(ids)) & (page_of >= 0) & (page_of < pages)
    x = np.zeros((n, heads, dim))
    p, o = (torch.from_numpy(i[there]).to(cache.device) for i in (page_of, at % page))
    where = (p, slice(None), o) if heads_first else (p, o)
    rows = _np(cache[where])
    if scale is not None:
        rows = rows * scale[where].cpu().numpy().astype(np.float64)[..., None]
    x[there] = rows
    return x, there


def sees(n, ctx, parents=None, begin=0):
    """bool [n, ctx + n]: which cached tokens each of n new ones sees (ctx of them are older); parents: rows of the whole call."""
    m = np.zeros((n, ctx + n), bool)
    m[:, :ctx] = True
    for i in range(n):
        if parents is None:
            m[i, ctx:ctx + i + 1] = True
            continue
        at = begin + i
        while True:
            m[i, ctx + at - begin] = True
            up = int(parents[at])
            if up < begin or up >= at:
                break
            at = up
    return m


def attend(q, k, v, mask, scale, dtype, bits8):
    """One request: q [n, query heads, dim], k, v [tokens, heads, dim] float64, mask [n, tokens] -> (out, what a result of type
    dtype may be off by), both [n, query heads, dim].

    The bound: out is rounded once (half a step of its size). A weight goes into the product with v as two 16-bit numbers: cut off
    (a step at most, 2^-7 of it in bfloat16, 2^-10 in float16) and the rest, rounded to half a step of that: off by 2^-15 of it, 2^-20
    in float16 (whose rest is up to 2^-12 larger), where the smallest step is 2^-24 and the largest weight 2^7 at least: off by up to
    2^-32 of that, which is at most the sum. Over 8 bits the first is rounded: 2^-16. They are divided by the sum of the unrounded
    ones. A score is a sum of dim products in fp32 and some products more: off by (dim + 8) 2^-24 of the sum of its terms'
    magnitudes; that much, twice (the score's and the largest one's), is the relative error of a weight, and again of their sum.
    exp, its argument's roundings (2^-23 of its size, at most 100 for a weight that counts) and the fp32 sums' (2^-24 for each of a
    chain of at most 4096 terms and joins) come to 2^-11.5 at most, far less in practice: 2^-13 is allowed for them."""
    n, hq, dim = q.shape
    group = hq // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    p16 = 2.0 ** (-16 if bits8 else -20 if dtype is torch.float16 else -15)
    for h in range(hq):
        kk, vv = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kk.T * scale
        size = np.abs(q[:, h]) @ np.abs(kk).T * abs(scale)
        s = np.where(mask, s, -np.inf)
        top = s.max(1, initial=-np.inf, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        total = w.sum(1, keepdims=True)
        w = w / np.where(total > 0, total, 1.0)
        out[:, h] = w @ np.where(mask.any(0)[:, None], vv, 0.0)
        mag = w @ np.abs(np.where(mask.any(0)[:, None], vv, 0.0))
        off = (dim + 8) * 2.0 ** -24 * np.where(mask, size, 0).max(1, initial=0, keepdims=True)
        rel = p16 + 4 * off + 2.0 ** -13
        tol[:, h] = HALF[dtype] * np.abs(out[:, h]) * (1 + rel) + rel * mag
        if not bits8 and dtype is torch.float16:
            tol[:, h] += 2.0 ** -32 * (mask @ np.abs(np.where(mask.any(0)[:, None], vv, 0.0)))
            tol[:, h] += 2.0 ** -25  # (and the result's own smallest step)
    return out, tol


def beams(logits, scores, n):
    """logits float64 [beams, V], scores [beams] of one request -> lists of (token, parent, score), best first."""
    every = []
    for b, (x, s) in enumerate(zip(logits, scores)):
        x = np.where(np.isnan(x), -np.inf, x)
        m = x.max()
        if not (math.isfinite(m) and math.isfinite(s)):
            continue
        lse = math.log(np.exp(x - m).sum())
        t = np.flatnonzero(x > -np.inf)
        every += list(zip((-(((x[t] - m) - lse) + s)).tolist(), [b] * len(t), t.tolist()))
    every.sort()
    return [(t, b, -v) for v, b, t in every[:n]]


def reorder(cache, table, seq_len, parents, first, heads_first):
    """cache [n, pages, page, ...] (numpy) after the call."""
    out, page = cache.copy(), cache.shape[3 if heads_first else 2]
    groups, nb = parents.shape
    width, pages = table.shape[1], cache.shape[1]
    for g in range(groups):
        lo = 0 if first is None else int(first[g])
        for b in range(nb):
            p = int(parents[g, b])
            if not 0 <= p < nb or lo < 0:
                continue
            dst, src = g * nb + b, g * nb + p
            for t in range(lo, min(int(seq_len[dst]), int(seq_len[src]), width * page)):
                i, o = divmod(t, page)
                a, z = int(table[src, i]), int(table[dst, i])
                if 0 <= a < pages and 0 <= z < pages:
                    if heads_first:
                        out[:, z, :, o] = cache[:, a, :, o]
                    else:
                        out[:, z, o] = cache[:, a, o]
    return out
