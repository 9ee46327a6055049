"""GPU parity of the paged cache's operators (kv.write, kv.read, kv.attend, kv.reorder) against the oracle's statements in 64 bits,
whose docstrings derive what a computed result may be off by; and runs of them with page steps, verify rounds and beams."""
import importlib

import numpy as np
import pytest
import torch

from oracle import kv_ref as kr

pytestmark = pytest.mark.gpu

BF, HF, F32, E4, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


def _kv():
    return importlib.import_module("goethe-engine_amd").kv


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def _gen(gpu, seed):
    return torch.Generator(device=gpu).manual_seed(seed)


def _cache(g, dtype, pages, page, heads, dim, heads_first):
    """Keys, values, scales of a cache whose every slot holds something."""
    shape = (pages, heads, page) if heads_first else (pages, page, heads)
    if dtype in (E4, I8):
        if dtype is I8:
            k, v = (torch.randint(-127, 128, (*shape, dim), generator=g, device=g.device, dtype=torch.int8) for _ in range(2))
        else:
            k, v = ((_rand(g, *shape, dim) * 60).clamp(-448, 448).to(E4) for _ in range(2))
        return k, v, tuple(torch.rand(shape, generator=g, device=g.device) * 0.02 + 0.002 for _ in range(2))
    return _rand(g, *shape, dim).to(dtype), _rand(g, *shape, dim).to(dtype), None


def _pages(g, lengths, page, width=None, spare=3):
    """A table with each request's own pages, -1 past them, and the number of pages."""
    held = [(n + page - 1) // page for n in lengths]
    width = width or max(max(held), 1)
    ids = torch.randperm(sum(held) + spare, generator=g, device=g.device).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=g.device)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = ids[at:at + n]
        at += n
    return table, sum(held) + spare


# ---- write ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", [BF, HF, E4, I8])
@pytest.mark.parametrize("source", [BF, HF, F32])
def test_write(ge, gpu, cache, source):
    """Every pair of types, both orders, dims from 8 to 256: bit for bit what the definition gives; slots that are negative or past
    the cache are skipped and the other slots left as they were."""
    for seed, (dim, heads, page, first) in enumerate([(8, 1, 1, False), (64, 3, 16, True), (80, 5, 24, False), (128, 8, 16, False),
                                                      (136, 2, 7, True), (256, 1, 32, False)]):
        g = _gen(gpu, seed)
        keys, values, scales = _cache(g, cache, 9, page, heads, dim, first)
        n = min(9 * page, 37)
        slot = torch.randperm(9 * page, generator=g, device=gpu)[:n]
        slot[::5] = torch.tensor([-1, 9 * page, 2 ** 40, -2 ** 40], device=gpu).repeat(n)[:len(slot[::5])]
        k = (_rand(g, n, heads, dim) * torch.exp(2 * _rand(g, n, heads, 1))).to(source)
        v = _rand(g, n, heads, dim).to(source)
        v[0], v[n // 2, 0, :5] = 0, 0
        want, ws = kr.write(slot, k, v, keys, values, scales, first)
        ge.kv.write(slot, k, v, keys, values, scales=scales, heads_first=first)
        for i, c in enumerate((keys, values)):
            got = kr._np(c)
            if cache in (BF, HF):
                want[i] = kr._np(torch.from_numpy(want[i]).float().to(cache))  # (rounded once, from fp32)
            assert np.array_equal(got, want[i])
            if scales is not None:
                assert np.array_equal(scales[i].cpu().numpy(), ws[i])


@pytest.mark.parametrize("cache", [E4, I8])
def test_write_edges_of_8_bits(ge, gpu, cache):
    """Rows of zeros, of the largest and smallest numbers, ties between two values, NaN and infinities (which read as NaN)."""
    x = torch.zeros(12, 1, 16, device=gpu)
    m = kr.MOST[cache]
    x[1], x[2], x[3, 0, 3] = 3.4e38, -1e-45, 1e-38
    x[4, 0] = torch.arange(16, device=gpu) * m / 15
    x[5, 0, 0], x[5, 0, 1:] = m, torch.arange(15, device=gpu) + 0.5
    x[6, 0, 0], x[6, 0, 1:] = m, 2.0 ** -torch.arange(15, device=gpu).float()
    x[7, 0, 0], x[7, 0, 1:] = -m, 2.0 ** -10 * torch.arange(15, device=gpu)
    x[8, 0, 5], x[9, 0, 5], x[10, 0, 5], x[11, 0, 15] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[8, 0, 0] = 1
    keys, values, scales = _cache(_gen(gpu, 0), cache, 4, 4, 1, 16, False)
    slot = torch.arange(12, device=gpu) + 2
    want, ws = kr.write(slot, x, x.flip(0), keys, values, scales, False)
    ge.kv.write(slot, x, x.flip(0), keys, values, scales=scales)
    for c, w, s, z in zip((keys, values), want, scales, ws):
        assert np.array_equal(kr._np(c), w) and np.array_equal(s.cpu().numpy(), z, equal_nan=True)
    k, _ = ge.kv.read(keys, values, torch.arange(4, dtype=torch.int32, device=gpu)[None], [0, 12], first=[2], scales=scales, dtype=F32)
    assert torch.isnan(k[8:]).all() and torch.isfinite(k[:8]).all() and (k[0] == 0).all()


def test_write_strides(ge, gpu):
    """Rows that are slices of one projection, at steps of any kind; caches that are layers of one array; scales of an order of
    their own. What lies between stays."""
    g = _gen(gpu, 3)
    qkv = _rand(g, 50, 12, 64).to(BF)
    big = torch.zeros((6, 3, 2, 10, 4, 64), dtype=BF, device=gpu)  # [pages, layers, keys and values, page, heads, dim]
    keys, values = big[:, 1, 0], big[:, 1, 1]
    slot = torch.randperm(60, generator=g, device=gpu)[:50]
    want, _ = kr.write(slot, qkv[:, 4:8], qkv[:, 8:], keys, values, None, False)
    ge.kv.write(slot, qkv[:, 4:8], qkv[:, 8:], keys, values)
    assert np.array_equal(kr._np(keys), want[0]) and np.array_equal(kr._np(values), want[1])
    assert (big[:, ::2] == 0).all()
    # a source of unaligned rows, slots of a step, 8 bits with scales heads first
    odd = _rand(g, 50, 4, 69)[:, :, 1:65]
    keys8, values8, _ = _cache(g, I8, 6, 10, 4, 64, False)
    scales = tuple(torch.zeros((6, 4, 10), device=gpu).transpose(1, 2) for _ in range(2))
    twice = torch.stack([slot, slot], 1)[:, 0]
    want, ws = kr.write(twice, odd, odd, keys8, values8, scales, False)
    ge.kv.write(twice, odd, odd, keys8, values8, scales=scales)
    assert np.array_equal(kr._np(keys8), want[0]) and np.array_equal(scales[1].cpu().numpy(), ws[1])
    ge.kv.write(slot[:0], odd[:0], odd[:0], keys8, values8, scales=scales)
    assert np.array_equal(kr._np(keys8), want[0])


# ---- read ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", [BF, HF, E4, I8])
@pytest.mark.parametrize("out", [BF, HF, F32])
def test_read(ge, gpu, cache, out):
    """Ragged requests, empty ones among them, read from any first token; rows off by their rounding alone (a product in fp32, then
    half a step of the rows' type)."""
    for seed, (dim, heads, page, first) in enumerate([(8, 2, 1, False), (72, 3, 16, True), (128, 8, 24, False), (192, 1, 5, True)]):
        g = _gen(gpu, seed)
        lengths = [5, 0, 33, 1, 0, 0, 64, 17, 0]
        table, pages = _pages(g, lengths, page)
        keys, values, scales = _cache(g, cache, pages, page, heads, dim, first)
        start = [min(n, s) for n, s in zip(lengths, [0, 0, 7, 0, 0, 3, 31, 17, 0])]
        begin = np.concatenate([[0], np.cumsum(np.array(lengths) - start)])
        k, v = ge.kv.read(keys, values, table, begin.tolist(), first=start, scales=scales, dtype=out, heads_first=first)
        assert k.shape == (begin[-1], heads, dim) and k.dtype is out
        for c, s, got in ((keys, 0, k), (values, 1, v)):
            want = np.concatenate([kr.tokens(c, scales[s] if scales else None, table[r].tolist(), start[r], lengths[r] - start[r],
                                             first)[0] for r in range(len(lengths))])
            assert (np.abs(kr._np(got) - want) <= (kr.HALF[out] + 2.0 ** -23) * np.abs(want) + (2.0 ** -25 if out is HF else 0)).all()


def test_read_leaves_and_zeros(ge, gpu):
    """Rows past the last request stay, rows whose token or page is out of range are zero, offsets out of order touch nothing else."""
    g = _gen(gpu, 1)
    table, pages = _pages(g, [24, 24, 24], 8)
    keys, values, _ = _cache(g, BF, pages, 8, 2, 64, False)
    out = tuple(torch.full((40, 2, 64), 7.0, dtype=BF, device=gpu) for _ in range(2))
    bad = table.clone()
    bad[1, 1], bad[2, 0] = pages, -5
    k, v = ge.kv.read(keys, values, bad, torch.tensor([0, 10, 20, 30], dtype=torch.int32, device=gpu),
                      first=torch.tensor([-3, 4, 20], dtype=torch.int32, device=gpu), max_tokens=40, out=out)
    assert k is out[0] and (k[30:] == 7).all() and (v[30:] == 7).all()
    where = [[(0, t) if t >= 0 else None for t in range(-3, 7)], [(1, t) if t < 8 or t >= 16 else None for t in range(4, 14)],
             [None] * 10]  # (request 2: from its token 20 on, past its table after four)
    for row, at in enumerate(sum(where[:2], [])):
        want = torch.zeros((2, 64), dtype=BF, device=gpu) if at is None else keys[bad[at[0], at[1] // 8].long(), at[1] % 8]
        assert torch.equal(k[row], want), row
    assert torch.equal(k[20:24], keys[bad[2, 2].long(), 4:8]) and (k[24:30] == 0).all()
    for begin in ([5, 3, 9, 40], [0, 0, 0, 0], [-9, -8, 2 ** 31 - 1, 4], [40, 30, 20, 10]):
        o = tuple(torch.full((40, 2, 64), 7.0, dtype=BF, device=gpu) for _ in range(2))
        ge.kv.read(keys, values, table, torch.tensor(begin, dtype=torch.int32, device=gpu), max_tokens=40, out=o)
    torch.cuda.synchronize()


def test_read_many_requests(ge, gpu):
    """More requests than a wave looks at in one step, of zero to three tokens."""
    g = _gen(gpu, 2)
    rng = np.random.default_rng(0)
    lengths = rng.integers(0, 4, 9000)
    lengths[4000:4500] = 0
    held = int((lengths > 0).sum())
    table = torch.full((9000, 1), -1, dtype=torch.int32, device=gpu)
    table[torch.from_numpy(lengths > 0).to(gpu), 0] = torch.randperm(held, generator=g, device=gpu).int()
    keys, values, _ = _cache(g, HF, held, 4, 1, 8, False)
    begin = np.concatenate([[0], np.cumsum(lengths)])
    k, v = ge.kv.read(keys, values, table, begin, dtype=HF)
    req = np.repeat(np.arange(9000), lengths)
    at = torch.from_numpy(np.arange(begin[-1]) - begin[req]).to(gpu)
    ids = table[torch.from_numpy(req).to(gpu), 0].long()
    assert torch.equal(k, keys[ids, at]) and torch.equal(v, values[ids, at])


# ---- attend --------------------------------------------------------------------------------------------------------------

def _check(ge, q, keys, values, scales, table, lengths, news, first, parents=None, scale=None, served=None, **kw):
    """kv.attend against the oracle, request by request; rows past the last request stay as they were."""
    gpu = q.device
    begin = np.concatenate([[0], np.cumsum(news)])
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device=gpu)
    kw.setdefault("max_new", max(1, max(news)))
    got = ge.kv.attend(q, keys, values, table, torch.tensor(lengths, dtype=torch.int32, device=gpu),
                       begin=torch.tensor(begin, dtype=torch.int32, device=gpu), scales=scales, heads_first=first,
                       parents=None if parents is None else torch.tensor(parents, dtype=torch.int32, device=gpu), scale=scale,
                       out=out, **kw)
    assert got is out and (out[begin[-1]:] == 9).all()
    got, qn, worst = kr._np(out), kr._np(q), 0.0
    ks, vs = scales or (None, None)
    for r, (n, ln) in enumerate(zip(news, lengths)):
        if n == 0:
            continue
        a = got[begin[r]:begin[r + 1]]
        if served is not None and not served[r]:
            assert (a == 0).all()
            continue
        ids = table[r].tolist()
        k, there = kr.tokens(keys, ks, ids, 0, ln, first)
        v, _ = kr.tokens(values, vs, ids, 0, ln, first)
        mask = kr.sees(n, ln - n, parents, begin[r]) & there
        want, tol = kr.attend(qn[begin[r]:begin[r + 1]], k, v, mask, float(np.float32(q.shape[2] ** -0.5 if scale is None else scale)),
                              q.dtype, keys.dtype in kr.MOST)
        off = np.abs(a - want)
        assert (off <= tol).all(), (r, n, ln, float((off / np.maximum(tol, 1e-30)).max()))
        worst = max(worst, float((off / np.maximum(tol, 1e-30)).max()))
    return worst


KINDS = [(BF, BF), (HF, HF), (BF, E4), (HF, E4), (BF, I8), (HF, I8)]
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 600, 1, 1030]


@pytest.mark.parametrize("query,cache", KINDS)
@pytest.mark.parametrize("dim,heads,group,page,first", [(128, 2, 4, 16, False), (64, 3, 1, 32, True), (80, 5, 3, 24, False),
                                                        (8, 1, 7, 1, False), (256, 1, 8, 64, True), (136, 2, 2, 5, False),
                                                        (96, 1, 17, 128, False), (192, 2, 40, 16, True)])
def test_attend_one_token(ge, gpu, query, cache, dim, heads, group, page, first):
    """One new token a request, at lengths around every tile and page end."""
    g = _gen(gpu, dim + page)
    table, pages = _pages(g, EDGES, page)
    keys, values, scales = _cache(g, cache, pages, page, heads, dim, first)
    q = _rand(g, len(EDGES), heads * group, dim).to(query)
    _check(ge, q, keys, values, scales, table, EDGES, [1] * len(EDGES), first)
    b = ge.kv.attend(q, keys, values, table, torch.tensor(EDGES, device=gpu), scales=scales, heads_first=first)
    a = ge.kv.attend(q, keys, values, table, torch.tensor(EDGES, device=gpu), begin=list(range(len(EDGES) + 1)), scales=scales,
                     heads_first=first)
    assert torch.equal(a, b)


@pytest.mark.parametrize("query,cache", KINDS)
@pytest.mark.parametrize("dim,heads,group,page,first", [(128, 2, 4, 16, False), (80, 3, 5, 24, True), (64, 1, 1, 1, False), (256, 1, 2, 32, False)])
def test_attend_chains(ge, gpu, query, cache, dim, heads, group, page, first):
    """Ragged chains of new tokens, requests without any, requests that are nothing but new tokens; spare rows stay."""
    g = _gen(gpu, page)
    news = [1, 0, 7, 13, 2, 40, 9, 5, 0, 33]
    lengths = [1, 0, 7, 45, 300, 40, 41, 5, 77, 513]
    table, pages = _pages(g, lengths, page)
    keys, values, scales = _cache(g, cache, pages, page, heads, dim, first)
    q = _rand(g, sum(news) + 6, heads * group, dim).to(query)
    _check(ge, q, keys, values, scales, table, lengths, news, first)


@pytest.mark.parametrize("query,cache,group,page", [(BF, BF, 4, 16), (HF, HF, 1, 24), (BF, E4, 8, 1), (HF, I8, 3, 64)])
def test_attend_trees(ge, gpu, query, cache, group, page):
    """Trees of up to 64 nodes: chains, stars, random ones; entries that are no earlier row of the request end a path."""
    g = _gen(gpu, 5)
    rng = np.random.default_rng(1)
    news, lengths = [9, 1, 64, 20, 33, 0, 64, 12], [100, 1, 64, 533, 40, 9, 1000, 12]
    begin = np.concatenate([[0], np.cumsum(news)])
    par = np.full(begin[-1], -1)
    for r, n in enumerate(news):
        for i in range(1, n):
            par[begin[r] + i] = begin[r] + (i - 1 if r == 2 else 0 if r == 3 else int(rng.integers(0, i)))
    par[begin[4] + 5], par[begin[4] + 6], par[begin[4] + 7] = begin[4] + 5, begin[4] - 3, 10 ** 6
    par[begin[7]] = 0
    table, pages = _pages(g, lengths, page)
    keys, values, scales = _cache(g, cache, pages, page, 2, 128, False)
    q = _rand(g, sum(news), 2 * group, 128).to(query)
    _check(ge, q, keys, values, scales, table, lengths, news, False, parents=par.tolist())


@pytest.mark.parametrize("cache", [BF, E4])
def test_attend_long(ge, gpu, cache):
    """A long request beside short ones (its parts are joined), an odd page, and a prompt of many new tokens."""
    g = _gen(gpu, 7)
    for lengths, news, group in (([70001, 3, 900], [1, 1, 1], 4), ([9000], [2], 1), ([1500, 2100], [700, 300], 2)):
        table, pages = _pages(g, lengths, 48)
        keys, values, scales = _cache(g, cache, pages, 48, 2, 64, False)
        q = _rand(g, sum(news), 2 * group, 64).to(BF)
        _check(ge, q, keys, values, scales, table, lengths, news, False)


def test_attend_many_requests(ge, gpu):
    """More requests than tickets, most of them short, some empty."""
    g = _gen(gpu, 8)
    rng = np.random.default_rng(2)
    lengths = rng.integers(1, 40, 5000).tolist()
    lengths[17] = 3000
    table, pages = _pages(g, lengths, 16)
    keys, values, _ = _cache(g, BF, pages, 16, 1, 64, False)
    q = _rand(g, 5000, 2, 64).to(BF)
    got = ge.kv.attend(q, keys, values, table, lengths)
    for r in [*range(0, 5000, 97), 17, 4999]:
        k, there = kr.tokens(keys, None, table[r].tolist(), 0, lengths[r], False)
        v, _ = kr.tokens(values, None, table[r].tolist(), 0, lengths[r], False)
        want, tol = kr.attend(kr._np(q[r:r + 1]), k, v, there[None], 64 ** -0.5, BF, False)
        assert (np.abs(kr._np(got[r:r + 1]) - want) <= tol).all(), r


def test_attend_scores_of_every_size(ge, gpu):
    """Weights that are all alike, one that outweighs the rest at either end, scores far from zero, a scale of zero and below."""
    g = _gen(gpu, 9)
    lengths = [300, 300, 300, 77]
    table, pages = _pages(g, lengths, 16)
    for query in (BF, HF):
        keys, values, _ = _cache(g, query, pages, 16, 2, 64, False)
        q = _rand(g, 4, 4, 64).to(query)
        keys[table[1, 0], 0] *= 8
        keys[table[2, 18], 11] *= 8
        for scale in (0.0, 0.125, -0.125, 4.0, 2.0 ** -30):
            _check(ge, q, keys, values, None, table, lengths, [1] * 4, False, scale=scale)


@pytest.mark.parametrize("cache", [BF, HF, E4, I8])
@pytest.mark.parametrize("page", [16, 24, 5])
def test_attend_reads_no_more_than_it_sees(ge, gpu, cache, page):
    """NaN and infinities in pages of others, behind the last token and in scales there change nothing; a table's entries past a
    request's pages are anything."""
    g = _gen(gpu, 10)
    lengths, news = [37, 1, 100, 0, 64, 255], [1, 1, 5, 0, 3, 2]
    table, pages = _pages(g, lengths, page, width=60, spare=9)
    keys, values, scales = _cache(g, cache, pages, page, 2, 80, False)
    q = _rand(g, sum(news), 4, 80).to(BF if cache in (E4, I8) else cache)
    used = torch.zeros((pages, page), dtype=torch.bool, device=gpu)
    for r, n in enumerate(lengths):
        for t in range(n):
            used[table[r, t // page].long(), t % page] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=gpu)
    for c in (keys, values):
        if cache is not I8:
            fill = bad[torch.randint(0, 3, c.shape, generator=g, device=gpu)]
            c.copy_(torch.where(used[..., None, None], c.float(), fill if cache is not E4 else torch.full_like(fill, float("nan"))).to(cache))
    for s in scales or ():
        s.copy_(torch.where(used[..., None], s, float("nan")))
    behind = torch.arange(60, device=gpu) >= torch.tensor([(n + page - 1) // page for n in lengths], device=gpu)[:, None]
    table[behind] = torch.randint(-2 ** 31, 2 ** 31 - 1, (int(behind.sum()),), generator=g, device=gpu, dtype=torch.int64).int()
    _check(ge, q, keys, values, scales, table, lengths, news, False)


@pytest.mark.parametrize("page", [16, 24])
def test_attend_pages_and_numbers_out_of_range(ge, gpu, page):
    """Pages out of range are not seen (a request of nothing else gives 0); lengths, offsets and statuses out of order give zeros
    or nothing, and their neighbours are right."""
    g = _gen(gpu, 11)
    lengths, news = [50, 50, 90, 64, 33, 70], [1, 2, 1, 1, 3, 1]
    table, pages = _pages(g, lengths, page)
    keys, values, _ = _cache(g, BF, pages, page, 2, 64, False)
    q = _rand(g, sum(news), 4, 64).to(BF)
    table[0, 0], table[1, 1], table[3, :] = -1, pages, pages + 7
    table[2, 2] = -2 ** 31
    _check(ge, q, keys, values, None, table, lengths, news, False)
    assert (ge.kv.attend(q[:6], keys, values, table, lengths)[3] == 0).all()
    status = torch.tensor([0, 1, 0, 0, 2, 0], dtype=torch.int32, device=gpu)
    _check(ge, q, keys, values, None, table, lengths, news, False, status=status, served=[True, False, True, True, False, True])
    cap = table.shape[1] * page
    odd = [50, 1, cap + 1, -7, 2, 2 ** 31 - 1]  # fewer than their new tokens, past the table, negative
    got = ge.kv.attend(q, keys, values, table, torch.tensor(odd, device=gpu), begin=[0, 1, 3, 4, 5, 8, 9])
    assert (got[1:] == 0).all() and (got[0] != 0).any()
    for begin in ([0, 1, 0, 4, 5, 8, 9], [-4, 1, 3, 4, 5, 8, 9], [0, 1, 3, 4, 5, 8, 2 ** 31 - 1], [9, 8, 7, 6, 5, 4, 3]):
        out = torch.full_like(q, 9.0)
        ge.kv.attend(q, keys, values, table, torch.tensor(lengths, device=gpu), begin=torch.tensor(begin, dtype=torch.int32, device=gpu),
                     max_new=3, out=out)
        assert torch.isfinite(out).all()
    out = torch.full_like(q, 9.0)  # a request of more new tokens than max_new: the later ones are left out
    ge.kv.attend(q, keys, values, table, torch.tensor([50, 50], device=gpu).repeat(3), begin=[0, 1, 3, 4, 5, 8, 9], max_new=2, out=out)
    assert (out[7] == 9).all() and (out[8] != 9).any()


def test_attend_strides(ge, gpu):
    """Queries inside one projection, caches that are layers of one array, tables inside wider ones, unaligned queries."""
    g = _gen(gpu, 12)
    lengths, news = [100, 37, 250], [2, 1, 4]
    table, pages = _pages(g, lengths, 16)
    wide = torch.full((3, 40), -9, dtype=torch.int32, device=gpu)
    wide[:, 5:5 + table.shape[1]] = table
    big = _rand(g, pages, 2, 2, 16, 3, 64).to(BF)
    qkv = _rand(g, 7, 12, 64).to(BF)
    for q in (qkv[:, :6], _rand(g, 7, 6, 67).to(BF)[:, :, 2:66], qkv[:, ::2], _rand(g, 6, 7, 64).to(BF).transpose(0, 1)):
        _check(ge, q, big[:, 1, 0], big[:, 1, 1], None, wide[:, 5:5 + table.shape[1]], lengths, news, False)
    one = _rand(g, pages, 16, 3, 64).to(BF)
    _check(ge, qkv[:, :3], one, one, None, table, lengths, news, False)  # values that are the keys


def test_attend_twice_is_the_same(ge, gpu):
    """Parts are joined in their order: the same bits at every call."""
    g = _gen(gpu, 13)
    lengths = [20000, 5, 3000, 12000]
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, E4, pages, 16, 2, 128, False)
    q = _rand(g, 4, 16, 128).to(BF)
    first = ge.kv.attend(q, keys, values, table, lengths, scales=scales)
    for _ in range(5):
        assert torch.equal(first, ge.kv.attend(q, keys, values, table, lengths, scales=scales))


def test_attend_past_32_bits(ge, gpu):
    """A cache of more than 2^32 elements: pages at its end."""
    page, heads, dim = 64, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 40
    keys = torch.zeros((pages, page, heads, dim), dtype=I8, device=gpu)
    values = torch.zeros_like(keys)
    scales = tuple(torch.full((pages, page, heads), 0.01, device=gpu) for _ in range(2))
    g = _gen(gpu, 14)
    ids = torch.cat([torch.arange(pages - 20, pages, device=gpu), torch.arange(5, device=gpu)]).int()[None]
    for p in ids[0].tolist():
        for c in (keys, values):
            c[p] = torch.randint(-127, 128, c.shape[1:], generator=g, device=gpu, dtype=I8)
    q = _rand(g, 1, 16, dim).to(BF)
    small = ids[0].long()
    want = ge.kv.attend(q, keys[small], values[small], torch.arange(25, dtype=torch.int32, device=gpu)[None], [1590],
                        scales=tuple(s[small] for s in scales))
    assert torch.equal(ge.kv.attend(q, keys, values, ids, [1590], scales=scales), want)
    k, v = _rand(g, 30, heads, dim).to(BF), _rand(g, 30, heads, dim).to(BF)
    slot = torch.arange(30, device=gpu) + (pages * page - 30)
    ge.kv.write(slot, k, v, keys, values, scales=scales)
    w, ws = kr.to_8(kr._np(k), I8)
    assert np.array_equal(kr._np(keys[-1, -30:]), w) and np.array_equal(scales[0][-1, -30:].cpu().numpy(), ws)
    back, _ = ge.kv.read(keys, values, torch.tensor([[pages - 1]], dtype=torch.int32, device=gpu), [0, 30], first=[34], scales=scales, dtype=F32)
    assert np.array_equal(back.cpu().numpy(), (w.astype(np.float32) * ws[..., None]))


# ---- reorder -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,shape,first", [(BF, (8, 64), False), (torch.uint8, (5, 80), True), (torch.uint8, (3, 7), False),
                                               (torch.float32, (1, 1), True), (torch.int8, (2, 18), True)])
@pytest.mark.parametrize("beams,groups,page", [(1, 2, 4), (2, 3, 16), (4, 2, 7), (7, 3, 1), (8, 1, 24), (16, 2, 16), (32, 1, 5)])
def test_reorder(ge, gpu, dtype, shape, first, beams, groups, page):
    """Permutations, one beam that all continue, parents out of range; prompts that stay, lengths that differ."""
    rng = np.random.default_rng(beams * 100 + page)
    g = _gen(gpu, beams)
    lengths = rng.integers(0, 90, groups).repeat(beams)
    lengths[rng.random(len(lengths)) < 0.1] //= 2
    table, pages = _pages(g, lengths.tolist(), page, width=100)
    each = (pages, shape[0], page, *shape[1:]) if first else (pages, page, *shape)
    caches = torch.randint(-128, 128, (3, *each), generator=g, device=gpu).to(dtype)
    parents = rng.integers(-1, beams + 1, (groups, beams)) if groups > 1 else rng.permutation(beams)[None]
    parents[-1] = beams - 1 if beams in (4, 16) else parents[-1]
    prompt = rng.integers(0, 30, groups) if groups > 1 else None
    want = kr.reorder(caches.cpu().to(torch.int64).numpy(), table.cpu().numpy(), lengths, parents, prompt, first)
    for stacked in (True, False):
        c = caches.clone()
        ge.kv.reorder(c if stacked else ge.paged.Caches(list(c), heads_first=first), table, torch.from_numpy(lengths).to(gpu),
                      torch.from_numpy(parents).to(gpu), first=None if prompt is None else prompt.tolist(), heads_first=first)
        assert np.array_equal(c.cpu().to(torch.int64).numpy(), want)


def test_reorder_bad_pages(ge, gpu):
    """Pages out of range, rows past the table, a negative first: nothing outside is touched, the rest is moved."""
    g = _gen(gpu, 4)
    table, pages = _pages(g, [30] * 4, 8)
    caches = torch.randint(0, 256, (2, pages, 8, 2, 16), generator=g, device=gpu).to(torch.uint8)
    table[0, 1], table[1, 2], table[3, 0] = -1, pages, 2 ** 31 - 1
    parents = np.array([[1, 0], [1, 1]])
    for lengths, prompt in ([30] * 4, [0, 0]), ([2 ** 31 - 1] * 4, [3, 0]), ([30, 30, -5, 30], [2 ** 31 - 1, 0]), ([30] * 4, [-1, 2]):
        want = kr.reorder(caches.cpu().numpy(), table.cpu().numpy(), lengths, parents, prompt, False)
        c = caches.clone()
        ge.kv.reorder(c, table, lengths, torch.from_numpy(parents).to(gpu), first=prompt)
        assert np.array_equal(c.cpu().numpy(), want)


@pytest.mark.parametrize("query,cache", [(BF, BF), (HF, HF), (BF, E4), (HF, I8)])
@pytest.mark.parametrize("tree", [False, True])
def test_attend_bad_values_of_unseen_tokens(ge, gpu, query, cache, tree):
    """NaN and infinities in the keys and values of new tokens reach the tokens that see them and no others; a row written with a
    NaN (whose 8-bit scale is NaN) likewise."""
    g = _gen(gpu, 21)
    lengths, news, group, page = [50, 9, 300], [9, 9, 20], 4, 16
    table, pages = _pages(g, lengths, page)
    keys, values, scales = _cache(g, cache, pages, page, 2, 80, False)
    q = _rand(g, sum(news), 2 * group, 80).to(query)
    begin = np.concatenate([[0], np.cumsum(news)])
    par = None
    if tree:
        par = np.concatenate([begin[r] + np.array([-1 - begin[r]] + [(i - 1) // 2 for i in range(1, n)]) for r, n in enumerate(news)])
    clean = ge.kv.attend(q, keys, values, table, lengths, begin=begin.tolist(), parents=par, scales=scales)
    for r, i, what, value in [(0, 5, "v", float("nan")), (1, 0, "v", float("inf")), (2, 12, "v", -float("inf")), (0, 7, "k", float("nan")),
                              (2, 19, "both", float("inf"))]:
        t = lengths[r] - news[r] + i
        at = (table[r, t // page].long(), t % page)
        was = [x[at].clone() for x in (keys, values, *(scales or ()))]
        row = torch.ones((1, 2, 80), device=gpu)
        row[0, 1, 3] = value
        kk = row if what in ("k", "both") else torch.ones_like(row)
        vv = row if what in ("v", "both") else torch.ones_like(row)
        ge.kv.write((at[0] * page + at[1]).reshape(1), kk, vv, keys, values, scales=scales)
        got = ge.kv.attend(q, keys, values, table, lengths, begin=begin.tolist(), parents=par, scales=scales)
        for rr, n in enumerate(news):
            sees = kr.sees(n, 0, None if par is None else par, begin[rr])
            for k in range(n):
                a, b = got[begin[rr] + k].float(), clean[begin[rr] + k].float()
                if rr != r or not sees[k, i]:
                    assert torch.equal(a, b), (r, i, what, rr, k)
                elif what == "v":
                    assert torch.isfinite(a[:group]).all()  # (the first head's row is fine)
                    if cache in (BF, HF):
                        assert torch.isfinite(a[group:]).sum() == group * 79 and (
                            torch.isnan(a[group:, 3]).all() if value != value else (a[group:, 3] == value).all())
                    else:
                        assert torch.isnan(a[group:]).all()
        for x, w in zip((keys, values, *(scales or ())), was):
            x[at] = w


@pytest.mark.parametrize("query,cache", KINDS)
@pytest.mark.parametrize("dim,heads,group", [(128, 8, 4), (80, 12, 3), (64, 4, 2)])
def test_attend_heads_together(ge, gpu, query, cache, dim, heads, group):
    """Tokens enough that, their heads lying together, a wave takes a head of its own: requests that share their pages (a table
    may name a page twice), chains or a tree, short and empty ones among them; and the same caches with the heads ahead."""
    g = _gen(gpu, dim + heads)
    many = 44 if heads > 8 else 68 if heads == 8 else 132
    news = ([2, 1, 0, 3] if group < 4 else [1, 1, 0, 1]) * (many // 4)
    lengths = [10000 - 13 * r if r % 4 else 17 for r in range(many)]
    lengths[2] = 0
    par = None
    if group == 3:
        begin = np.concatenate([[0], np.cumsum(news)])
        par = [-1 if i == 0 else int(begin[r]) for r, n in enumerate(news) for i in range(n)]
    one, pages = _pages(g, [10000], 16)
    table = one.repeat(many, 1)
    keys, values, scales = _cache(g, cache, pages, 16, heads, dim, False)
    q = _rand(g, sum(news), heads * group, dim).to(query)
    args = dict(begin=np.concatenate([[0], np.cumsum(news)]), parents=par, max_new=3)
    got = ge.kv.attend(q, keys, values, table, lengths, scales=scales, **args)
    turned = [x.transpose(1, 2).contiguous() for x in (keys, values, *(scales or ()))]
    ahead = ge.kv.attend(q, turned[0], turned[1], table, lengths, scales=tuple(turned[2:]) or None, heads_first=True, **args)
    k, _ = kr.tokens(keys, scales and scales[0], one[0].tolist(), 0, 10000, False)
    v, _ = kr.tokens(values, scales and scales[1], one[0].tolist(), 0, 10000, False)
    begin, qn = args["begin"], kr._np(q)
    for r in [0, 1, 3, 4, many // 2 + 1, many - 1]:
        n, ln = news[r], lengths[r]
        want, tol = kr.attend(qn[begin[r]:begin[r + 1]], k[:ln], v[:ln], kr.sees(n, ln - n, par, begin[r]), float(np.float32(dim ** -0.5)),
                              query, cache in kr.MOST)
        for x in (got, ahead):
            assert (np.abs(kr._np(x[begin[r]:begin[r + 1]]) - want) <= tol).all(), r
    # every row: what one order of the cache gives is what the other gives, to twice the bound's size
    off = (got.float() - ahead.float()).abs()
    assert (off <= 2 ** -6 * (ahead.float().abs() + ahead.float().abs().mean())).all()


@pytest.mark.parametrize("cache", [BF, HF, E4, I8])
def test_attend_bad_values_of_older_tokens(ge, gpu, cache):
    """A NaN or an infinity in an older token's value reaches every new token of its request, wherever it lies: beside the new
    ones, in a block with a page that is out of range, far from both."""
    g = _gen(gpu, 22)
    lengths, news, page = [70, 70, 130], [6, 1, 4], 8
    table, pages = _pages(g, lengths, page)
    table[2, 3] = -1
    keys, values, scales = _cache(g, cache, pages, page, 2, 64, False)
    query = HF if cache is HF else BF
    q = _rand(g, sum(news), 4, 64).to(query)
    begin = [0, 6, 7, 11]
    clean = ge.kv.attend(q, keys, values, table, lengths, begin=begin, scales=scales)
    for r, t, value in [(0, 63, float("inf")), (0, 3, float("nan")), (1, 68, -float("inf")), (2, 33, float("inf")), (2, 20, float("nan")),
                        (2, 120, float("inf"))]:
        at = (table[r, t // page].long(), t % page)
        was = [x[at].clone() for x in (keys, values, *(scales or ()))]
        row = torch.ones((1, 2, 64), device=gpu)
        row[0, 1, 3] = value
        ge.kv.write((at[0] * page + at[1]).reshape(1), torch.ones_like(row), row, keys, values, scales=scales)
        got = ge.kv.attend(q, keys, values, table, lengths, begin=begin, scales=scales).float()
        for rr in range(3):
            a = got[begin[rr]:begin[rr + 1]]
            if rr != r:
                assert torch.equal(a, clean[begin[rr]:begin[rr + 1]].float()), (r, t)
            elif cache in (BF, HF):
                assert torch.isfinite(a[:, :2]).all() and torch.isfinite(a[:, 2:]).sum() == news[r] * 2 * 63, (r, t)
                assert torch.isnan(a[:, 2:, 3]).all() if value != value else (a[:, 2:, 3] == value).all(), (r, t)
            else:
                assert torch.isfinite(a[:, :2]).all() and torch.isnan(a[:, 2:]).all(), (r, t)
        for x, w in zip((keys, values, *(scales or ())), was):
            x[at] = w


@pytest.mark.parametrize("query,cache,dim,heads,group", [(BF, BF, 128, 2, 4), (HF, I8, 80, 3, 5), (BF, E4, 256, 1, 3)])
def test_attend_prompts_beside_single_tokens(ge, gpu, query, cache, dim, heads, group):
    """A step of a long prompt's chunk, short ones and single tokens; a wide max_new over the same rows changes no bit."""
    g = _gen(gpu, dim + group)
    news = [1, 1, 130, 0, 17, 1, 70, 1]
    lengths = [900, 1, 333, 0, 17, 64, 71, 2000]
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, cache, pages, 16, heads, dim, False)
    q = _rand(g, sum(news) + 3, heads * group, dim).to(query)
    _check(ge, q, keys, values, scales, table, lengths, news, False)
    begin = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=gpu)
    seq = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    a, b = (ge.kv.attend(q, keys, values, table, seq, begin=begin, scales=scales, max_new=m)[:sum(news)] for m in (130, 220))
    assert torch.equal(a, b)


def test_attend_new_tokens_past_what_is_counted(ge, gpu):
    """More new tokens times cached ones than 2^32 blocks: refused."""
    x = torch.zeros((1, 1, 1, 8), dtype=BF, device=gpu)
    table = torch.zeros((1, (1 << 31) - 1), dtype=torch.int32, device="meta").expand(1, -1)
    q = torch.zeros((1 << 12, 1, 8), dtype=BF, device=gpu)
    with pytest.raises(ValueError, match="fewer new ones"):
        ge.kv.attend(q, x, x, table, [1], begin=[0, 1 << 12], max_new=1 << 12)
