"""How far attention's results are from the definition in 64 bits: little more than their own rounding, whatever the type of the
cache, the spread of the weights and the size of the values."""
import numpy as np
import pytest
import torch

from oracle import kv_ref as kr
from test_gpu_kv import BF, E4, HF, I8, KINDS, _cache, _gen, _pages, _rand

pytestmark = pytest.mark.gpu


def _both(ge, q, keys, values, scales, table, lengths, news, parents=None, rows=None, scale=None):
    """kv.attend's and the oracle's outputs [rows, query heads, dim], float64, and the oracle's bound, of the requests `rows`."""
    begin = np.concatenate([[0], np.cumsum(news)])
    got = kr._np(ge.kv.attend(q, keys, values, table, lengths, begin=begin, scales=scales, parents=parents, scale=scale))
    ks, vs = scales or (None, None)
    out = []
    for r in range(len(news)) if rows is None else rows:
        ids, at = table[r].tolist(), slice(begin[r], begin[r + 1])
        k, there = kr.tokens(keys, ks, ids, 0, lengths[r], False)
        v, _ = kr.tokens(values, vs, ids, 0, lengths[r], False)
        mask = kr.sees(news[r], lengths[r] - news[r], parents, begin[r]) & there
        scale_of = float(np.float32(q.shape[2] ** -0.5 if scale is None else scale))
        out.append((got[at], *kr.attend(kr._np(q[at]), k, v, mask, scale_of, q.dtype, keys.dtype in kr.MOST)))
    return [np.concatenate(x) for x in zip(*out)]


def _rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


@pytest.mark.parametrize("query,cache", KINDS)
@pytest.mark.parametrize("what", ["trees", "chains", "long", "one"])
def test_attend_is_off_by_its_rounding(ge, gpu, query, cache, what):
    """The rms error over a call is that of the results' own rounding: every weight goes into the product to 2^-15 of it (2^-20 in
    a float16 cache, 2^-16 in 8 bits), a rounding whose rms is a quarter of that, independent of the other weights', so that the sum
    is off by about 2^-17 of its size (2^-22, 2^-18); the results' own rounding is 2^-8 / sqrt(12) to twice that, 2^-9.8 at least, in
    float16 2^-12.8. The scores' fp32 sums, 2^-20 at these sizes, add less. So at most sqrt(1 + 2^-10) of the rounding's rms is
    expected, and 1.02 allowed. A block of 32 tokens left out of n alike moves the results by sqrt(32 / n) of their size: 2^-6 of it at
    the longest here, ten times the rounding."""
    g = _gen(gpu, 31)
    parents, dim, group = None, 128, 4
    if what == "trees":
        news, lengths = [9] * 6, [900, 64, 9, 1500, 333, 2000]
        begin = np.concatenate([[0], np.cumsum(news)])
        parents = np.concatenate([begin[r] + np.array([-1 - begin[r]] + [(i - 1) // 2 for i in range(1, 9)]) for r in range(6)])
    elif what == "chains":
        news, lengths, dim, group = [6, 1, 3, 5, 2, 40], [700, 1, 60, 1300, 31, 40], 80, 3
    elif what == "long":
        news, lengths, dim = [1, 1, 2], [100003, 9, 30011], 64
    else:
        news, lengths, group = [1] * 8, [33, 64, 100, 1, 257, 1000, 3000, 31], 2
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, cache, pages, 16, 2, dim, False)
    q = _rand(g, sum(news), 2 * group, dim).to(query)
    got, want, tol = _both(ge, q, keys, values, scales, table, lengths, news, parents)
    assert (np.abs(got - want) <= tol).all()
    rounded = kr._np(torch.from_numpy(want).to(query))
    assert _rms(got - want) <= 1.02 * _rms(rounded - want), (_rms(got - want), _rms(rounded - want))
    if what == "long":  # (each request by itself: the short one's results are large)
        for i in (slice(0, 1), slice(2, 4)):
            assert _rms(got[i] - want[i]) <= 1.02 * _rms(rounded[i] - want[i])


@pytest.mark.parametrize("query,cache", [(HF, HF), (BF, BF), (HF, I8), (BF, E4)])
def test_attend_a_sink_and_a_long_tail(ge, gpu, query, cache):
    """One token of weight 1 and 131072 of 2^-25.1 each, together 2^-8.1, that share its wave's maximum: they count. As many
    requests as workgroups run at once, so that a wave has a quarter of a request."""
    n, many, dim = 131073, 768, 8
    table = torch.randperm(n // 64 + 1, generator=_gen(gpu, 32), device=gpu).int()[None].repeat(many, 1)
    pages = table.shape[1]
    keys = torch.zeros((pages, 64, 1, dim), device=gpu)
    values = torch.ones((pages, 64, 1, dim), device=gpu)
    keys[table[0, 0].long(), 0], values[table[0, 0].long(), 0] = 25.1 * np.log(2) / dim, -1
    scales = None
    if cache in kr.MOST:
        keys[table[0, 0].long(), 0] = 2
        scales = tuple(torch.full((pages, 64, 1), x, device=gpu) for x in (float(25.1 * np.log(2) / dim / 2), 1.0))
    keys, values = keys.to(cache), values.to(cache)
    q = torch.ones((many, 1, dim), device=gpu).to(query)
    got, want, tol = _both(ge, q, keys, values, scales, table, [n] * many, [1] * many, rows=[0, 1, 400, many - 1], scale=1.0)
    assert -0.9935 < want[0, 0, 0] < -0.991
    assert (np.abs(got - want) <= tol).all(), float(np.abs(got - want).max())


@pytest.mark.parametrize("cache", [BF, E4, I8])
def test_attend_values_of_every_size(ge, gpu, cache):
    """Values near the end of fp32's range, and far below 1: sums over many tokens of one weight, over ones whose weight grows
    up to 2^7.9 before the maximum follows, joined or not, are as exact as at any size."""
    g = _gen(gpu, 33)
    lengths = [1, 32, 300, 5000, 40000]
    table, pages = _pages(g, lengths, 16)
    keys, _, scales = _cache(g, cache, pages, 16, 1, 64, False)
    held = {BF: [-1.75, 1.0, 1.25, 1.9375], E4: [-448.0, 256.0, 320.0, 384.0], I8: [-127.0, 64.0, 100.0, 126.0]}[cache]
    end = {BF: 2.0 ** 127, E4: 2.0 ** 119, I8: 2.0 ** 121 * 0.98}[cache]  # (1.9375 * 2^127 = 3.3e38)
    codes = torch.tensor(held, device=gpu)[torch.randint(0, 4, (pages, 16, 1, 64), generator=g, device=gpu)].double()
    q = _rand(g, len(lengths), 4, 64).to(BF)
    grow = torch.arange(40000, device=gpu) / 40000 * 5.4  # (natural: 2^7.8)
    for rising in (False, True):
        k = torch.zeros((pages, 16, 1, 64), device=gpu)
        if rising:
            k.view(-1, 1, 64)[(table[4].long()[:, None] * 16 + torch.arange(16, device=gpu)).reshape(-1)[:40000], 0, 0] = grow
            q[:] = 0
            q[..., 0] = 8
        ks = None
        if cache in kr.MOST:
            ks = torch.full((pages, 16, 1), 5.4 / kr.MOST[cache], device=gpu)
            k = torch.round(k / ks[..., None]) if cache is I8 else k / ks[..., None]
        for size in (end, 1.0, 2.0 ** -70):
            v, vs = (codes * size).to(BF) if cache is BF else codes.to(cache), torch.full((pages, 16, 1), size, device=gpu)
            got, want, tol = _both(ge, q, k.to(cache), v, None if cache is BF else (ks, vs), table, lengths, [1] * 5)
            assert np.isfinite(want).all() and np.abs(want).max() > 0
            assert np.isfinite(got).all(), (rising, size)
            assert (np.abs(got - want) <= tol).all(), (rising, size, float((np.abs(got - want) / tol).max()))


def test_attend_under_a_bound_far_above_its_rows(ge, gpu):
    """A max_new of 2^24 over four new tokens of 256 query heads a head (2^32 rows at most, 2^31 with 128): the scratch memory is that of
    any bound that fills the row tiles, and so are the results."""
    lib, kv = ge._lib, ge.kv
    rows = lib.handle(gpu.index, 1, 1).rows
    size, at = (kv._CACHE.size, lib.K_BF16, 200, 16, 1, 64), (1024, 64, 64)
    for heads in (128, 130, 200, 256):
        wide, some = (kv._work_bytes(gpu.index, rows, size, at, (1, 4, heads, lib.K_BF16, m, 200)) for m in (1 << 24, 1000))
        assert wide == some > 0
    g = _gen(gpu, 34)
    lengths, news = [3001], [4]
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, BF, pages, 16, 1, 64, False)
    for heads in (128, 200, 256):
        q = _rand(g, 4, heads, 64).to(BF)
        got, want, tol = _both(ge, q, keys, values, scales, table, lengths, news)
        assert (np.abs(got - want) <= tol).all()
        wide = ge.kv.attend(q, keys, values, table, lengths, begin=[0, 4], max_new=1 << 24)
        assert (np.abs(kr._np(wide) - want) <= tol).all()


def test_attention_work_counts_its_rows(ge, gpu):
    """New tokens times a head's query heads past 2^32, over one page of one token: the library refuses them too."""
    lib, kv = ge._lib, ge.kv
    size, at = (kv._CACHE.size, lib.K_BF16, 1, 1, 1, 8), (8, 8, 8)
    rows = lib.handle(gpu.index, 1, 1).rows
    assert kv._work_bytes(gpu.index, rows, size, at, (1, 1 << 24, 255, lib.K_BF16, 1 << 24, 1)) > 0
    for heads in (256, 300, 512):
        with pytest.raises(RuntimeError, match="fewer new ones"):
            kv._work_bytes(gpu.index, rows, size, at, (1, 1 << 24, heads, lib.K_BF16, 1 << 24, 1))


def test_attention_takes_scales_to_2_to_127(ge, gpu):
    """Scores of a scale of 2^127 that are 0 are 0, and equal; the library refuses what is past it."""
    g = _gen(gpu, 35)
    table, pages = _pages(g, [40], 16)
    keys, values, _ = _cache(g, BF, pages, 16, 1, 64, False)
    q = torch.zeros((1, 2, 64), device=gpu).to(BF)
    for scale in (2.0 ** 127, -(2.0 ** 127)):
        got, want, tol = _both(ge, q, keys, values, None, table, [40], [1], scale=scale)
        assert (np.abs(got - want) <= tol).all()
    lib, kv = ge._lib, ge.kv
    c = kv._CACHE.pack(kv._CACHE.size, lib.K_BF16, 1, 1, 1, 8, 0, 0, 8, 8, 8, *[0] * 5)
    for scale, ok in ((2.0 ** 127, True), (3e38, False), (-3e38, False), (float("inf"), False), (float("nan"), False)):
        a = kv._ATTEND.pack(kv._ATTEND.size, 1, 1, 1, lib.K_BF16, 1, *[0] * 6, 1, scale, *[0] * 7)
        if ok:
            assert lib.handle(gpu.index, 1, 1).call("gsk_attention_work", c, a) >= 0
            continue
        with pytest.raises(RuntimeError, match="scale"):
            lib.handle(gpu.index, 1, 1).call("gsk_attention_work", c, a)
