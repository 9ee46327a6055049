"""NaNs and infinities in attention: which results they reach, whatever the cut of the work and the weights of their tokens."""
import numpy as np
import pytest
import torch

from oracle import kv_ref as kr
from test_gpu_kv import BF, E4, HF, I8, _cache, _gen, _pages, _rand

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _poison(ge, keys, values, scales, table, r, t, value, first_head=1, element=3):
    """Token t of request r written anew, with a value row of ones in all heads but `first_head`, that has `value` in it."""
    page, heads, dim = keys.shape[1:]
    row = torch.ones((1, heads, dim), device=keys.device)
    row[0, first_head, element] = value
    at = (table[r, t // page].long(), t % page)
    was = values[at].clone(), None if scales is None else scales[1][at].clone()
    if scales is None:
        values[at] = row[0].to(values.dtype)
    else:
        slot = (at[0] * page + at[1]).reshape(1)
        k, s = keys[at].clone(), scales[0][at].clone()
        ge.kv.write(slot, row, row, keys, values, scales=scales)
        keys[at], scales[0][at] = k, s
    return at, was


def _undo(values, scales, at, was):
    values[at] = was[0]
    if scales is not None:
        scales[1][at] = was[1]


@pytest.mark.parametrize("query,cache", [(BF, BF), (HF, HF), (BF, E4), (HF, I8)])
@pytest.mark.parametrize("shape", ["chain", "star", "random"])
def test_bad_values_of_a_tree_over_two_shares(ge, gpu, query, cache, shape):
    """A request's new tokens lie on both sides of a border of the work's shares (35 blocks of 32 in four: a border at token 320): a
    NaN or an infinity reaches the descendants on the other side too, and no other row."""
    g = _gen(gpu, 41)
    lengths, news = [330, 256], [20, 1]
    rng = np.random.default_rng(3)
    par = np.array([-1] + [i - 1 if shape == "chain" else 0 if shape == "star" else int(rng.integers(max(i - 4, 0), i)) for i in range(1, 20)]
                   + [-1])
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, cache, pages, 16, 2, 64, False)
    q = _rand(g, 21, 2, 64).to(query)
    run = lambda: ge.kv.attend(q, keys, values, table, lengths, begin=[0, 20, 21], parents=par, scales=scales)  # noqa: E731
    clean, sees = run(), kr.sees(20, 0, par, 0)
    for i, value in [(1, INF), (9, NAN), (0, -INF), (10, INF), (19, NAN)]:
        at, was = _poison(ge, keys, values, scales, table, 0, 310 + i, value)
        got = run()
        assert torch.equal(got[20], clean[20])
        for k in range(20):
            a = got[k].float()
            if not sees[k, i]:
                assert torch.equal(got[k], clean[k]), (i, k)
                continue
            assert torch.isfinite(a[0]).all(), (i, k)
            if scales is None:
                assert torch.isfinite(a[1]).sum() == 63 and (torch.isnan(a[1, 3]) if value != value else a[1, 3] == value), (i, k)
            else:
                assert torch.isnan(a[1]).all(), (i, k)
        _undo(values, scales, at, was)
    assert torch.equal(run(), clean)


@pytest.mark.parametrize("query,cache", [(BF, BF), (HF, HF), (BF, E4), (HF, I8)])
def test_bad_values_of_small_weight(ge, gpu, query, cache):
    """A token whose weight is too small for fp32 (its score 320 below the largest) is seen all the same: a NaN or an infinity in
    its value reaches the result, whichever wave or share has it; the other requests and heads have none."""
    g = _gen(gpu, 42)
    lengths, news = [64, 40, 5000, 700], [1, 3, 2, 4]
    begin = np.concatenate([[0], np.cumsum(news)])
    table, pages = _pages(g, lengths, 16)
    keys, values, scales = _cache(g, cache, pages, 16, 2, 64, False)
    if scales is None:
        keys[..., 0] = 0
    else:
        keys.view(torch.int8)[..., 0] = 0
        scales[0].fill_(0.01)
    q = (_rand(g, sum(news), 4, 64) * 0.05).to(query)
    q[..., 0] = 16
    high, scale = (40.0, 0.5) if scales is None else (120.0, 17.0)  # (16 * 40 * 0.5 = 320; 8 bits: 16 * 1.2 * 17 = 326)
    bits = torch.int16 if scales is None else torch.int8
    high = torch.tensor(high, device=gpu).to(cache).view(bits)
    tokens = [(0, 3, [40]), (0, 63, [0]), (1, 5, [33]), (1, 39, [3]), (2, 7, [4000]), (2, 4000, [7]), (3, 699, [2]), (3, 2, [600]),
              (3, 698, [650]), (0, 63, [40]), (1, 33, [36]), (1, 39, [35]), (2, 4995, [4993]), (2, 4999, [4994]), (3, 680, [690])]
    run = lambda: ge.kv.attend(q, keys, values, table, lengths, begin=begin, scales=scales, scale=scale)  # noqa: E731
    for r, t, tops in tokens:
        old = keys.clone()
        for x in tops:
            keys.view(bits)[table[r, x // 16].long(), x % 16, :, 0] = high
        clean = run()
        for value in (NAN, INF):
            at, was = _poison(ge, keys, values, scales, table, r, t, value)
            got = run().float()
            for rr in range(4):
                for k in range(begin[rr], begin[rr + 1]):
                    n = lengths[rr] - news[rr] + k - begin[rr]  # (the last token that it sees)
                    if rr != r or n < t:
                        assert torch.equal(got[k], clean[k].float()), (r, t, rr, k)
                    elif scales is None:
                        assert not torch.isfinite(got[k, 2:, 3]).any() and torch.isfinite(got[k]).sum() == 4 * 64 - 2, (r, t, k, value)
                    else:
                        assert torch.isnan(got[k, 2:]).all() and torch.isfinite(got[k, :2]).all(), (r, t, k, value)
            _undo(values, scales, at, was)
        keys.copy_(old)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 72, 96, 104, 128, 136, 160, 192, 200, 224, 232, 256])
def test_keys_of_minus_infinity(ge, gpu, dtype, dim):
    """A key with -inf in any of its places has the score -inf (its queries are above 0 there): the token has no weight, as if it was
    not there, whatever lies past dim in the registers; where every token is so, the result is 0."""
    g = _gen(gpu, dim)
    lengths, news = [70, 33, 5], [1, 2, 1]
    table, pages = _pages(g, lengths, 16)
    keys, values, _ = _cache(g, dtype, pages, 16, 1, dim, False)
    q = _rand(g, 4, 2, dim).abs().to(dtype) + 0.125
    begin, off = [0, 1, 3, 4], {0: [0, 1, 40, 69], 1: [3, 32], 2: [0, 1, 2, 3, 4]}
    for place in sorted({0, 3, 7, dim // 2, dim - 1}):
        k = keys.clone()
        for r, ts in off.items():
            for t in ts:
                k[table[r, t // 16].long(), t % 16, 0, place] = -INF
        got = kr._np(ge.kv.attend(q, k, values, table, lengths, begin=begin))
        assert (got[3] == 0).all()
        for r in (0, 1):
            kk, there = kr.tokens(keys, None, table[r].tolist(), 0, lengths[r], False)
            vv, _ = kr.tokens(values, None, table[r].tolist(), 0, lengths[r], False)
            mask = kr.sees(news[r], lengths[r] - news[r]) & there
            mask[:, off[r]] = False
            want, tol = kr.attend(kr._np(q[begin[r]:begin[r + 1]]), kk, vv, mask, float(np.float32(dim ** -0.5)), dtype, False)
            assert (np.abs(got[begin[r]:begin[r + 1]] - want) <= tol).all(), (place, r)
