"""GPU parity of beam.select against the oracle's full sort in 64 bits.

A score may be off by its rounding to fp32 and by the log of a row's sum: its many small terms are fp32 (1 ulp of exp, the
argument's roundings, a chain of at most 33 additions: below 40 * 2^-24 = 2.4e-6 of the sum), so tokens of different beams whose
scores are closer than LSE may come in either order; anything else is in the oracle's order."""
import numpy as np
import pytest
import torch

from oracle import kv_ref as kr

pytestmark = pytest.mark.gpu
LSE = 2.4e-6


def _check(o, logits, scores, n):
    x, s = kr._np(logits), kr._np(scores.float())
    r, b = s.shape
    tokens, parents, got = o.tokens.cpu().numpy(), o.parents.cpu().numpy(), o.scores.cpu().numpy()
    assert tokens.shape == parents.shape == got.shape == (r, n) and o.scores.dtype is torch.float32
    for i in range(r):
        rows = x[i * b:(i + 1) * b]
        want = kr.beams(rows, s[i], n + 8)
        near = [k for k in range(len(want) - 1) if want[k][1] != want[k + 1][1] and want[k][2] - want[k + 1][2] <= 2 * LSE]
        loose = {k for k in near} | {k + 1 for k in near}
        for k in range(n):
            if k >= len(want):
                assert (tokens[i, k], parents[i, k], got[i, k]) == (-1, -1, -np.inf)
                continue
            t, p, v = want[k]
            assert abs(got[i, k] - v) <= LSE + abs(v) * 2.0 ** -24, (i, k, got[i, k], v)
            if k not in loose:
                assert (tokens[i, k], parents[i, k]) == (t, p), (i, k)
        assert len({(int(t), int(p)) for t, p in zip(tokens[i], parents[i]) if t >= 0}) == min(n, len(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("requests,beams,n,vocab", [(1, 1, 1, 1), (1, 1, 8, 5), (3, 4, 8, 8191), (2, 5, 64, 8193), (1, 4, 8, 128256),
                                                    (5, 3, 6, 50257), (1, 32, 64, 20000), (2, 8, 16, 32000), (40, 2, 4, 1000)])
def test_select(ge, gpu, dtype, requests, beams, n, vocab):
    g = torch.Generator(device=gpu).manual_seed(vocab + n)
    x = (torch.randn((requests * beams, vocab), generator=g, device=gpu) * 3).to(dtype)
    s = -torch.rand((requests, beams), generator=g, device=gpu) * 8
    _check(ge.beam.select(x, s, n), x, s, n)


@pytest.mark.parametrize("vocab", [700, 9001, 40000])
def test_ties(ge, gpu, vocab):
    """Rows of few values, rows of one value, beams alike: the lower beam, then the lower token; more ties than a list holds."""
    g = torch.Generator(device=gpu).manual_seed(vocab)
    x = torch.randint(0, 3, (12, vocab), generator=g, device=gpu).float()
    x[4:8] = 1.5
    x[8:12] = torch.randn(vocab, generator=g, device=gpu).bfloat16().float()
    s = torch.tensor([[-1.0, -2.0, -1.0, -1.5], [-3.0] * 4, [-2.0, -2.0, -2.0, -2.0]], device=gpu)
    for n in (1, 8, 64):
        _check(ge.beam.select(x, s, n), x, s, n)
        _check(ge.beam.select(x.bfloat16(), s, n), x, s, n)


def test_sorted_rows(ge, gpu):
    """Rows that ascend or descend by token, and one slice that holds every large token."""
    v = 30000
    x = torch.linspace(-20, 20, v, device=gpu).repeat(6, 1)
    x[1], x[2] = x[0].flip(0), 0
    x[2, 9000:9100] = torch.linspace(5, 6, 100, device=gpu)
    x[3, 16384:16384 + 2000] = 30 + torch.arange(2000, device=gpu) * 0.001
    s = -torch.arange(6, device=gpu).float().reshape(2, 3)
    for n in (3, 64):
        _check(ge.beam.select(x, s, n), x, s, n)


def test_masks_and_bad_rows(ge, gpu):
    """-inf everywhere but a few tokens, NaN, +inf, beams without a score: what is left, then -1."""
    v, inf, nan = 20000, float("inf"), float("nan")
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.full((16, v), -inf, device=gpu)
    x[0, [3, 9000, 19999]] = torch.tensor([1.0, 2.0, 3.0], device=gpu)
    x[1] = torch.randn(v, generator=g, device=gpu)
    x[1, ::2] = nan
    x[2] = torch.randn(v, generator=g, device=gpu)
    x[2, 777] = inf
    x[4:8] = torch.randn((4, v), generator=g, device=gpu)
    x[8, 5] = -3.4028234663852886e38
    x[9] = -3.4028234663852886e38
    x[10] = 3.4028234663852886e38
    x[12:14] = nan
    x[15, 0] = 0
    s = torch.tensor([[0.0, -1, 0, 0], [-inf, nan, inf, -2], [-1, -1, -1, 0], [0, 0, 0, -7]], device=gpu)
    for n in (1, 5, 64):
        for dtype in (torch.float32, torch.bfloat16):
            _check(ge.beam.select(x.to(dtype), s, n), x.to(dtype), s, n)
    assert ge.beam.select(x[12:15], torch.zeros((1, 3), device=gpu), 2).tokens.tolist() == [[-1, -1]]


def test_strides_and_types(ge, gpu):
    """Logits inside wider rows, at odd offsets, by columns; scores in 64 bits and by columns; no requests."""
    g = torch.Generator(device=gpu).manual_seed(4)
    big = torch.randn((8, 9003), generator=g, device=gpu)
    s = -torch.rand((4, 2), generator=g, device=gpu, dtype=torch.float64).t()
    for x in (big[:, :9000], big[:, 1:8999], big.bfloat16()[:, 3:9001], big[:, ::3], big.half()[:, :512].t().contiguous().t()):
        _check(ge.beam.select(x, s.contiguous() if x.shape[1] == 9000 else s, 6), x, s, 6)
    assert ge.beam.select(big[:0], s[:0], 6).tokens.shape == (0, 6)


def test_calls_share_a_stream(ge, gpu):
    """Many calls of several sizes without a wait between them, and a captured one replayed with eager calls between."""
    g = torch.Generator(device=gpu).manual_seed(5)
    cases = [(torch.randn((r * b, v), generator=g, device=gpu), -torch.rand((r, b), generator=g, device=gpu), n)
             for r, b, n, v in ((3, 4, 8, 30000), (1, 8, 16, 100000), (50, 2, 4, 9000))]
    got = [ge.beam.select(*c) for _ in range(3) for c in cases]
    for i, o in enumerate(got):
        _check(o, *cases[i % 3])
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ge.beam.select(*cases[0])
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        o = ge.beam.select(*cases[0])
    for k in range(3):
        cases[0][0].copy_(torch.randn(cases[0][0].shape, generator=g, device=gpu))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _check(o, *cases[0])
        with torch.cuda.stream(stream):
            _check(ge.beam.select(*cases[1]), *cases[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("far", [16.875, 12.5, 9.0])
@pytest.mark.parametrize("peaks,n", [(1, 1), (1, 4), (3, 1), (40, 2), (700, 64), (2000, 8)])
def test_sums_of_peaked_rows(ge, gpu, dtype, far, peaks, n):
    """A few tokens (or more than a list holds) at 0 and a hundred thousand others far below, all alike or spread out: a row's sum is
    off by its far terms' own errors, never by what adding them to the large ones costs. Of each term below the listed ones, with t
    its distance from the maximum: t's rounding and its product's with log2 e, 2^-24 |t| each, and exp2's, 2^-23; so 2^-24 (2 |t| + 4)
    of it is allowed. Terms at the maximum itself are exact."""
    v = 128256
    g = torch.Generator(device=gpu).manual_seed(peaks)
    x = torch.full((4, v), -far, device=gpu)
    x[1] -= torch.rand(v, generator=g, device=gpu) * 4
    x[3] = 50 - far
    for i in range(4):
        x[i, torch.randperm(v, generator=g, device=gpu)[:peaks]] = 50.0 if i == 3 else 0.0
    x = x.to(dtype)
    s = torch.tensor([[0.0, -0.25, -0.5, -0.75]], device=gpu)
    for rows in ([0], [1], [2], [3], [0, 1, 2, 3]):
        o = ge.beam.select(x[rows], s[:, :len(rows)].contiguous(), n)
        xs = kr._np(x[rows])
        t = xs.max(1, keepdims=True) - xs
        w = np.exp(-t)
        lse = xs.max(1) + np.log(w.sum(1))
        near = [np.flatnonzero(z >= np.partition(z, -n)[-n]).tolist() for z in xs]
        want = sorted((lse[b] - xs[b, i] + 0.25 * b, b, i) for b in range(len(rows)) for i in near[b])[:n]
        tol = ((w * (2 * t + 4) * 2.0 ** -24 * (t > 0)).sum(1) / w.sum(1)).max()
        got = o.scores.cpu().numpy()[0]
        for k, (less, beam, token) in enumerate(want):
            score = -less
            assert abs(float(got[k]) - score) <= tol + abs(score) * 2.0 ** -24 + 1e-11, (rows, k, float(got[k]) - score, tol)
            assert (int(o.tokens[0, k]), int(o.parents[0, k])) == (token, beam), (rows, k)


def test_close_beams_in_order(ge, gpu):
    """Beams whose rows have one peak, in the first slice or the last, and whose far tokens are a few more or fewer: their order is that
    of their sums, whose differences (9e-8 and more) are above their errors (2^-24 * 38 of the far terms' 0.0059, 1.4e-8)."""
    v = 128256
    x = torch.full((4, v), -16.875, device=gpu)
    for i, (cut, peak) in enumerate([(0, 5), (4, 124240), (2, 5), (6, 124240)]):
        x[i, 100:100 + cut] = -float("inf")
        x[i, peak] = 0
    o = ge.beam.select(x, torch.zeros((1, 4), device=gpu), 4)
    assert o.parents.tolist() == [[3, 1, 2, 0]] and o.tokens.tolist() == [[124240, 124240, 5, 5]]
