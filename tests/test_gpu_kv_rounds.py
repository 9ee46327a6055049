"""The paged cache's operators as a program runs them: rounds of draft trees over a cache in 8 bits (step, write, attend, the accepted
path moved with its scales), beams over a cache (step, write, attend, select, reorder), whole rounds in a captured graph, two
streams at once. The reference keeps every request's tokens as a list and attends to them in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import kv_ref as kr

pytestmark = pytest.mark.gpu
BF, E4, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8
HEADS, GROUP, DIM = 2, 4, 64


class Toy:
    """One layer whose keys, values and queries are rows of tables by token id."""

    def __init__(self, gpu, vocab=97, seed=0):
        g = torch.Generator(device=gpu).manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
        self.k, self.v = r(vocab, HEADS, DIM).to(BF), r(vocab, HEADS, DIM).to(BF)
        self.q = r(vocab, HEADS * GROUP, DIM).to(BF)
        self.out = r(HEADS * GROUP * DIM, vocab)

    def held(self, cache):
        """What a cache of this type holds of the tables, float64."""
        k, v = kr._np(self.k), kr._np(self.v)
        if cache is BF:
            return k, v
        (k, ks), (v, vs) = kr.to_8(k, cache), kr.to_8(v, cache)
        return k * ks.astype(np.float64)[..., None], v * vs.astype(np.float64)[..., None]


def _new_cache(gpu, cache, pages, page, first):
    """Two stacked arrays, keys and values, and their scales, so that one call moves both."""
    shape = (2, pages, HEADS, page) if first else (2, pages, page, HEADS)
    data = torch.zeros((*shape, DIM), device=gpu).to(cache)
    scales = torch.zeros((*shape, 1), device=gpu) if cache is not BF else None
    return data, scales


def _pair(scales):
    return None if scales is None else (scales[0, ..., 0], scales[1, ..., 0])


def _attended(toy, held, tokens, history, mask, cache):
    """Queries of `tokens` over the history (token ids): the oracle's answer and its bound."""
    k, v = (x[np.array(history, np.int64)].reshape(len(history), HEADS, DIM) for x in held)
    return kr.attend(kr._np(toy.q[torch.tensor(tokens, device=toy.q.device)]), k, v, mask, float(np.float32(DIM ** -0.5)), BF, cache is not BF)


@pytest.mark.parametrize("cache,first,page", [(BF, False, 16), (E4, True, 8), (I8, False, 5)])
def test_rounds_of_trees(ge, gpu, cache, first, page):
    toy, rng = Toy(gpu), np.random.default_rng(page)
    held = toy.held(cache)
    r, rounds = 4, 6
    pages = ge.paged.PageTable(r, 60, page, 30, device=gpu)
    data, scales = _new_cache(gpu, cache, 60, page, first)
    lists = [list(rng.integers(0, 97, n)) for n in (7, 23, 1, 40)]

    def run(step, tokens, parents, most):
        ids = torch.tensor(tokens, device=gpu)
        ge.kv.write(step.slot, toy.k[ids], toy.v[ids], data[0], data[1], scales=_pair(scales), heads_first=first)
        return ge.kv.attend(toy.q[ids], data[0], data[1], pages.table, step.seq_len, begin=step.begin, status=step.status,
                            parents=parents, max_new=most, scales=_pair(scales), heads_first=first)

    step = pages.step([len(x) for x in lists])
    o = kr._np(run(step, sum(lists, []), None, 40))
    at = 0
    for x in lists:
        want, tol = _attended(toy, held, x, x, kr.sees(len(x), 0), cache)
        assert (np.abs(o[at:at + len(x)] - want) <= tol).all()
        at += len(x)
    keep = torch.tensor([len(x) for x in lists], dtype=torch.int32, device=gpu)
    for k in range(rounds):
        sizes = rng.integers(1, 12, r)
        begin = np.concatenate([[0], np.cumsum(sizes)])
        par = [-1 if i == 0 else int(begin[a] + rng.integers(0, i)) for a in range(r) for i in range(sizes[a])]
        toks = rng.integers(0, 97, begin[-1]).tolist()
        step = pages.step(sizes.tolist(), keep=keep, max_tokens=int(begin[-1]))
        assert step.status.tolist() == [0] * r
        o = kr._np(run(step, toks, torch.tensor(par, dtype=torch.int32, device=gpu), 12))
        nodes = np.full((r, 12), -1, np.int32)
        for a in range(r):
            mine = toks[begin[a]:begin[a + 1]]
            mask = kr.sees(int(sizes[a]), len(lists[a]), par, begin[a])
            want, tol = _attended(toy, held, mine, lists[a] + mine, mask, cache)
            assert (np.abs(o[begin[a]:begin[a + 1]] - want) <= tol).all(), (k, a)
            path, node = [], int(begin[a] + rng.integers(0, sizes[a]))
            while node >= 0:
                path.append(node)
                node = par[node]
            nodes[a, :len(path)] = path[::-1]
            lists[a] = lists[a] + [toks[i] for i in path[::-1]]
        lens = torch.from_numpy((nodes >= 0).sum(1).astype(np.int32)).to(gpu)
        anchor, e_nodes = torch.from_numpy(begin[:-1].astype(np.int32)).to(gpu), torch.from_numpy(nodes).to(gpu)
        ge.paged.keep_path(data, step.slot, anchor, lens, e_nodes, heads_first=first)
        if scales is not None:
            ge.paged.keep_path(scales, step.slot, anchor, lens, e_nodes, heads_first=first)
        keep = lens
    # what is cached is the lists, read back
    step = pages.step([0] * r, keep=keep)
    begin = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    assert step.seq_len.tolist() == [len(x) for x in lists]
    k, v = ge.kv.read(data[0], data[1], pages.table, begin, scales=_pair(scales), dtype=torch.float32, heads_first=first)
    ids = np.array(sum(lists, []))
    assert np.abs(kr._np(k) - held[0][ids]).max() <= 2 ** -22 * np.abs(held[0]).max()
    assert np.abs(kr._np(v) - held[1][ids]).max() <= 2 ** -22 * np.abs(held[1]).max()


def test_a_request_without_pages(ge, gpu):
    """A step that a request's pages ran out in: nothing is written for it and its rows are zero, the others' are right."""
    toy = Toy(gpu)
    pages = ge.paged.PageTable(3, 6, 4, 4, device=gpu)
    data, _ = _new_cache(gpu, BF, 6, 4, False)
    lists = [[1, 2, 3, 4, 5], [6] * 17, [7, 8]]
    step = pages.step([5, 17, 2], max_tokens=30)
    assert step.status.tolist() == [0, ge._lib.STEP_FULL, 0]
    ids = torch.tensor(sum(lists, []) + [0] * 6, device=gpu)
    ge.kv.write(step.slot, toy.k[ids], toy.v[ids], data[0], data[1])
    out = torch.full((30, HEADS * GROUP, DIM), 3.0, dtype=BF, device=gpu)
    ge.kv.attend(toy.q[ids], data[0], data[1], pages.table, step.seq_len, begin=step.begin, status=step.status, max_new=17, out=out)
    o, held = kr._np(out), toy.held(BF)
    assert (o[5:22] == 0).all() and (o[24:] == 3).all()
    for a, x in ((0, lists[0]), (22, lists[2])):
        want, tol = _attended(toy, held, x, x, kr.sees(len(x), 0), BF)
        assert (np.abs(o[a:a + len(x)] - want) <= tol).all()
    assert int((data[0] != 0).any(-1).any(-1).sum()) == 7


@pytest.mark.parametrize("cache,first,beams,page", [(BF, False, 4, 8), (E4, True, 3, 16)])
def test_beam_search(ge, gpu, cache, first, beams, page):
    """Beams that each hold their own pages: every step's attention against the beams' token lists, the selection against the
    oracle's on the same logits, the caches after the reorder."""
    toy = Toy(gpu, seed=3)
    held, requests, prompt = toy.held(cache), 2, [[5, 9, 11], [40, 41, 42, 43, 44, 45, 46, 47, 48]]
    rows = requests * beams
    pages = ge.paged.PageTable(rows, 40, page, 5, device=gpu)
    data, scales = _new_cache(gpu, cache, 40, page, first)
    lists = [list(prompt[r]) for r in range(requests) for _ in range(beams)]
    scores = torch.full((requests, beams), -float("inf"), device=gpu)
    scores[:, 0] = 0
    step = pages.step([len(x) for x in lists])
    new = [list(x) for x in lists]
    for k in range(8):
        ids = torch.tensor(sum(new, []), device=gpu)
        ge.kv.write(step.slot, toy.k[ids], toy.v[ids], data[0], data[1], scales=_pair(scales), heads_first=first)
        o = ge.kv.attend(toy.q[ids], data[0], data[1], pages.table, step.seq_len, begin=step.begin, max_new=9, scales=_pair(scales),
                         heads_first=first)
        last = torch.tensor(np.cumsum([len(x) for x in new]) - 1, device=gpu)
        for b in range(rows):
            want, tol = _attended(toy, held, lists[b][-1:], lists[b], np.ones((1, len(lists[b])), bool), cache)
            assert (np.abs(kr._np(o[last[b]])[None] - want) <= tol).all(), (k, b)
        logits = o[last].float().reshape(rows, -1) @ toy.out
        best = ge.beam.select(logits, scores, beams)
        s = kr._np(scores)
        for r in range(requests):
            want = kr.beams(kr._np(logits[r * beams:(r + 1) * beams]), s[r], beams)
            assert [(int(t), int(p)) for t, p in zip(best.tokens[r], best.parents[r])] == [w[:2] for w in want], (k, r)
        ge.kv.reorder(data, pages.table, step.seq_len, best.parents, first=[len(p) for p in prompt], heads_first=first)
        if scales is not None:
            ge.kv.reorder(scales, pages.table, step.seq_len, best.parents, first=[len(p) for p in prompt], heads_first=first)
        parents, tokens = best.parents.cpu().numpy(), best.tokens.cpu().numpy()
        lists = [lists[r * beams + parents[r, b]] + [int(tokens[r, b])] for r in range(requests) for b in range(beams)]
        step = pages.step([1] * rows, keep=[len(x) for x in new])
        new, scores = [x[-1:] for x in lists], best.scores


@pytest.mark.parametrize("cache", [BF, E4])
def test_rounds_in_a_graph(ge, gpu, cache):
    """A decode step (books, write, attention) captured once and replayed as successive steps, with eager calls of the same stream's
    handle between the replays; the same steps made eagerly give the same bits."""
    toy = Toy(gpu)
    r, page = 5, 16
    start = [300, 2000, 1, 77, 16]
    s = torch.cuda.Stream(gpu)

    def fresh():
        pages = ge.paged.PageTable(r, 400, page, 140, device=gpu)
        data, scales = _new_cache(gpu, cache, 400, page, False)
        step = pages.step(start)
        ids = torch.arange(sum(start), device=gpu) * 31 % 97
        ge.kv.write(step.slot, toy.k[ids], toy.v[ids], data[0], data[1], scales=_pair(scales))
        return pages, data, scales

    def one(pages, data, scales, ids, keep, add):
        step = pages.step(add, keep=keep, max_tokens=r)
        ge.kv.write(step.slot, toy.k[ids], toy.v[ids], data[0], data[1], scales=_pair(scales))
        return ge.kv.attend(toy.q[ids], data[0], data[1], pages.table, step.seq_len, begin=step.begin, status=step.status, max_new=1,
                            scales=_pair(scales))

    steps = [torch.randint(0, 97, (r,), device=gpu) for _ in range(5)]
    keeps = [torch.tensor(start if k == 0 else [1] * r, dtype=torch.int32, device=gpu) for k in range(5)]
    add = torch.ones(r, dtype=torch.int32, device=gpu)
    state = fresh()
    want = [one(*state, i, k, add).clone() for i, k in zip(steps, keeps)]
    state = fresh()
    big = torch.randn((3000, 2 * GROUP, DIM), device=gpu).to(BF)
    ids, keep = steps[0].clone(), keeps[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        other = fresh()
        one(*other, ids, keep, add)  # (opens the stream's handle)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = one(*state, ids, keep, add)
        for k in range(5):
            ids.copy_(steps[k])
            keep.copy_(keeps[k])
            graph.replay()
            assert torch.equal(out, want[k]), k
            ge.kv.attend(big, other[1][0], other[1][1], other[0].table[:1].contiguous(), [2200], begin=[0, 2000],
                         max_new=2000, scales=_pair(other[2]))
            ge.beam.select(torch.randn((4, 5000), device=gpu), torch.zeros((1, 4), device=gpu), 8)
    torch.cuda.synchronize()
    del graph
    ge._lib.release_captured()


def test_a_capture_without_a_handle_is_refused(ge, gpu):
    """attend and select on a stream that no handle is open for: refused, and the capture goes on."""
    toy = Toy(gpu)
    data, _ = _new_cache(gpu, BF, 8, 16, False)
    table = torch.arange(8, dtype=torch.int32, device=gpu)[None]
    s, x = torch.cuda.Stream(gpu), torch.zeros(4, device=gpu)
    n, ids = torch.tensor([100], dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int64, device=gpu)
    logits, scores = torch.randn((2, 50), device=gpu), torch.zeros((1, 2), device=gpu)
    q = toy.q[ids]
    torch.cuda.synchronize()
    ge._lib._handles.pop((gpu.index, s.cuda_stream), None)  # (streams come from a pool)
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            x.add_(1)
            with pytest.raises(RuntimeError, match="before the capture"):
                ge.kv.attend(q, data[0], data[1], table, n)
            with pytest.raises(RuntimeError, match="before the capture"):
                ge.beam.select(logits, scores, 2)
        graph.replay()
        s.synchronize()
        assert x.tolist() == [1.0] * 4
        assert ge.kv.attend(q, data[0], data[1], table, n).shape == q.shape


def test_two_streams_at_once(ge, gpu):
    """Calls in flight on two streams do not meet: each has its own tickets and scratch memory."""
    toy = Toy(gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    pages, page = 700, 16
    data, _ = _new_cache(gpu, BF, pages, page, False)
    data.copy_(torch.randn(data.shape, generator=g, device=gpu))
    table = torch.randperm(pages, generator=g, device=gpu).int().reshape(2, 350)
    q = toy.q[torch.arange(12, device=gpu)]
    args = [([5000, 5600], [0, 4, 12]), ([5600, 17], [0, 11, 12])]
    logits = [torch.randn((8, 60000), generator=g, device=gpu) for _ in range(2)]
    scores = torch.zeros((2, 4), device=gpu)

    def one(i):
        n, b = args[i]
        c = ge.beam.select(logits[i], scores, 8)
        return ge.kv.attend(q, data[0], data[1], table, n, begin=b, max_new=11), c.tokens, c.scores

    want = [one(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    got = [[], []]
    for k in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(one(i))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))
