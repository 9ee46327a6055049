"""Commits of verify rounds on the GPU (spec.VerifyCall.commit, spec.Chains.commit) where a step could not serve every request:
lengths, tables and queues against the oracle's bookkeeping, whole numbers compared exactly."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import round_ref as rr

pytestmark = pytest.mark.gpu


def _same(t, ref, m, want):
    for name, x in (("begin", m.begin), ("slot", m.slot), ("pos", m.pos), ("req", m.req), ("seq", m.seq_len), ("status", m.status)):
        assert x.cpu().tolist() == [int(k) for k in want[name]], name
    c, r = t.counters.cpu().tolist(), t.requests
    assert c[2:2 + r] == ref.length and c[2 + r:] == [len(p) for p in ref.pages]
    ring, table = t.ring.cpu().tolist(), t.table.cpu().tolist()
    assert c[1] == len(ref.free) and [ring[(c[0] + i) % len(ring)] for i in range(c[1])] == list(ref.free)
    assert [table[k][:len(p)] for k, p in enumerate(ref.pages)] == ref.pages
    ref.check()


# (three requests of one page each out of four; then request 1's tokens do not fit, or request 1's numbers are out of range)
CASES = [("full", [3, 14, 4], 1), ("bad", [3, 3, 4], 2)]


def _tables(ge, gpu, add, bad):
    t, ref = ge.paged.PageTable(3, 4, 8, 3, device=gpu), rr.Pages(3, 4, 8, 3)
    _same(t, ref, t.step([4, 5, 6]), ref.step([4, 5, 6]))
    keep = [2, 40 if bad else 5, 1]
    m, want = t.step(add, keep=keep), ref.step(add, keep)
    _same(t, ref, m, want)
    return t, ref, m, want


@pytest.mark.parametrize("ends", [None, [False, True, True]])
@pytest.mark.parametrize("name,add,status", CASES)
def test_trees_after_a_step_that_served_not_every_request(ge, gpu, name, add, status, ends):
    t, ref, m, want = _tables(ge, gpu, add, name == "bad")
    assert want["status"] == [0, status, 0]
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn((sum(add), 300), generator=g, device=gpu)
    best = x.argmax(1).cpu().tolist()
    at = np.concatenate([[0], np.cumsum(add)])
    reqs = [dict(target=x[at[k]:at[k + 1]], parents=list(range(add[k] - 1)), params=ge.sampling.SamplingParams(), seed=1,
                 tokens=best[at[k]:at[k + 1] - 1]) for k in range(3)]  # (every draft accepted)
    call = ge.spec.VerifyCall(reqs)
    call.launch()
    assert call.e_len.cpu().tolist() == add
    c = torch.arange(2 * 4 * 8 * 16, device=gpu).reshape(2, 4, 8, 16).float()
    was = c.clone()
    nxt = call.commit(m, t, c, [1, 1, 1], ends=ends)
    keep = [add[0], 0, add[2]] if ends is None else [add[0], -1, -1]
    _same(t, ref, nxt, ref.step([1, 1, 1], keep))
    assert torch.equal(c, was)  # (chains: nothing moves)


@pytest.mark.parametrize("ends", [None, [False, True, True]])
@pytest.mark.parametrize("name,add,status", CASES)
def test_chains_after_a_step_that_served_not_every_request(ge, gpu, name, add, status, ends):
    t, ref, m, want = _tables(ge, gpu, add, name == "bad")
    assert want["status"] == [0, status, 0]
    drafts = [k - 1 for k in add]
    p = torch.softmax(torch.randn((sum(add), 300), device=gpu, generator=torch.Generator(device=gpu).manual_seed(3)), 1)
    o = ge.spec.verify_chains(p, [7] * sum(drafts), np.concatenate([[0], np.cumsum(drafts)]), [0.0] * sum(drafts), [0.5] * 3)
    assert o.emit_len.cpu().tolist() == add  # (a coin of zero takes every draft)
    nxt = o.commit(t, [1, 1, 1], ends=ends, step=m)
    keep = [add[0], 0, add[2]] if ends is None else [add[0], -1, -1]
    _same(t, ref, nxt, ref.step([1, 1, 1], keep))


def test_a_dry_pool_commits_nothing_round_after_round(ge, gpu):
    """A request that no page is left for keeps its length over rounds until another ends, as the loop runs: one step from the
    next, nothing read back."""
    t, ref = ge.paged.PageTable(2, 4, 4, 4, device=gpu), rr.Pages(2, 4, 4, 4)
    m, want = t.step([4, 8]), ref.step([4, 8])
    lens = [4, 8]
    p = torch.softmax(torch.randn((8, 99), device=gpu, generator=torch.Generator(device=gpu).manual_seed(4)), 1)
    o = None
    for rnd in range(6):
        ends, add = [rnd >= 3, False], [4 if rnd < 3 else 0, 4]
        if o is None:
            m, want = t.step(add, keep=lens), ref.step(add, lens)
        else:
            m = o.commit(t, add, ends=ends, step=m)
            keep = [-1 if e else n if s == 0 else 0 for e, n, s in zip(ends, lens, want["status"])]
            want = ref.step(add, keep)
        _same(t, ref, m, want)
        o = ge.spec.verify_chains(p, [1] * 6, [0, 3, 6], [0.0] * 6, [0.5] * 2)
        lens = o.emit_len.cpu().tolist()
    assert ref.length == [0, 12]


def test_a_refused_commit_leaves_caches_and_books(ge, gpu):
    """Whatever a commit refuses, the one made after it moves each path once."""
    t = ge.paged.PageTable(2, 12, 4, 4, device=gpu)
    u = ge.paged.PageTable(2, 12, 4, 4, device=gpu)
    parents = [[0, 0, 2, 3], [0]]
    sizes = [5, 2]
    x = torch.randn((7, 200), device=gpu, generator=torch.Generator(device=gpu).manual_seed(6))
    best = x.argmax(1).cpu().tolist()
    toks = [[(best[0] + 1) % 200, best[0], best[2], best[3]], [(best[5] + 1) % 200]]  # (the path 0, 2, 3, 4; and 0 alone)
    at = [0, 5]
    call = ge.spec.VerifyCall([dict(target=x[at[k]:at[k] + sizes[k]], parents=parents[k], tokens=toks[k], seed=1,
                                    params=ge.sampling.SamplingParams()) for k in range(2)])
    call.launch()
    assert call.e_len.cpu().tolist() == [4, 1]
    c = torch.arange(2 * 12 * 4 * 8, device=gpu).reshape(2, 12, 4, 8).float()
    d = c.clone()
    m, n = t.step(sizes), u.step(sizes)
    was, books = c.clone(), t.counters.clone()
    for kw in (dict(add=torch.ones(2, dtype=torch.int32, device=gpu)), dict(add=torch.ones(2), max_tokens=2), dict(add=[1]),
               dict(add=[1, 1], depth=torch.zeros(2)), dict(add=[1, 1], ends=[True]), dict(add=[1, 1], caches=c.cpu()),
               dict(add=[1, 1], caches=c[0, 0])):
        with pytest.raises((ValueError, RuntimeError)):
            call.commit(m, t, **{"caches": c, **kw})
        assert torch.equal(c, was) and torch.equal(t.counters, books)
    call.commit(m, t, c, [1, 1])
    call.keep_path(n, d)
    u.step([1, 1], keep=call.e_len)
    assert not torch.equal(c, was) and torch.equal(c, d) and torch.equal(t.counters, u.counters)


@pytest.mark.parametrize("room", [None, 3])
def test_an_end_whose_successor_does_not_fit_gives_its_pages_back(ge, gpu, room):
    """No pages left for it, a full table row, or (room) past the map's end: the ended request holds nothing after the step, in
    place and into other counters, and the next step has its pages."""
    for most, add in ((11, [44, 4]), (10, [41, 0])):
        t, ref = ge.paged.PageTable(2, 10, 4, most, device=gpu), rr.Pages(2, 10, 4, most)
        _same(t, ref, t.step([24, 16]), ref.step([24, 16]))
        keep, into = [-1, 16], torch.zeros_like(t.counters)
        n = sum(add) if room is None else room
        tried = t.step(add, keep=keep, max_tokens=n, into=into)
        m, want = t.step(add, keep=keep, max_tokens=n), ref.step(add, keep, None, n)
        _same(t, ref, m, want)
        assert want["status"][0] == 1 and torch.equal(into, t.counters) and torch.equal(tried.slot, m.slot)
        assert t.held.tolist()[0] == 0 and t.free.item() == 6
        _same(t, ref, t.step([20, 4]), ref.step([20, 4]))


@pytest.mark.parametrize("r", [3, 300, 1500])
def test_ends_in_a_dry_pool(ge, gpu, r):
    """Many steps over a pool that stays dry, half the requests ending in each, their successors of any length."""
    t, ref = ge.paged.PageTable(r, 3 * r, 4, 9, device=gpu), rr.Pages(r, 3 * r, 4, 9)
    rng = np.random.default_rng(r)
    kept_to, freed = np.zeros(r, np.int64), 0
    for k in range(10):
        keep = np.where(rng.random(r) < 0.5, -1, np.minimum(rng.integers(0, 5, r), kept_to))
        add = rng.integers(0, 42, r)
        held = [len(p) for p in ref.pages]
        m, want = t.step(add, keep=keep), ref.step(add, keep)
        _same(t, ref, m, want)
        kept_to = np.where(np.array(want["status"]) == 0, add, 0)
        freed += sum(held[i] for i in range(r) if keep[i] < 0 and want["status"][i] == 1)
    assert freed > 0


@pytest.mark.parametrize("anchor", [-1, -2, -(2 ** 31)])
@pytest.mark.parametrize("depth", [4, 70])
def test_a_request_without_an_anchor_moves_nothing(ge, gpu, anchor, depth):
    """A padded request's anchor is negative: the places after it are other requests' (entry -anchor's is place 0)."""
    c = torch.arange(2 * 40 * 4 * 8, device=gpu).reshape(2, 40, 4, 8).float()
    slot = torch.arange(160, device=gpu)
    nodes = torch.arange(80, 80 + 2 * depth, device=gpu).reshape(2, depth).int() % 160
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    want = c.clone()
    ge.paged.keep_path(c, slot, i32(anchor, anchor), i32(depth, 3), nodes)
    assert torch.equal(c, want)
    ge.paged.keep_path(c, slot, i32(anchor, 3), i32(depth, 3), nodes)  # (a request beside it still moves)
    rows = want.view(2, 160, 8)
    rows[:, 4:6] = rows[:, nodes[1, 1:3].long()].clone()
    assert torch.equal(c, want)


@pytest.mark.parametrize("r", [5, 700, 1300])
def test_keep_of_a_step_that_served_not_every_request(ge, gpu, r):
    """PageTable.step(of=): what counts as kept is masked by that step's status, in place and into other counters."""
    t, ref = ge.paged.PageTable(r, 2 * r, 4, 4, device=gpu), rr.Pages(r, 2 * r, 4, 4)
    rng = np.random.default_rng(r)
    add = rng.integers(0, 18, r)
    m, want = t.step(add), ref.step(add)
    _same(t, ref, m, want)
    seen = set()
    for k in range(8):
        keep = np.where(rng.random(r) < 0.3, -1, rng.integers(0, 5, r))
        nxt, laid = rng.integers(0, 9, r), want["status"]
        into = torch.zeros_like(t.counters)
        tried = t.step(nxt, keep=keep, into=into, of=m)
        m = t.step(nxt, keep=keep, of=m)
        want = ref.step(nxt, keep, laid=laid)
        _same(t, ref, m, want)
        assert torch.equal(into, t.counters) and torch.equal(tried.slot, m.slot)
        seen |= set(laid)
    assert seen == {0, 1, 2} or r == 5


def test_the_steps_own_status_is_not_the_one_before(ge, gpu):
    lib = ge._lib
    t = ge.paged.PageTable(2, 8, 4, 4, device=gpu)
    add = torch.zeros(2, dtype=torch.int32, device=gpu)
    out = torch.full((16,), -7, dtype=torch.int64, device=gpu)
    p = lib.Pages(C.sizeof(lib.Pages), 2, 4, 8, 4, 0, t.table.data_ptr(), 4, t.ring.data_ptr(), t.counters.data_ptr(),
                  t.counters.data_ptr())
    s = lib.Step(C.sizeof(lib.Step), 0, None, add.data_ptr(), None, out.data_ptr(), None, None, None, out.data_ptr(),
                 out.data_ptr(), torch.cuda.current_stream().cuda_stream, out.data_ptr())
    with pytest.raises(RuntimeError, match="another step"):
        lib.device_handle(gpu.index).call("gsp_pages_step", C.byref(p), C.byref(s))
    torch.cuda.synchronize()
    assert (out == -7).all()
