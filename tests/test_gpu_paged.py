"""GPU parity of gsp_pages_step (paged.PageTable.step) and gsp_keep_path (paged.keep_path) against the oracle's bookkeeping,
and rounds of the two with the verify calls. Everything is whole numbers or copies: compared exactly."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import round_ref as rr

pytestmark = pytest.mark.gpu


def _same(t, ref, m, want):
    """A step's map and the state after it against the oracle's."""
    for name, x in (("begin", m.begin), ("slot", m.slot), ("pos", m.pos), ("req", m.req), ("seq", m.seq_len), ("status", m.status)):
        got = x.cpu().numpy()
        assert np.array_equal(got, np.array(want[name], got.dtype)), (name, got, want[name])
    c = m.counters.cpu().numpy()
    r = t.requests
    assert c[2:2 + r].tolist() == ref.length and c[2 + r:].tolist() == [len(p) for p in ref.pages]
    ring, table = t.ring.cpu().numpy(), t.table.cpu().numpy()
    assert c[1] == len(ref.free) and [int(ring[(c[0] + i) % len(ring)]) for i in range(c[1])] == list(ref.free)
    for k in range(r):
        assert table[k, :len(ref.pages[k])].tolist() == ref.pages[k], k
    ref.check()


@pytest.mark.parametrize("r,page,pool,most", [(1, 1, 7, 5), (1, 16, 40, 1), (3, 4, 11, 6), (64, 16, 90, 9), (257, 24, 330, 8),
                                              (1023, 8, 3000, 6), (1024, 32, 1300, 5), (1025, 1, 9000, 17), (2500, 16, 4000, 4)])
def test_steps(ge, gpu, r, page, pool, most):
    """Many steps of one table in place: tokens kept and dropped, requests that end and start, pools that run dry (later
    requests without new pages still served), full rows, a queue that wraps round."""
    t, ref = ge.paged.PageTable(r, pool, page, most, device=gpu), rr.Pages(r, pool, page, most)
    rng = np.random.default_rng(r * 100 + page)
    kept_to = np.zeros(r, np.int64)
    seen = set()
    for k in range(12):
        keep = np.minimum(rng.integers(0, 9, r), kept_to)
        keep[rng.random(r) < 0.15] = -1
        add = rng.integers(0, 9, r) * (rng.random(r) < 0.8)
        long = rng.random(r) < 0.1
        add[long] = rng.integers(0, most * page + 3, r)[long]
        depth = None
        if k % 3 == 1:
            depth = rng.integers(0, 5, int(add.sum()))
        m = t.step(torch.from_numpy(add).to(gpu) if k % 2 else add, keep=keep, depth=depth, max_tokens=int(add.sum()))
        want = ref.step(add, keep, depth)
        _same(t, ref, m, want)
        kept_to = np.where(np.array(want["status"]) == 0, add, 0)
        seen |= set(want["status"])
    assert seen >= {0, 1} or r == 1


def test_a_step_into_other_counters_can_be_made_again(ge, gpu):
    """into=: the table's own counters stay, so the step can be repeated (the same pages) or made otherwise."""
    t, ref = ge.paged.PageTable(40, 200, 8, 6, device=gpu), rr.Pages(40, 200, 8, 6)
    rng = np.random.default_rng(1)
    add = rng.integers(0, 20, 40)
    _same(t, ref, t.step(add), ref.step(add))
    keep = np.where(rng.random(40) < 0.2, -1, np.minimum(add, rng.integers(0, 20, 40)))
    nxt = rng.integers(0, 12, 40)
    into, old = torch.zeros_like(t.counters), t.counters.clone()
    t.step(rng.integers(0, 30, 40), keep=keep, into=into)  # (a step that is then not taken)
    first = t.step(nxt, keep=keep, into=into)
    assert torch.equal(t.counters, old) and first.counters is into
    got = [x.clone() for x in (first.slot, first.pos, first.counters)]
    again = t.step(nxt, keep=keep, into=into)
    assert all(torch.equal(a, b) for a, b in zip(got, (again.slot, again.pos, again.counters)))
    t.counters.copy_(into)
    _same(t, ref, again, ref.step(nxt, keep))


def test_map_longer_and_shorter_than_the_tokens(ge, gpu):
    """Entries past the tokens are -1, 0, -1 (a captured batch of fixed size); requests past the map's end get nothing, one
    that only gives back still does."""
    t, ref = ge.paged.PageTable(5, 50, 4, 8, device=gpu), rr.Pages(5, 50, 4, 8)
    add = [3, 0, 7, 1, 0]
    _same(t, ref, t.step(add, max_tokens=4000), ref.step(add, max_tokens=4000))
    add, keep = [2, 9, 1, 0, 3], [1, 0, 7, -1, 0]
    m, want = t.step(add, keep=keep, max_tokens=8), ref.step(add, keep, max_tokens=8)
    assert want["status"] == [0, 1, 1, 0, 1]
    _same(t, ref, m, want)
    add = [0] * 5
    _same(t, ref, t.step(add, max_tokens=0), ref.step(add, max_tokens=0))
    _same(t, ref, t.step(add), ref.step(add))


def test_numbers_out_of_range(ge, gpu):
    """Bad keep, add and state leave their request as it was (a bad queue: every request); nothing is read past the arrays."""
    t, ref = ge.paged.PageTable(4, 20, 4, 5, device=gpu), rr.Pages(4, 20, 4, 5)
    add = [5, 6, 7, 8]
    _same(t, ref, t.step(add), ref.step(add))
    add, keep = [-1, 2, 2 ** 31 - 1, 1], [0, 9, 1, 2 ** 31 - 1]
    m, want = t.step(add, keep=keep, max_tokens=100), ref.step(add, keep, max_tokens=100)
    assert want["status"] == [2, 2, 1, 2]
    c = m.counters.cpu().tolist()
    assert m.status.cpu().tolist() == want["status"] and c[2:] == ref.length + [len(p) for p in ref.pages]
    assert (m.slot == -1).all() and m.begin.cpu().tolist() == [0, 0, 2, 2 ** 31 - 1, 2 ** 31 - 1]
    good = t.counters.clone()
    for i, bad in ((0, -1), (0, 20), (1, -5), (1, 21), (2, -1), (6, 6), (7, -1), (9, 2 ** 31 - 1)):
        t.counters.copy_(good)
        t.counters[i] = bad
        was, ring, table = t.counters.clone(), t.ring.clone(), t.table.clone()
        m = t.step([9, 9, 9, 9], keep=[0, 0, 0, 0], max_tokens=64)
        st = m.status.cpu().tolist()
        assert all(s == 2 for s in st) if i < 2 else st[(i - 2) % 4] == 2
        if i < 2:
            assert torch.equal(t.counters, was) and torch.equal(t.ring, ring) and torch.equal(t.table, table)
            assert (m.slot == -1).all()
        else:
            k = (i - 2) % 4
            assert t.counters[2 + k] == was[2 + k] and t.counters[6 + k] == was[6 + k]
            assert (m.slot[9 * k:9 * k + 9] == -1).all() and torch.equal(t.table[k], table[k])


def test_table_rows_with_a_stride(ge, gpu):
    """A table that is part of a wider one: what lies past its columns is left."""
    wide = torch.full((6, 9), -5, dtype=torch.int32, device=gpu)
    ref = rr.Pages(6, 60, 4, 5)
    counters = torch.zeros(14, dtype=torch.int32, device=gpu)
    counters[1] = 60
    t = ge.paged.PageTable.of(wide[:, :5], torch.arange(60, dtype=torch.int32, device=gpu), counters, 4)
    add = [20, 21, 1, 0, 17, 5]
    _same(t, ref, t.step(add), ref.step(add))
    assert (wide[:, 5:] == -5).all()


def test_long_steps(ge, gpu):
    """Prompts of a long batch: more tokens than the launch has threads."""
    r, page = 700, 16
    t, ref = ge.paged.PageTable(r, 70000, page, 600, device=gpu), rr.Pages(r, 70000, page, 600)
    rng = np.random.default_rng(2)
    add = rng.integers(0, 1500, r)
    _same(t, ref, t.step(torch.from_numpy(add).to(gpu), max_tokens=int(add.sum()) + 77), ref.step(add, None, None, int(add.sum()) + 77))
    keep = np.where(rng.random(r) < 0.5, -1, add)
    add = rng.integers(0, 3, r)
    _same(t, ref, t.step(add, keep=keep), ref.step(add, keep))


def test_steps_in_a_graph(ge, gpu):
    """A captured step replayed: each replay is the next step of the table; eager steps in between."""
    r = 33
    t, ref = ge.paged.PageTable(r, 400, 8, 12, device=gpu), rr.Pages(r, 400, 8, 12)
    add, keep = (torch.zeros(r, dtype=torch.int32, device=gpu) for _ in range(2))
    rng = np.random.default_rng(3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _same(t, ref, t.step(add, keep=keep, max_tokens=300), ref.step([0] * r, [0] * r, None, 300))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            m = t.step(add, keep=keep, max_tokens=300)
        last = np.zeros(r, np.int64)
        for k in range(9):
            a = rng.integers(0, 10, r)
            kp = np.where(rng.random(r) < 0.1, -1, np.minimum(last, rng.integers(0, 10, r)))
            if k % 4 == 3:
                mm = t.step(a, keep=kp, max_tokens=300)
            else:
                add.copy_(torch.from_numpy(a))
                keep.copy_(torch.from_numpy(kp))
                g.replay()
                mm = m
            s.synchronize()
            want = ref.step(a, kp, None, 300)
            _same(t, ref, mm, want)
            last = np.where(np.array(want["status"]) == 0, a, 0)


def test_c_refusals(ge, gpu):
    lib = ge._lib
    h = lib.handle(gpu.index, 1, 1)
    t = ge.paged.PageTable(2, 8, 4, 4, device=gpu)
    buf = torch.full((64,), -7, dtype=torch.int64, device=gpu)

    def call(**kw):
        p, s = lib.Pages(), lib.Step()
        p.size, s.size = C.sizeof(lib.Pages), C.sizeof(lib.Step)
        p.requests, p.page, p.pool, p.max_pages, p.table_ld = 2, 4, 8, 4, 4
        p.table, p.ring, p.counters, p.counters_out = (x.data_ptr() for x in (t.table, t.ring, t.counters, t.counters))
        s.max_tokens = 4
        s.add = s.begin = s.slot = s.seq_len = s.status = buf.data_ptr()
        s.stream = torch.cuda.current_stream().cuda_stream
        for k, v in kw.items():
            setattr(p if hasattr(p, k) and k != "size" else s, k, v)
        with h.lock:
            rc = h.L.gsp_pages_step(h.h, C.byref(p), C.byref(s))
        return rc, h.L.gse_last_error(h.h).decode()

    for kw, rc, text in ((dict(table=None), lib.E_ARG, "required"), (dict(add=None), lib.E_ARG, "required"),
                         (dict(slot=None), lib.E_ARG, "required"), (dict(page=0), lib.E_ARG, "> 0"),
                         (dict(pool=0), lib.E_ARG, "> 0"), (dict(max_pages=0), lib.E_ARG, "> 0"),
                         (dict(table_ld=3), lib.E_ARG, "table_ld"), (dict(pool=1 << 31), lib.E_UNSUPPORTED, "2^31"),
                         (dict(page=1 << 29), lib.E_UNSUPPORTED, "2^31"), (dict(max_tokens=1 << 31), lib.E_UNSUPPORTED, "2^30"),
                         (dict(size=0), lib.E_ARG, "short")):
        got, why = call(**kw)
        assert got == rc and text in why, (kw, got, why)
    assert call(requests=0)[0] == 0
    torch.cuda.synchronize()
    assert (buf == -7).all() and t.counters.tolist() == [0, 8, 0, 0, 0, 0]


# ---- paths -----------------------------------------------------------------------------------------------------------

def _paths(rng, r, nodes, depth):
    """Ascending paths (the anchor first) of random lengths, some whose targets are later entries' sources."""
    lens = rng.integers(0, depth + 1, r)
    nd = np.full((r, depth), -1, np.int64)
    for k in range(r):
        if lens[k]:
            nd[k, 0] = 0
            nd[k, 1:lens[k]] = np.sort(rng.choice(np.arange(1, nodes), lens[k] - 1, replace=False))
    return lens, nd


SHAPES = [((9, 16, 8, 128), torch.bfloat16, False), ((9, 16, 3, 40), torch.bfloat16, False), ((30, 5, 7), torch.uint8, False),
          ((40, 4, 3, 5), torch.float16, False), ((9, 8, 16, 64), torch.bfloat16, True), ((11, 5, 24, 80), torch.uint8, True),
          ((12, 3, 16, 6), torch.float32, True), ((150, 1, 2, 12), torch.int8, False)]


@pytest.mark.parametrize("shape,dtype,heads_first", SHAPES)
@pytest.mark.parametrize("stacked", [True, False])
def test_paths(ge, gpu, shape, dtype, heads_first, stacked):
    """Every layout against the entries moved one after the other; slots outside the paths are left."""
    rng = np.random.default_rng(sum(shape))
    n, page = 5, shape[2] if heads_first else shape[1]
    slots = shape[0] * page
    r, nodes, depth = 9, 16, 7
    k = torch.from_numpy(rng.integers(-100, 100, (n, *shape))).to(dtype)
    lens, nd = _paths(rng, r, nodes, depth)
    slot = np.sort(rng.permutation(slots)[:r * nodes].reshape(r, nodes), 1) if slots >= r * nodes else None
    assert slot is not None
    rng.permuted(slot, axis=1, out=slot)
    slot = slot.reshape(-1)
    anchor = np.arange(r) * nodes
    nodes_abs = np.where(nd >= 0, nd + anchor[:, None], -1)
    want = k.clone()
    view = want.transpose(2, 3) if heads_first else want        # [n, pages, page, heads, ...]
    rr.keep_path(lambda s: view[:, s // page, s % page].clone(), lambda s, d: view[:, s // page, s % page].copy_(d), slot, anchor,
                 lens, nodes_abs)
    dev = [torch.from_numpy(x).to(gpu) for x in (slot, anchor, lens, nodes_abs)]
    c = k.to(gpu)
    parts = c if stacked else ge.paged.Caches([c[i].clone() for i in range(n)], heads_first)
    ge.paged.keep_path(parts, dev[0], *(x.int() for x in dev[1:]), heads_first=heads_first)
    got = c if stacked else torch.stack(parts.tensors)
    assert torch.equal(got.cpu(), want)
    if stacked:  # (a second call moves again: what the oracle does)
        rr.keep_path(lambda s: view[:, s // page, s % page].clone(), lambda s, d: view[:, s // page, s % page].copy_(d), slot,
                     anchor, lens, nodes_abs)
        ge.paged.keep_path(c, dev[0], *(x.int() for x in dev[1:]), heads_first=heads_first)
        assert torch.equal(c.cpu(), want)


def test_path_views(ge, gpu):
    """Caches that are views: keys and values of one tensor, heads apart, bases off 16 bytes."""
    rng = np.random.default_rng(5)
    r, nodes = 4, 6
    slot = rng.permutation(40)[:r * nodes]
    anchor, lens = np.arange(r) * nodes, np.array([3, 1, 4, 6])
    nd = np.array([[0, 2, 5, -1, -1, -1], [0, -1, -1, -1, -1, -1], [0, 3, 4, 5, -1, -1], [0, 1, 2, 3, 4, 5]])
    nd = np.where(nd >= 0, nd + anchor[:, None], -1)
    args = [torch.from_numpy(slot).to(gpu)] + [torch.from_numpy(x).int().to(gpu) for x in (anchor, lens, nd)]
    base = torch.from_numpy(rng.integers(0, 99, (10, 2, 4, 5, 24))).to(torch.bfloat16)
    for cut in (lambda x: [x[:, 0], x[:, 1]], lambda x: [x[:, 0, :, 1:], x[:, 1, :, 1:]], lambda x: [x[:, 0, :, :, 3:], x[:, 1, :, :, 3:]],
                lambda x: [x[:, 0, :, :, 1:9]]):
        want, got = base.clone(), base.to(gpu)
        for v in cut(want):
            rr.keep_path(lambda s: v[s // 4, s % 4].clone(), lambda s, d: v[s // 4, s % 4].copy_(d), slot, anchor, lens, nd)
        ge.paged.keep_path(ge.paged.Caches(cut(got)), *args)
        assert torch.equal(got.cpu(), want)


def test_path_entries_out_of_range_are_skipped(ge, gpu):
    c = torch.arange(2 * 4 * 4 * 8, device=gpu).reshape(2, 4, 4, 8).float()
    was = c.clone()
    slot = torch.tensor([0, -1, 16, 3, 2 ** 40, 5], device=gpu)
    nodes = torch.tensor([[0, 1, 2], [0, 99, -4], [3, 3, 5], [4, 5, 5]], dtype=torch.int32, device=gpu)
    ge.paged.keep_path(c, slot, torch.tensor([0, 0, -1, 2 ** 31 - 4], dtype=torch.int32, device=gpu),
                       torch.tensor([3, 2 ** 31 - 1, 2, 3], dtype=torch.int32, device=gpu), nodes)
    want = was.clone()
    assert torch.equal(c[0, 0, 1:], want[0, 0, 1:]) and torch.equal(c[:, 1:], want[:, 1:])
    ge.paged.keep_path(c, slot[:0], torch.zeros(0, dtype=torch.int32, device=gpu), torch.zeros(0, dtype=torch.int32, device=gpu),
                       torch.zeros((0, 3), dtype=torch.int32, device=gpu))


def test_path_past_32_bits(ge, gpu):
    """Slots more than 2^32 bytes into a cache."""
    pages, page, row = 34000, 16, 8192
    c = torch.zeros((1, pages, page, row), dtype=torch.uint8, device=gpu)
    top = pages * page - 1
    c[0, -1] = torch.arange(page, device=gpu, dtype=torch.uint8)[:, None]
    slot = torch.tensor([7, top - 9, top, top - 3], device=gpu)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    ge.paged.keep_path(c, slot, one(0), one(3), one(0, 2, 3)[None])
    assert (c[0, -1, page - 10] == page - 1).all() and (c[0, -1, page - 1] == page - 4).all()
    ge.paged.keep_path(c, slot.flip(0), one(0), one(3), one(0, 2, 3)[None])
    assert (c[0, -1, page - 1] == page - 1).all() and (c[0, -1, page - 10] == 0).all() and (c[0, 0] == 0).all()


def test_path_c_refusals(ge, gpu):
    lib = ge._lib
    h = lib.handle(gpu.index, 1, 1)
    c = torch.zeros((2, 3, 4, 16), device=gpu)
    ints = torch.zeros(64, dtype=torch.int32, device=gpu)
    slot = torch.zeros(8, dtype=torch.int64, device=gpu)

    def call(**kw):
        p = lib.Path()
        p.size, p.requests, p.tokens, p.caches = C.sizeof(lib.Path), 2, 8, 2
        p.slot, p.anchor, p.emit_len, p.emit_nodes, p.emit_ld = slot.data_ptr(), ints.data_ptr(), ints.data_ptr(), ints.data_ptr(), 3
        p.cache, p.cache_stride, p.page, p.pages, p.chunks, p.chunk_bytes = c.data_ptr(), 768, 4, 3, 1, 64
        p.page_stride, p.token_stride = 256, 64
        p.stream = torch.cuda.current_stream().cuda_stream
        for k, v in kw.items():
            setattr(p, k, v)
        with h.lock:
            return h.L.gsp_keep_path(h.h, C.byref(p)), h.L.gse_last_error(h.h).decode()

    for kw, rc, text in ((dict(slot=None), lib.E_ARG, "required"), (dict(cache=None), lib.E_ARG, "required"),
                         (dict(page=0), lib.E_ARG, "> 0"), (dict(chunk_bytes=0), lib.E_ARG, "> 0"), (dict(emit_ld=0), lib.E_ARG, "> 0"),
                         (dict(token_stride=-64), lib.E_ARG, ">= 0"), (dict(cache_ptrs=ints.data_ptr(), align=0), lib.E_ARG, "align"),
                         (dict(cache_ptrs=ints.data_ptr(), align=12), lib.E_ARG, "align"),
                         (dict(chunk_bytes=1 << 31), lib.E_UNSUPPORTED, "2^30"), (dict(caches=1 << 26), lib.E_UNSUPPORTED, "2^30"),
                         (dict(size=4), lib.E_ARG, "short")):
        got, why = call(**kw)
        assert got == rc and text in why, (kw, got, why)
    assert call(requests=0)[0] == 0 and call(caches=0)[0] == 0


# ---- rounds ----------------------------------------------------------------------------------------------------------

def test_rounds_of_trees(ge, gpu):
    """Steps, verify rounds over logits and path moves as an engine would run them, nothing read back in between: after every
    round the cache holds each request's tokens at its slots, in order."""
    S = ge.sampling.SamplingParams
    trees = [[0, 1, 2, 0, 4, 5], [0, 0, 0, 1, 2, 4], [], [0, 1]]
    r, v, page = len(trees), 997, 4
    sizes = [len(p) + 1 for p in trees]
    total = sum(sizes)
    anchors = np.concatenate([[0], np.cumsum(sizes)])
    depth = []
    for p in trees:
        d = [0]
        for x in p:
            d.append(d[x] + 1)
        depth += d
    t = ge.paged.PageTable(r, 120, page, 30, device=gpu)
    caches = torch.full((3, 120, page, 2, 8), -1.0, device=gpu)   # (a cache row holds its token's id and its position)
    host = [[int(k) + 1] for k in range(r)]                        # the requests' tokens, the last one not in the cache yet
    g = torch.Generator(device=gpu).manual_seed(9)
    keep, moved = None, 0
    for rnd in range(6):
        m = t.step(np.array(sizes, np.int32), keep=keep, depth=np.array(depth, np.int32), max_tokens=total)
        assert m.begin.cpu().tolist() == anchors.tolist() and (m.status == 0).all()
        assert m.pos.cpu().tolist() == [len(host[k]) - 1 + depth[anchors[k] + j] for k in range(r) for j in range(sizes[k])]
        x = torch.randn((total, v), generator=g, device=gpu) * 3
        best = x.argmax(1).cpu().tolist()
        reqs, toks = [], []
        for k, p in enumerate(trees):  # some branch of the tree follows the target's choices
            a = anchors[k]
            tok = [best[a + par] if (rnd + j) % 2 or j >= 3 else (best[a + par] + 1) % v for j, par in enumerate(p)]
            reqs.append(dict(target=x[a:a + sizes[k]], tokens=tok, parents=p, params=S(), seed=k, nout=rnd))
            toks += [host[k][-1]] + tok
        ids = torch.tensor(toks, device=gpu).float()
        rows = torch.stack([ids, m.pos.float()], 1).repeat(1, 8).reshape(total, 8, 2).transpose(1, 2)
        caches[:, m.slot // page, m.slot % page] = rows.contiguous()
        call = ge.spec.VerifyCall(reqs)
        call.launch()
        call.keep_path(m, caches)
        with pytest.raises(ValueError):
            call.keep_path(t.step([1] * r, keep=call.e_len, into=torch.zeros_like(t.counters)), caches)  # another round's
        keep = call.e_len
        for k, (new, path, why) in enumerate(call.result()):
            assert why is None and len(new) == len(path)
            moved += sum(path[i] != i for i in range(len(path)))
            host[k] += new
    assert moved > 5
    m = t.step([0] * r, keep=keep)
    assert m.seq_len.cpu().tolist() == [len(h) - 1 for h in host]
    table = t.table.cpu().numpy()
    for k in range(r):
        for i, tok in enumerate(host[k][:-1]):
            row = caches[:, table[k, i // page], i % page].cpu()
            assert (row[:, 0] == tok).all() and (row[:, 1] == i).all(), (k, i, tok, row[0, :, 0])


def test_rounds_of_chains(ge, gpu):
    """Chains against probability rows, captured with the step in one graph: each replay is a round."""
    r, k, v, page = 6, 3, 1200, 4
    t = ge.paged.PageTable(r, 200, page, 40, device=gpu)
    ref = rr.Pages(r, 200, page, 40)
    g = torch.Generator(device=gpu).manual_seed(3)
    d = r * k
    keep = torch.zeros(r, dtype=torch.int32, device=gpu)
    add = torch.full((r,), k + 1, dtype=torch.int32, device=gpu)
    begin = torch.arange(0, d + 1, k, dtype=torch.int32, device=gpu)
    p, q = torch.zeros((d + r, v), device=gpu), torch.zeros((d, v), device=gpu)
    tok = torch.zeros(d, dtype=torch.int32, device=gpu)
    coin, u = torch.zeros(d, dtype=torch.float64, device=gpu), torch.zeros(r, dtype=torch.float64, device=gpu)

    def fill():
        z = torch.randn((d + r, v), generator=g, device=gpu) * 2
        zq = z.view(r, k + 1, v)[:, :k].reshape(d, v) + 0.3 * torch.randn((d, v), generator=g, device=gpu)
        p.copy_(torch.softmax(z, 1))
        q.copy_(torch.softmax(zq, 1))
        tok.copy_((zq - torch.rand((d, v), generator=g, device=gpu).clamp_(1e-9, 1 - 6e-8).log_().neg_().log_()).argmax(1))
        coin.copy_(torch.rand(d, generator=g, device=gpu, dtype=torch.float64))
        u.copy_(torch.rand(r, generator=g, device=gpu, dtype=torch.float64))

    def one():
        m = t.step(add, keep=keep, max_tokens=r * (k + 1))
        o = ge.spec.verify_chains(p, tok, begin, coin, u, draft=q, max_drafts=k)
        keep.copy_(o.emit_len)
        return m, o

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lens = np.zeros(r, np.int64)
    with torch.cuda.stream(s):
        graph = None
        for rnd in range(7):
            fill()
            if rnd == 2:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    m, o = one()
            if graph is None:
                m, o = one()
            else:
                graph.replay()
            s.synchronize()
            want = ref.step([k + 1] * r, lens, None, r * (k + 1))
            _same(t, ref, m, want)
            chains = rr.chains(p.double().cpu().numpy(), q.double().cpu().numpy(), tok.cpu().numpy(), begin.cpu().numpy(),
                               coin.cpu().numpy(), u.cpu().numpy())
            assert o.tolist() == [(c[0], None) for c in chains]
            lens = np.array([len(c[0]) for c in chains])
    assert keep.cpu().tolist() == lens.tolist() and len(set(lens.tolist())) > 1


def test_commits(ge, gpu):
    """VerifyCall.commit and Chains.commit: the same as the calls they stand for, requests that end among them."""
    S = ge.sampling.SamplingParams
    trees = [[0, 1, 0, 3], [0, 0, 2], [0]]
    sizes, v = [5, 4, 2], 500
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn((11, v), generator=g, device=gpu) * 3
    best = x.argmax(1).cpu().tolist()
    at = [0, 5, 9]
    reqs = [dict(target=x[at[k]:at[k] + sizes[k]], parents=p, params=S(), seed=1,
                 tokens=[(best[at[k] + par] + (k == 0 and j == 0)) % v for j, par in enumerate(p)])
            for k, p in enumerate(trees)]
    out = []
    for ends in (None, [False, True, False], torch.tensor([True, False, True], device=gpu)):
        both = []
        for whole in (True, False):
            t = ge.paged.PageTable(3, 40, 4, 6, device=gpu)
            m = t.step(sizes)
            c = torch.arange(2 * 40 * 4 * 8, device=gpu).reshape(2, 40, 4, 8).float()
            call = ge.spec.VerifyCall(reqs)
            call.launch()
            if whole:
                nxt = call.commit(m, t, c, [2, 2, 2], ends=ends)
            else:
                call.keep_path(m, c)
                keep = call.e_len.tolist() if ends is None else [-1 if e else n for n, e in zip(call.e_len.tolist(), list(ends))]
                nxt = t.step([2, 2, 2], keep=keep)
            both.append((c, nxt.slot, nxt.pos, nxt.seq_len, t.counters, t.table, t.ring))
        assert all(torch.equal(a, b) for a, b in zip(*both))
        out.append(both[0])
    assert not torch.equal(out[0][4], out[1][4]) and call.e_len.tolist()[0] > 1
    short = ge.spec.VerifyCall(reqs, emit_ld=1)  # a walk cut at one token keeps one
    t = ge.paged.PageTable(3, 40, 4, 6, device=gpu)
    m = t.step(sizes)
    short.launch()
    assert short.commit(m, t, c, [0, 0, 0]).seq_len.tolist() == [len(r[0]) for r in short.result()] == [1, 1, 1]
    o = ge.spec.verify_chains(torch.softmax(x[:6], 1), best[:3], [0, 3, 3, 3], [0.0] * 3, [0.5] * 3)
    t, u = (ge.paged.PageTable(3, 40, 4, 6, device=gpu) for _ in range(2))
    t.step([4, 1, 1]), u.step([4, 1, 1])
    a = o.commit(t, [1, 1, 1], ends=[False, False, True])
    b = u.step([1, 1, 1], keep=[o.emit_len.tolist()[0], 1, -1])
    assert torch.equal(a.slot, b.slot) and torch.equal(t.counters, u.counters) and (t.length.tolist()[1:] == [1, 0])
    with pytest.raises(ValueError):
        o.commit(t, [1, 1, 1], ends=[True])
