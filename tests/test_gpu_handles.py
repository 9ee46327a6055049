"""Handles of captured calls on the GPU (_lib.handle)."""
import gc
import weakref

import numpy as np
import pytest
import torch

from oracle import round_ref as rr

pytestmark = pytest.mark.gpu


def _chains(gpu, v, seed):
    """Arguments on the device, and the oracle's answer."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    p = torch.softmax(torch.randn((7, v), generator=g, device=gpu) * 2, 1)
    q = torch.softmax(torch.randn((4, v), generator=g, device=gpu) * 2, 1)
    rng = np.random.default_rng(seed)
    tok, begin, coin, u = rng.integers(0, v, 4), np.array([0, 3, 3, 4]), rng.random(4) * 1e-3, rng.random(3)
    want = [(w[0], None) for w in rr.chains(p.double().cpu().numpy(), q.double().cpu().numpy(), tok, begin, coin, u)]
    i32 = lambda x: torch.from_numpy(x).int().to(gpu)  # noqa: E731
    f64 = lambda x: torch.from_numpy(x).to(gpu)  # noqa: E731
    return dict(target=p, tokens=i32(tok), begin=i32(begin), coins=f64(coin), u=f64(u), draft=q, max_drafts=3), want


def test_a_graph_outlives_its_streams_handle(ge, gpu):
    """A captured call, then eager ones that replace the stream's handle and push it out of the cache: the captured handle
    stays open (checked before any replay), and replays agree with the oracle, other calls in between."""
    lib, chains = ge._lib, ge.spec.verify_chains
    small, want = _chains(gpu, 3001, 1)
    large, want_l = _chains(gpu, 150001, 2)
    s = torch.cuda.Stream(gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        assert chains(**small).tolist() == want
        old = weakref.ref(lib.handle(gpu.index, 1, 3001))
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = chains(**small)
        assert chains(**large).tolist() == want_l
        assert lib.handle(gpu.index, 1, 150001) is not old()
    others = [torch.cuda.Stream(gpu) for _ in range(lib.MAX_HANDLES + 1)]
    for o in others:
        with torch.cuda.stream(o):
            assert chains(**small).tolist() == want
    gc.collect()
    assert old() is not None and old().h and all(h is not old() for h in lib._handles.values())
    with torch.cuda.stream(s):
        for _ in range(3):
            out.tokens.fill_(-9)
            out.emit_len.fill_(-9)
            graph.replay()
            assert out.tolist() == want
            assert chains(**large).tolist() == want_l
    torch.cuda.synchronize()
    del graph
    lib.release_captured()
    gc.collect()
    assert old() is None


def test_a_capture_that_needs_a_handle_is_refused(ge, gpu):
    """On a stream without a handle, or with a smaller one, the call is refused and the capture ends as any other."""
    chains = ge.spec.verify_chains
    args, want = _chains(gpu, 2003, 3)
    more, want_m = _chains(gpu, 2005, 4)
    s = torch.cuda.Stream(gpu)
    x = torch.zeros(4, device=gpu)
    torch.cuda.synchronize()
    ge._lib._handles.pop((gpu.index, s.cuda_stream), None)  # (streams come from a pool: another test's may be this one)
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            x.add_(1)
            with pytest.raises(RuntimeError, match="not open"):
                chains(**args)
        assert chains(**args).tolist() == want
        h = ge._lib.handle(gpu.index, 1, 2003)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            x.add_(1)
            if h.vocab < 2005:
                with pytest.raises(RuntimeError, match="before the capture"):
                    chains(**more)
        graph.replay()
        s.synchronize()
        assert x.tolist() == [1.0] * 4
        assert chains(**more).tolist() == want_m


def test_page_calls_on_many_streams_leave_the_cache(ge, gpu):
    """Page steps and path moves on more streams than the cache holds: every handle in it stays, and their answers agree."""
    lib = ge._lib
    args, want = _chains(gpu, 2003, 5)
    assert ge.spec.verify_chains(**args).tolist() == want
    was = list(lib._handles.items())
    add, ref = [5, 0, 9], rr.Pages(3, 12, 4, 4)
    slot, status = (ref.step(add)[k] for k in ("slot", "status"))
    one = torch.zeros(1, dtype=torch.int32, device=gpu)
    nodes = torch.tensor([[0, 3]], dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    for _ in range(lib.MAX_HANDLES + 2):
        with torch.cuda.stream(torch.cuda.Stream(gpu)):
            t = ge.paged.PageTable(3, 12, 4, 4, device=gpu)
            m = t.step(add)
            c = torch.arange(12 * 4 * 8, device=gpu).reshape(1, 12, 4, 8).float()
            ge.paged.keep_path(c, m.slot, one, one + 2, nodes)
            assert m.slot.tolist() == slot and m.status.tolist() == status
            assert c[0, 0, 1].tolist() == list(range(24, 32))  # (node 3's row, in the place after the anchor)
    assert list(lib._handles.items()) == was
