"""The operators around a verify round (include/gsp.h) without a GPU: the oracle's pins, the binding's structs against the
header, and the refusals of the Python layer."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import round_ref as rr
from oracle import sampling_ref as ora
from oracle import spec_ref as spo

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---- the oracle ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("onehot", [False, True])
def test_the_emitted_tokens_law_is_the_targets(onehot):
    """Over a draft drawn from q and a grid of coins and draws, the first emitted token has the target's law: p and q are
    multiples of 1/8 and the grids' points midpoints of 1/64, so the counts are exact but for the residual's cells."""
    p = np.array([[1, 3, 0, 4], [2, 2, 2, 2]]) / 8
    q = np.array([[3, 1, 2, 2]]) / 8
    grid = (np.arange(64) + 0.5) / 64
    law = np.zeros(4)
    for x in range(4):
        px = 1.0 if onehot and x == 1 else 0.0 if onehot else q[0][x]
        if not px:
            continue
        for coin in grid:
            for u in grid:
                out, probs, bad = rr.chain(p, None if onehot else q, [x], [coin], u)
                assert not bad and probs[0] == p[0][out[0]]
                law[out[0]] += px / 64 / 64
    # (the residual's law over 64 midpoints is off by less than a cell per border)
    assert np.abs(law - p[0]).max() < 2 / 64


def test_one_draft_is_mss_with_one_kid():
    rng = np.random.default_rng(0)
    for k in range(300):
        v = int(rng.integers(1, 40))
        p = rng.random((2, v)) ** 3 * (rng.random((2, v)) < 0.7) + 1e-6
        p /= p.sum(1, keepdims=True)
        q = rng.random(v) ** 3 * (rng.random(v) < 0.7) + 1e-6
        q /= q.sum()
        x, onehot, seed = int(rng.integers(0, v)), k % 3 == 0, int(rng.integers(0, 2 ** 63))
        want = spo.mss(p[0], [(x, None if onehot else q)], seed, 7)
        coin = ora.uniform(ora.mix(seed, spo.SALT_ACC), 7)
        out, _, bad = rr.chain(p, None if onehot else q[None], [x], [coin], ora.uniform(ora.mix(seed, spo.SALT_RES), 7))
        assert not bad
        assert out[0] == want[0] and (len(out) == 2) == (want[1] is not None)


def test_draw_edges():
    w = np.array([0.0, 2.0, 0.0, 1.0, -5.0, 0.0])
    assert [rr.draw(w, u) for u in (0.0, 0.5, 2 / 3, 0.67, 1 - 2.0 ** -53, 1.0)] == [1, 1, 1, 3, 3, 3]
    assert rr.draw(np.zeros(3), 0.5) == rr.draw(np.array([1.0, np.nan]), 0.1) == rr.draw(np.array([1.0, np.inf]), 0.1) == -1


def test_pages_known_answers():
    g = rr.Pages(3, 8, 4, 4)
    m = g.step([5, 1, 0])
    assert m["slot"] == [0, 1, 2, 3, 4, 8] and m["pos"] == [0, 1, 2, 3, 4, 0] and m["status"] == [0, 0, 0]
    assert m["begin"] == [0, 5, 6, 6] and m["seq"] == [5, 1, 0]
    # request 0 keeps three of five (one page left over, taken again), 1 ends, 2 starts with 17 tokens: past four pages
    m = g.step([3, 0, 17], [3, -1, 0])
    assert m["slot"][:3] == [3, 4, 5] and m["status"] == [0, 0, 1] and m["slot"][3:] == [-1] * 17
    assert list(g.free) == [3, 4, 5, 6, 7, 2]
    m = g.step([16, 16, 16], [3, 0, 0])  # six free pages: request 0 (at 6) takes four more: past its row
    assert m["status"] == [1, 0, 1] and len(g.free) == 2
    g.check()


# ---- the binding -----------------------------------------------------------------------------------------------------

def test_structs_and_symbols_match_the_header(ge, tmp_path):
    lib = ge._lib
    header = os.path.join(ROOT, "include", "gsp.h")
    names = set(re.findall(r"GSE_API\s+[\w\s\*]+?\b(gsp_\w+)\s*\(", open(header).read()))
    assert names == set(lib.ROUND_SIGNATURES)
    L = lib.bind()
    pairs = [("gsp_chains", lib.Chains), ("gsp_pages", lib.Pages), ("gsp_step", lib.Step), ("gsp_path", lib.Path)]
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "gsp.h"\nint main(void) {\n'
    for t, cls in pairs:
        src += f'printf("%zu\\n", sizeof({t}));\n' + "".join(f'printf("%zu\\n", offsetof({t}, {f}));\n' for f, _ in cls._fields_)
    src += 'printf("%d %d %d %d %d %d %d\\n", GSP_F64, GSP_F32, GSP_BF16, GSP_F16, GSP_STEP_OK, GSP_STEP_FULL, GSP_STEP_BAD);}\n'
    (tmp_path / "a.c").write_text(src)
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")],
                   check=True)
    got = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.splitlines()
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert [int(x) for x in got[:-1]] == want
    assert [int(x) for x in got[-1].split()] == [lib.P_F64, lib.P_F32, lib.P_BF16, lib.P_F16, lib.STEP_OK, lib.STEP_FULL,
                                                 lib.STEP_BAD]
    for n in names:  # no handle, no call
        assert getattr(L, n)(*([None] * len(lib.ROUND_SIGNATURES[n][1]))) == lib.E_ARG


# ---- refusals --------------------------------------------------------------------------------------------------------

def test_verify_chains_refuses(ge):
    p, q = torch.rand(5, 10), torch.rand(3, 10)
    ok = dict(target=p, tokens=[1, 2, 3], begin=[0, 2, 3], coins=[0.1, 0.2, 0.3], u=[0.5, 0.5], draft=q)

    def refused(match, **kw):
        with pytest.raises(ValueError, match=match):
            ge.spec.verify_chains(**{**ok, **kw})

    refused("target", target=p[:4])                                   # a row short
    refused("target", target=p.to(torch.float8_e4m3fn))
    refused("target", target=p[0])
    refused("draft", draft=q[:, :9])
    refused("draft", draft=q[:2])
    refused("draft", draft=q.to(torch.int32))
    refused("coins", coins=[0.1])
    refused("draws", u=[0.5])
    refused("max_drafts", max_drafts=-1)
    refused("one dimension", tokens=torch.ones((3, 1), dtype=torch.int32))
    refused("V = 0", target=p[:, :0], draft=None)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="HIP device"):
            ge.spec.verify_chains(**ok)


def _table(ge, r=3, pool=8, page=4, most=4):
    return ge.paged.PageTable(r, pool, page, most, device="cpu")


def test_page_table_refuses(ge):
    t = _table(ge)
    assert t.free.tolist() == [8] and t.length.tolist() == [0] * 3 and t.held.tolist() == [0] * 3
    for bad in ((0, 8, 4, 4), (3, 0, 4, 4), (3, 8, 0, 4), (3, 8, 4, 0)):
        with pytest.raises(ValueError):
            ge.paged.PageTable(*bad, device="cpu")
    of = ge.paged.PageTable.of
    for kw in (dict(table=t.table.long()), dict(table=t.table.t()), dict(ring=t.ring[None]), dict(counters=t.counters[1:]),
               dict(page=0), dict(table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), dict(counters=t.counters.float())):
        with pytest.raises(ValueError):
            of(**{**dict(table=t.table, ring=t.ring, counters=t.counters, page=4), **kw})
    for kw in (dict(add=[1, 2]), dict(add=[1, 2, 3], keep=[0]), dict(add=[1, 2, 3], depth=[0, 0]), dict(add=[1, 1, 1], max_tokens=-1),
               dict(add=[1, 1, 1], into=torch.zeros(7, dtype=torch.int32))):
        with pytest.raises(ValueError):
            t.step(**kw)
    with pytest.raises(RuntimeError):  # state on the host
        t.step([1, 1, 1])


def test_keep_path_refuses(ge):
    k = torch.zeros(2, 6, 4, 3, 8)
    ok = dict(caches=k, slot=torch.zeros(9, dtype=torch.int64), anchor=torch.zeros(2, dtype=torch.int32),
              emit_len=torch.ones(2, dtype=torch.int32), emit_nodes=torch.zeros((2, 3), dtype=torch.int32))
    for kw in (dict(caches=k[0, 0]), dict(caches=k[:1].expand(2, 6, 4, 3, 8)), dict(slot=ok["slot"].int()),
               dict(emit_len=ok["emit_len"][:1]), dict(emit_nodes=ok["emit_nodes"][:1]), dict(caches=k.permute(0, 1, 2, 4, 3)),
               dict(caches=k[:, :1].expand(2, 6, 4, 3, 8)), dict(caches=k[..., ::2])):
        with pytest.raises(ValueError):
            ge.paged.keep_path(**{**ok, **kw})
    with pytest.raises(RuntimeError):
        ge.paged.keep_path(**ok)
    C_ = ge.paged.Caches
    for bad in ([], [k[0], k[1].double()], [k[0], k[1][:3]], [k[0], k[0]]):
        with pytest.raises(ValueError):
            C_(bad)


def test_cache_layouts(ge):
    """(pages, page, chunks, chunk bytes, page / token / chunk strides)"""
    lay = lambda t, hf=False: ge.paged._layout(t.shape, t.stride(), t.element_size(), hf)  # noqa: E731
    t = torch.zeros(6, 4, 3, 8, dtype=torch.bfloat16)
    assert lay(t) == (6, 4, 1, 48, 192, 48, 0)
    assert lay(t[:, :, 1:]) == (6, 4, 1, 32, 192, 48, 0)
    assert lay(t[..., :4]) == (6, 4, 3, 8, 192, 48, 16)          # heads apart
    assert lay(t, True) == (6, 3, 4, 16, 192, 16, 48)            # [pages, 4 heads, 3 tokens, 8]
    assert lay(t.transpose(1, 2)) == (6, 3, 4, 16, 192, 16, 48)
    assert lay(torch.zeros(5, 4, 7, dtype=torch.uint8)) == (5, 4, 1, 7, 28, 7, 0)
    # without gaps: the same, also where a dimension of one has a stride of its own
    dense = lambda t, hf=False: ge.paged._layout(t.shape, t.stride(), t.element_size(), hf, t.is_contiguous())  # noqa: E731
    assert dense(t) == lay(t) and dense(t, True) == lay(t, True)
    one = torch.zeros(400, dtype=torch.uint8).as_strided((5, 1, 2, 6), (12, 77, 6, 1))
    assert one.is_contiguous() and dense(one) == (5, 1, 1, 12, 12, 12, 0)
    one = torch.zeros(400, dtype=torch.uint8).as_strided((5, 2, 1, 6), (12, 6, 77, 1))
    assert one.is_contiguous() and dense(one, True) == (5, 1, 2, 6, 12, 6, 6)
