"""The commits of a verify round (spec.VerifyCall.commit, spec.Chains.commit) without a GPU: what they ask of the page table."""
import copy
from types import SimpleNamespace as NS

import numpy as np
import pytest
import torch

from oracle import round_ref as rr


class _Pages:
    """Takes a step's arguments in the place of a paged.PageTable, and says what then counts as kept."""

    def __init__(self):
        self.calls = []

    def step(self, add, keep=None, depth=None, max_tokens=None, of=None):
        return self._step(*self._ready(add, keep, depth, max_tokens, of=of))

    def _ready(self, add, keep, depth, max_tokens, into=None, of=None):
        return keep, of

    def _step(self, keep, of):
        self.calls.append([k if s == 0 or k < 0 else 0 for k, s in zip(keep.tolist(), of.status.tolist())])
        return "next"


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def _tree_call(ge, lens, ld=9):
    call = ge.spec.VerifyCall.__new__(ge.spec.VerifyCall)
    call.e_len, call.ld, call.longest = _i32(*lens), ld, 9
    call.keep_path = lambda *a: None
    return call


def _chains(ge, lens):
    return ge.spec.Chains(_i32(*lens), None, None, None)


ENDS = [(None, [5, 0, 0, 1]), ([True, False, True, False], [-1, 0, -1, 1])]


@pytest.mark.parametrize("ends,want", ENDS)
def test_a_commit_keeps_nothing_of_a_request_that_was_not_served(ge, ends, want):
    lib = ge._lib
    step = NS(status=_i32(lib.STEP_OK, lib.STEP_FULL, lib.STEP_BAD, lib.STEP_OK))
    lens, pages = (5, 4, 3, 1), _Pages()
    assert _tree_call(ge, lens).commit(step, pages, None, [1] * 4, ends=ends) == "next"
    assert _chains(ge, lens).commit(pages, [1] * 4, ends=ends, step=step) == "next"
    assert pages.calls == [want, want]
    cut = _Pages()  # (a walk cut at two tokens)
    _tree_call(ge, lens, ld=2).commit(step, cut, None, [1] * 4, ends=ends)
    assert cut.calls == [[min(k, 2) for k in want]]


def test_a_commit_with_a_step_of_other_requests_is_refused(ge):
    pages = ge.paged.PageTable(2, 8, 4, 4, device="cpu")
    with pytest.raises(ValueError, match="3 requests"):
        _chains(ge, (1, 2)).commit(pages, [1, 1], step=NS(status=_i32(0, 0, 0)))


def test_why_a_request_that_was_not_served_keeps_nothing():
    """The books alone cannot tell: tokens that a full step added nothing for fit the last page, and count as kept."""
    g = rr.Pages(2, 4, 16, 4)
    g.step([20, 32])
    g.step([0, 0], [20, 32])
    assert g.step([16, 0])["status"] == [1, 0]
    h = copy.deepcopy(g)
    m = g.step([1, 0], [5, 0])
    assert m["status"] == [0, 0] and m["pos"] == [25]  # (20 to 24 were never written)
    m = h.step([1, 0], [5, 0], laid=[1, 0])
    assert m["status"] == [0, 0] and m["pos"] == [20]


def test_a_refused_commit_moves_nothing(ge):
    """A path that moved before its commit was refused would move again in the commit made after."""
    call, moved = _tree_call(ge, (2, 1)), []
    call.keep_path = lambda *a: moved.append(a)
    step, pages = NS(status=_i32(0, 0)), ge.paged.PageTable(2, 8, 4, 4, device="cpu")
    for kw in (dict(add=[1]), dict(add=[1, 1], ends=[True]), dict(add=[1, 1], depth=[0]), dict(add=[1, 1], max_tokens=-1)):
        with pytest.raises(ValueError):
            call.commit(step, pages, None, **kw)
    with pytest.raises(RuntimeError):  # state on the host
        call.commit(step, pages, None, [1, 1])
    with pytest.raises(ValueError):
        call.commit(NS(status=_i32(0, 0, 0)), pages, None, [1, 1])
    assert not moved


def test_an_end_gives_its_pages_back_though_what_follows_does_not_fit():
    """Ten pages of four, six and four of them held: request 0 ends and 44 tokens in its place need eleven."""
    g = rr.Pages(2, 10, 4, 11)
    assert g.step([24, 16])["status"] == [0, 0]
    m = g.step([44, 4], [-1, 16])
    assert m["status"] == [1, 1] and m["seq"] == [0, 16] and list(g.free) == [0, 1, 2, 3, 4, 5] and not g.pages[0]
    g.check()
    m = g.step([20, 4], [0, 0])  # (the next step has them)
    assert m["status"] == [0, 0] and m["seq"] == [20, 20]
    m = g.step([2, 2], [-1, 9])  # past the pages held: left as it was
    assert m["status"] == [0, 2]


def test_numbers_that_are_no_integers_are_refused(ge):
    """Lists and arrays as tensors: a fraction is not cut off."""
    vec, cpu = ge.spec._vec, torch.device("cpu")
    for bad in ([1.5, 2.0], np.array([float("nan")]), np.array([float("inf")]), [1e30], torch.ones(2), ["1"]):
        with pytest.raises(ValueError, match="expected integers"):
            vec(bad, torch.int32, cpu)
    for good, want in (([], []), (np.concatenate([[0], np.cumsum([])]), [0]), ((1, -2), [1, -2]), (np.array([3, 2 ** 40]), [3, 2 ** 31 - 1]), ([-2 ** 40], [-2 ** 31]),
                       (np.array([2 ** 64 - 1], np.uint64), [2 ** 31 - 1]), (np.array([7], np.uint8), [7]),
                       (torch.tensor([5, -2 ** 40]), [5, -2 ** 31]), (range(3), [0, 1, 2])):
        got = vec(good, torch.int32, cpu)
        assert got.dtype is torch.int32 and got.tolist() == want
