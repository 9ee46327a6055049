"""The far ends of the calls around a verify round: rows of more segments than a wave reads at once, rows that are read again
because a draft's distribution is nowhere below the target's, paths of more entries than a wave has lanes, more requests
than a launch has rows of workgroups. Tokens and copies are compared exactly."""
import numpy as np
import pytest
import torch

from oracle import round_ref as rr

pytestmark = pytest.mark.gpu

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16}


def _draws(w, at):
    """The u that falls into the middle of each token of `at` in a row of weights w. The weights are multiples of 2^-26, at
    most 64 of them, so all their sums in fp64 are exact; u and its product with the sum are off by 2^-52 of it, and half a
    token is 2^-28 of it or more (a unit of 2^21 tokens of 64)."""
    c = np.cumsum(w)
    return np.array([(c[t] - 0.5 * w[t]) / c[-1] for t in at])


@pytest.mark.parametrize("target,draft", [("f64", "f64"), ("f64", None), ("f32", "f64"), ("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("v", [524287, 700001, 1 << 21])
def test_long_rows(ge, gpu, v, target, draft):
    """Chains of one draft, rejected or accepted, over rows of up to 2^21 tokens: the tokens that the draws fall into, at both
    ends, around the 512th segment of 1024 tokens and in between."""
    rng = np.random.default_rng(v)
    at = sorted({0, 1, 1023, 1024, v // 3, 262144, 524286, min(524288, v - 1), v // 2, v - 2, v - 1})
    p = torch.from_numpy(rng.integers(32, 64, (4, v)) / 2.0 ** 26).to(TYPES[target])
    q = torch.from_numpy(rng.integers(0, 32, (2, v)) / 2.0 ** 26).to(TYPES[draft]) if draft else None  # (all of it exact)
    pn, qn = p.double().numpy(), q.double().numpy() if draft else None
    tok = np.array([5, 5], np.int32)
    p[0, 5] = pn[0, 5] = 0.0                                  # request 0 rejects its draft, request 1 takes it
    if draft:
        q[:, 5] = torch.tensor([1.0, 1e-9], dtype=q.dtype)
        qn = q.double().numpy()
        res = np.maximum(pn[0] - qn[0], 0.0)
    else:
        res = pn[0]
    a, b = _draws(res, [t for t in at if t != 5]), _draws(pn[3], [t for t in at if t != 5])
    p, q = p.to(gpu), q.to(gpu) if draft else None
    for k, t in enumerate(x for x in at if x != 5):
        o = ge.spec.verify_chains(p, tok, [0, 1, 2], [0.5, 0.0], [a[k], b[k]], draft=q)
        assert o.tolist() == [([t], None), ([5, t], None)], (v, t)
    for u in (0.0, 1.0 - 2.0 ** -53):
        got = ge.spec.verify_chains(p, tok, [0, 1, 2], [0.5, 0.0], [u, u], draft=q).tolist()
        assert got == [(w[0], None) for w in rr.chains(pn, qn, tok, [0, 1, 2], [0.5, 0.0], [u, u])]


@pytest.mark.parametrize("target,draft", [("f64", "f64"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("v", [40, 128257, 600001])
def test_rows_with_nothing_above_the_drafts(ge, gpu, v, target, draft):
    """A draft row nowhere below the target's leaves nothing of it: the token comes from the target's row, read again."""
    rng = np.random.default_rng(v + 1)
    p = torch.from_numpy(rng.integers(32, 64, (4, v)) / 2.0 ** 26).to(TYPES[target])
    pn = p.double().numpy()
    q = (p[[0, 2]].double() * torch.tensor([[1.0], [2.0]])).to(TYPES[draft])
    at = sorted({0, v // 3, v // 2, v - 2, v - 1})
    a, b = _draws(pn[0], at), _draws(pn[2], at)
    p, q = p.to(gpu), q.to(gpu)
    for k, t in enumerate(at):
        o = ge.spec.verify_chains(p, [7, 9], [0, 1, 2], [1.0 - 2.0 ** -53 if k % 2 else 1.0, 0.75], [a[k], b[k]], draft=q)
        want = rr.chains(pn, q.double().cpu().numpy(), [7, 9], [0, 1, 2], [1.0 - 2.0 ** -53 if k % 2 else 1.0, 0.75], [a[k], b[k]])
        assert o.tolist() == [(w[0], None) for w in want] and want[1][0] == [t] and (k % 2 or want[0][0] == [t])


@pytest.mark.parametrize("stacked", [True, False])
@pytest.mark.parametrize("entries", [64, 65, 66, 128, 129, 200])
def test_long_paths(ge, gpu, entries, stacked):
    """Paths of more entries than a wave has lanes, each entry's source the target of one a few places on."""
    rng = np.random.default_rng(entries)
    r, nodes, page, n = 3, 230, 8, 2
    slot = rng.permutation(r * nodes + 30)[:r * nodes]
    anchor = np.arange(r) * nodes
    nd = np.stack([np.r_[0, np.sort(rng.choice(np.arange(1, nodes), entries - 1, replace=False))], np.r_[0, 2:entries + 1],
                   np.arange(entries)]) + anchor[:, None]
    lens = np.array([entries, entries, entries])
    k = torch.from_numpy(rng.integers(-100, 100, (n, -(-(r * nodes + 30) // page), page, 2, 8))).to(torch.bfloat16)
    want, c = k.clone(), k.to(gpu)
    rr.keep_path(lambda s: want[:, s // page, s % page].clone(), lambda s, d: want[:, s // page, s % page].copy_(d), slot, anchor,
                 lens, nd)
    parts = c if stacked else ge.paged.Caches([c[i].clone() for i in range(n)])
    i32 = lambda x: torch.from_numpy(x).int().to(gpu)  # noqa: E731
    ge.paged.keep_path(parts, torch.from_numpy(slot).to(gpu), i32(anchor), i32(lens), i32(nd))
    assert torch.equal((c if stacked else torch.stack(parts.tensors)).cpu(), want)


def test_paths_of_many_requests(ge, gpu):
    """More requests than a launch has rows of workgroups: three nodes each, the third moved behind the anchor."""
    r = 65535 + 70
    g = torch.Generator(device=gpu).manual_seed(1)
    c = torch.randint(0, 100, (1, -(-3 * r // 4), 4, 16), generator=g, device=gpu, dtype=torch.uint8)
    slot = torch.randperm(3 * r, generator=g, device=gpu)
    anchor = torch.arange(0, 3 * r, 3, device=gpu)
    lens = torch.randint(1, 3, (r,), generator=g, device=gpu)
    nodes = torch.stack([anchor, anchor + 2], 1)
    want = c.clone()
    rows, move = want.view(-1, 16), lens == 2
    rows[slot[anchor[move] + 1]] = rows[slot[anchor[move] + 2]].clone()
    ge.paged.keep_path(c, slot, anchor.int(), lens.int(), nodes.int())
    assert torch.equal(c, want) and move[65535:].any()
