"""GPU parity of gsp_verify_chains (spec.verify_chains) against the oracle's chains (fp64, numpy): lengths and tokens exactly
(a draw within rounding of a prefix border has a probability of about 1e-13), the target's weights as their fp32
roundings, exactly."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

from oracle import round_ref as rr
from oracle import sampling_ref as ora
from oracle import spec_ref as spo

pytestmark = pytest.mark.gpu

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _rows(rng, rows, v, dtype, dev, pad=0, zeros=0.3):
    """Probability rows of the type (heavy-tailed, some zeros) in a tensor of v + pad columns, and their values in fp64."""
    w = rng.random((rows, v)) ** 6 * (rng.random((rows, v)) >= zeros) + 1e-9
    w /= w.sum(1, keepdims=True)
    full = torch.full((rows, v + pad), float("nan"), dtype=torch.float64)
    full[:, :v] = torch.from_numpy(w)
    t = full.to(TYPES[dtype]).to(dev)[:, :v]
    return t, t.double().cpu().numpy()


def _batch(rng, lens, v, target="f32", draft="f32", dev=None, pad=0, near=0.6):
    """A ragged batch whose drafts are drawn from q, where q is near p (so that most are accepted)."""
    begin = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    d, r = int(begin[-1]), len(lens)
    t, p = _rows(rng, d + r, v, target, dev, pad)
    row = np.arange(d) + np.repeat(np.arange(r), lens)
    q = dt = None
    mix = p[row] * near + rng.random((d, v)) ** 6 * (1 - near) * 7 / v
    mix /= np.maximum(mix.sum(1, keepdims=True), 1e-300)
    if draft is not None:
        full = torch.zeros((max(d, 1), v + pad), dtype=torch.float64)
        full[:d, :v] = torch.from_numpy(mix)
        dt = full.to(TYPES[draft]).to(dev)[:d, :v]
        q = dt.double().cpu().numpy()
    c = mix.cumsum(1)
    tok = np.array([min(int((c[i] < rng.random() * c[i, -1]).sum()), v - 1) for i in range(d)], np.int32)
    return dict(target=t, tokens=tok, begin=begin, coins=rng.random(d), u=rng.random(r), draft=dt), p, q


def _check(ge, b, p, q, max_drafts=None, expect_error=()):
    o = ge.spec.verify_chains(**b, max_drafts=max_drafts)
    want = rr.chains(p, q, b["tokens"], b["begin"], b["coins"], b["u"])
    n, t, pr, st = (x.cpu().numpy() for x in (o.emit_len, o.tokens, o.probs, o.status))
    k = int(max_drafts if max_drafts is not None else max(np.diff(b["begin"]), default=0))
    assert t.shape == pr.shape == (len(want), k + 1)
    for r, (toks, probs, bad) in enumerate(want):
        assert (t[r, :n[r]].tolist(), st[r]) == (toks, int(bad)), (r, t[r], n[r], st[r], toks, bad)
        assert (t[r, n[r]:] == -1).all() and (pr[r, n[r]:] == 0).all()
        assert np.array_equal(pr[r, :n[r]], np.array(probs, np.float64).astype(np.float32)), (r, pr[r], probs)
    assert {r for r, w in enumerate(want) if w[2]} == set(expect_error)
    assert o.tolist() == [(toks, "error" if bad else None) for toks, _, bad in want]
    return want


SIZES = [1, 2, 63, 64, 65, 255, 256, 257, 1023, 2048, 4095, 4096, 4097, 8191, 16385, 50257, 128256, 262147]


@pytest.mark.parametrize("v", SIZES)
@pytest.mark.parametrize("kind", ["f32-f32", "bf16-none", "f64-f32", "f16-f16", "bf16-bf16", "f32-none", "f32-bf16"])
def test_sizes_and_types(ge, gpu, v, kind):
    """Ragged chains (none, one, several drafts) over every row type, rows with a stride of their own."""
    target, draft = (None if k == "none" else k for k in kind.split("-"))
    rng = np.random.default_rng(v)
    lens = [3, 0, 1, 5, 2] if v > 20000 else [3, 0, 1, 5, 2, 0, 4, 1, 1, 2, 6, 3]
    b, p, q = _batch(rng, lens, v, target, draft, gpu, pad=v % 3)
    want = _check(ge, b, p, q)
    # (a one-hot draft is accepted with the weight of its token alone: rarely over flat rows)
    assert v < 64 or draft is None or len({len(w[0]) for w in want}) > 1


def test_every_pair_of_types(ge, gpu):
    rng = np.random.default_rng(1)
    for target in TYPES:
        for draft in [None, *TYPES]:
            b, p, q = _batch(rng, [2, 3, 0, 1], 1237, target, draft, gpu, pad=5)
            _check(ge, b, p, q)


@pytest.mark.parametrize("target", list(TYPES))
def test_one_hot_drafts_accepted(ge, gpu, target):
    """Deterministic drafts with coins small enough that chains end anywhere."""
    rng = np.random.default_rng(17)
    b, p, q = _batch(rng, [5] * 20, 1500, target, None, gpu)
    row = np.arange(100) + np.repeat(np.arange(20), 5)
    b["coins"] *= 1.6 * p[row, b["tokens"]]
    want = _check(ge, b, p, q)
    assert {len(w[0]) for w in want} >= {1, 2, 3}


@pytest.mark.parametrize("kind", ["f32-bf16", "bf16-none"])
def test_a_draw_per_target_row(ge, gpu, kind):
    """u with an entry per target row: the one of the row drawn from is read."""
    target, draft = (None if k == "none" else k for k in kind.split("-"))
    rng = np.random.default_rng(19)
    lens = [3, 0, 1, 5, 2, 4, 4, 4]
    b, p, q = _batch(rng, lens, 4001, target, draft, gpu)
    b["u"] = rng.random(len(b["tokens"]) + len(lens))
    for coins in (b["coins"], b["coins"] * 0, b["coins"] * 0 + 0.999):
        b["coins"] = coins
        _check(ge, b, p, q)


def test_row_starts_at_every_alignment(ge, gpu):
    """Rows that start at any element of a 16-byte vector, target and draft apart."""
    rng = np.random.default_rng(2)
    for dtype, per in (("bf16", 8), ("f16", 8), ("f32", 4), ("f64", 2)):
        for off in range(per):
            b, p, q = _batch(rng, [2, 1], 5001, dtype, dtype, gpu)
            big = torch.full((p.size + off,), float("nan"), dtype=TYPES[dtype], device=gpu)
            big[off:] = b["target"].reshape(-1)
            b["target"] = big[off:].view(p.shape)
            _check(ge, b, p, q)


def test_many_requests(ge, gpu):
    """More requests than one resident round of workgroups and than the handle's rows."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 4, 700)
    b, p, q = _batch(rng, lens, 3001, "f32", "f32", gpu)
    _check(ge, b, p, q)
    lib = ge._lib
    h = lib.Handle(gpu.index, 1, 64)
    want = rr.chains(p, q, b["tokens"], b["begin"], b["coins"], b["u"])
    for _ in range(2):
        _, n, t, st = _raw(ge, h, b, 3, gpu)
        assert n.cpu().tolist() == [len(w[0]) for w in want]
        assert [t[r, :len(w[0])].tolist() for r, w in enumerate(want)] == [w[0] for w in want]


def _raw(ge, h, b, most, gpu, probs=False, stream=None, **kw):
    """gsp_verify_chains through the C ABI: (return code, emit_len, emit_tokens, status), without emit_probs by default."""
    lib = ge._lib
    dev = lambda x, t: torch.from_numpy(np.ascontiguousarray(x)).to(gpu, t)  # noqa: E731
    keep = [dev(b["tokens"], torch.int32), dev(b["begin"], torch.int32), dev(b["coins"], torch.float64), dev(b["u"], torch.float64)]
    r = len(b["u"])
    n, st = (torch.full((r,), -7, dtype=torch.int32, device=gpu) for _ in range(2))
    t = torch.full((r, most + 4), -7, dtype=torch.int32, device=gpu)
    c = lib.Chains()
    c.size, c.requests, c.vocab, c.max_drafts, c.drafts = C.sizeof(lib.Chains), r, b["target"].shape[1], most, len(b["tokens"])
    c.target_type, c.target, c.target_ld = ge.spec._PROB[b["target"].dtype], b["target"].data_ptr(), b["target"].stride(0)
    if b["draft"] is not None:
        c.draft_type, c.draft, c.draft_ld = ge.spec._PROB[b["draft"].dtype], b["draft"].data_ptr(), b["draft"].stride(0)
    c.token, c.begin, c.coin, c.u = (x.data_ptr() for x in keep)
    c.emit_len, c.emit_tokens, c.emit_ld, c.status = n.data_ptr(), t.data_ptr(), most + 4, st.data_ptr()
    c.stream = torch.cuda.current_stream(gpu).cuda_stream
    for k, val in kw.items():
        setattr(c, k, val)
    with h.lock:
        rc = h.L.gsp_verify_chains(h.h, C.byref(c))
    torch.cuda.synchronize()
    return rc, n, t, st


def test_columns_past_the_chains_are_left(ge, gpu):
    rng = np.random.default_rng(4)
    b, p, q = _batch(rng, [2, 0, 1], 500, "f32", "f32", gpu)
    rc, n, t, st = _raw(ge, ge._lib.handle(gpu.index, 1, 500), b, 2, gpu)
    assert rc == 0 and (t[:, 3:] == -7).all() and (t[:, :3] != -7).all()


def test_c_refusals(ge, gpu):
    """Bad arguments are errors with a text, and nothing is launched."""
    rng = np.random.default_rng(5)
    b, p, q = _batch(rng, [2, 0, 1], 500, "f32", "f32", gpu)
    lib = ge._lib
    h = lib.handle(gpu.index, 1, 500)
    for kw, rc, text in ((dict(target=None), lib.E_ARG, "required"), (dict(u=None), lib.E_ARG, "required"),
                         (dict(coin=None), lib.E_ARG, "token and coin"), (dict(target_type=4), lib.E_ARG, "type"),
                         (dict(draft_type=9), lib.E_ARG, "type"), (dict(target_ld=499), lib.E_ARG, "target_ld"),
                         (dict(draft_ld=1), lib.E_ARG, "draft_ld"), (dict(vocab=0), lib.E_ARG, "vocab"),
                         (dict(emit_ld=2), lib.E_ARG, "emit_ld"), (dict(u_rows=2), lib.E_ARG, "u_rows"), (dict(size=4), lib.E_ARG, "short"),
                         (dict(max_drafts=(1 << 30) + 1, emit_ld=1 << 40), lib.E_UNSUPPORTED, "2^30"),
                         (dict(drafts=1 << 30), lib.E_UNSUPPORTED, "2^30")):
        got, n, t, st = _raw(ge, h, b, 2, gpu, **kw)
        assert got == rc and text in h.L.gse_last_error(h.h).decode(), (kw, got, h.L.gse_last_error(h.h))
        assert (n == -7).all() and (t == -7).all() and (st == -7).all()
    assert _raw(ge, h, b, 2, gpu, requests=0)[0] == 0
    small = lib.Handle(gpu.index, 1, 64)  # (room for a row of 2 * 64 segments)
    got, n, t, st = _raw(ge, small, b, 2, gpu, vocab=200000, target_ld=200000, draft_ld=200000)
    assert got == lib.E_CAPACITY and "200000" in small.L.gse_last_error(small.h).decode() and (n == -7).all()
    with pytest.raises(ValueError):
        ge.spec.verify_chains(**{**b, "begin": torch.tensor(b["begin"], device=gpu)})  # its longest chain is not known


def test_edges_of_the_random_numbers(ge, gpu):
    """u at 0 and just below 1 (and past it), coins at 0, at the exact ratio and not a number."""
    v, rng = 9001, np.random.default_rng(6)
    lens = [2] * 8
    b, p, q = _batch(rng, lens, v, "f64", "f64", gpu, near=0.0)
    b["u"] = np.array([0.0, 1 - 2.0 ** -53, 1.0, 2.0, -1.0, np.nan, 0.5, 2.0 ** -60])
    row = np.arange(16) + np.repeat(np.arange(8), 2)
    qx, px = q[np.arange(16), b["tokens"]], p[row, b["tokens"]]
    b["coins"][0::4] = 0.0                             # accepted where p and q are positive
    b["coins"][1::4] = np.nan                          # rejected
    b["coins"][2::4] = px[2::4] / qx[2::4]             # at the border: rounds to either side
    for u_first in range(8):
        b["u"] = np.roll(b["u"], 1)
        _check(ge, b, p, q)


def test_special_values(ge, gpu):
    """Rows of zeros, of one token, with negative entries, NaN and infinities in the row drawn from and in the others."""
    v = 700
    rng = np.random.default_rng(7)
    for dtype in ("f32", "bf16", "f64"):
        b, p, q = _batch(rng, [1] * 12, v, dtype, dtype, gpu, near=0.0)
        t, d = b["target"].clone(), b["draft"].clone()
        b["coins"][:] = 0.9999
        for r in range(12):                      # a draft that is rejected for certain ...
            b["tokens"][r] = 13
            t[2 * r, 13], d[r, 13] = 0.0, 0.5
        t[0, 600] = float("nan")                 # request 0: a NaN in the row it draws from
        d[1, 5] = float("nan")
        t[4, 699] = float("inf")
        t[6, 0] = float("-inf")
        d[4, 1] = float("inf")
        t[10], d[5] = 0.0, 0.25                  # nothing left above q, and nothing in p
        t[12], d[6] = d[6] * 0.5, d[6]           # nothing left above q: drawn from p
        t[14] = -1.0                             # all negative
        t[16], t[16, 300] = -0.25, 2.0           # one positive
        t[18, 13], b["coins"][9] = 1.0, 0.0      # ... but request 9's is accepted, and its next row is
        t[19] = float("nan")                     # not valid: one token, then an error
        t[20, 13], b["coins"][10] = 1.0, 0.0
        t[21] = 0.0
        t[21, 699] = 1e-7                        # a single tiny weight
        t[23, 44] = float("nan")                 # request 11: the row after a rejected draft is not read
        b["target"], b["draft"] = t, d
        p, q = t.double().cpu().numpy(), d.double().cpu().numpy()
        want = _check(ge, b, p, q, expect_error={0, 1, 2, 3, 4, 5, 7, 9})
        assert want[8][0] == [300] and want[10][0] == [13, 699] and len(want[9][0]) == 1


@pytest.mark.parametrize("target", list(TYPES))
def test_smallest_weights_count(ge, gpu, target):
    """Rows whose weights are the type's smallest (fp64: small ones): they are summed and drawn from like any other,
    subnormal or not."""
    tiny = {"f64": 2.0 ** -1000, "f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[target]
    v, rng = 3001, np.random.default_rng(18)
    t = torch.zeros((8, v), dtype=TYPES[target], device=gpu)
    at = rng.choice(v, 5, replace=False)
    for k, x in enumerate(at):
        t[:, int(x)] = tiny * (k + 1)
    p = t.double().cpu().numpy()
    assert (p[0] > 0).sum() == 5
    b = dict(target=t, tokens=np.zeros(0, np.int32), begin=[0] * 9, coins=np.zeros(0), u=np.linspace(0.01, 0.99, 8), draft=None)
    want = _check(ge, b, p, None)
    assert len({w[0][0] for w in want}) > 2


def test_nothing_left_with_a_one_hot_draft(ge, gpu):
    """A deterministic draft that holds all of its row's mass and is rejected all the same (0.9 < coin) is drawn again; and
    a NaN at the draft's own token does not count among the rest."""
    p = np.zeros((4, 300))
    p[0, 7], p[1, 0] = 0.9, 1.0
    p[2] = 1 / 300
    p[2, 7] = np.nan
    p[3, 0] = 1.0
    b = dict(target=torch.from_numpy(p).to(gpu), tokens=np.array([7, 7]), begin=[0, 1, 2], coins=np.array([0.95, 0.1]),
             u=np.array([0.3, 0.3]), draft=None)
    want = _check(ge, b, p, None)
    assert want[0][0] == [7]


def test_padded_and_foreign_tokens_end_a_chain(ge, gpu):
    """Equal chains padded with -1, and tokens past the vocabulary: the chain ends there and the token comes from that row."""
    rng = np.random.default_rng(8)
    b, p, q = _batch(rng, [4] * 6, 333, "f32", "f32", gpu, near=1.0)
    b["coins"] *= 1e-3
    b["tokens"][[0, 5, 6, 7, 10, 11, 15]] = [-1, -1, -1, -1, 333, 2 ** 31 - 1, -2 ** 31]
    want = _check(ge, b, p, q)
    assert len(want[0][0]) == 1
    wide = dict(b, tokens=torch.from_numpy(b["tokens"].astype(np.int64)))
    wide["tokens"][10:12] = 2 ** 40 + 5
    assert ge.spec.verify_chains(**wide).tolist() == [(w[0], None) for w in want]


def test_long_chains(ge, gpu):
    """Chains past a wave's 64 drafts, ending inside and at the ends of its rounds."""
    rng = np.random.default_rng(9)
    lens = [130, 64, 65, 63, 128, 200]
    b, p, q = _batch(rng, lens, 97, "f32", "f32", gpu, near=1.0)
    b["coins"][:] = 0.0
    qx = q[np.arange(len(b["tokens"])), b["tokens"]]
    want = _check(ge, b, p, q, max_drafts=201)
    assert [len(w[0]) for w in want if not w[2]] == [n + 1 for n in lens] and qx.min() > 0
    for r, at in enumerate([64, 63, 64, 0, 127, 199]):
        b["coins"][b["begin"][r] + at] = np.nan
    want = _check(ge, b, p, q)
    assert [len(w[0]) for w in want] == [65, 64, 65, 1, 128, 200]


def test_no_drafts_and_no_requests(ge, gpu):
    rng = np.random.default_rng(10)
    b, p, q = _batch(rng, [0, 0, 0], 801, "bf16", "bf16", gpu)
    _check(ge, b, p, q)
    o = ge.spec.verify_chains(b["target"][:0], [], [0], [], [])
    assert o.tolist() == [] and o.tokens.shape == (0, 1)


def test_offsets_out_of_order(ge, gpu):
    """Requests whose offsets descend, pass the drafts or the longest chain: an error each, nothing of theirs is read; the
    others are answered."""
    rng = np.random.default_rng(11)
    b, p, q = _batch(rng, [2, 2, 2], 333, "f32", "f32", gpu)
    b["begin"] = np.array([0, 2, 1, 6, 7, -3, 2 ** 31 - 1], np.int32)
    b["u"] = rng.random(6)
    b["target"] = torch.cat([b["target"]] * 2)[:12].contiguous()
    p = b["target"].double().cpu().numpy()
    o = ge.spec.verify_chains(**b, max_drafts=4)
    assert o.status.cpu().tolist() == [0, 1, 1, 1, 1, 1] and o.emit_len.cpu().tolist()[1:] == [0] * 5
    assert (o.tokens[1:] == -1).all() and (o.probs[1:] == 0).all()
    assert o.tolist()[0][0] == rr.chain(p[:3], q[:2], b["tokens"][:2], b["coins"][:2], b["u"][0])[0]


@pytest.mark.parametrize("r,drafts,dtype", [(1040, 0, "bf16"), (600, 1, "bf16"), (260, 1, "f32"), (140, 1, "f64")])
def test_calls_past_the_last_level_cache(ge, gpu, r, drafts, dtype):
    """Calls of more than 256 MB of rows: the same answers, over an odd vocabulary, against fp64 sums row by row."""
    v = 130001
    g = torch.Generator(device=gpu).manual_seed(r)
    n = r * (drafts + 1)
    p = torch.rand((n, v), generator=g, device=gpu).pow_(8).to(TYPES[dtype])
    q = torch.rand((r, v), generator=g, device=gpu).pow_(8).to(TYPES[dtype]) if drafts else None
    assert r * v * p.element_size() * (2 if drafts else 1) >= 256 << 20
    tok = torch.randint(0, v, (r * drafts,), generator=g, device=gpu, dtype=torch.int32)
    coin, u = (torch.rand(k, generator=g, device=gpu, dtype=torch.float64) for k in (r * drafts, r))
    o = ge.spec.verify_chains(p, tok, torch.arange(0, r * drafts + 1, max(drafts, 1), dtype=torch.int32, device=gpu)
                              if drafts else torch.zeros(r + 1, dtype=torch.int32, device=gpu), coin, u, draft=q, max_drafts=drafts)
    want = []
    for k in range(r):
        row = p[k * (drafts + 1)].double()
        if drafts:
            x = int(tok[k])
            if bool(q[k, x] > 0) and bool(coin[k] * q[k, x].double() < row[x]):
                row, first = p[2 * k + 1].double(), [x]
            else:
                row, first = (row - q[k].double()).clamp(min=0), []
        else:
            first = []
        c = row.cumsum(0)
        want.append((first + [int(torch.searchsorted(c, u[k] * c[-1]))], None))
    assert o.tolist() == want
    if drafts:
        assert 0 < sum(len(w[0]) for w in want) - r < r


def test_rows_past_32_bits(ge, gpu):
    """Rows more than 2^31 elements (and 2^32 bytes) into the tensors."""
    v, d = 262144, 8198
    target = torch.zeros((d + 1, v), dtype=torch.bfloat16, device=gpu)
    draft = torch.zeros((d, v), dtype=torch.bfloat16, device=gpu)
    rng = np.random.default_rng(12)
    tail, p, q = _batch(rng, [3], v, "bf16", "bf16", gpu, near=0.9)
    target[d - 3:], draft[d - 3:] = tail["target"], tail["draft"]
    for coins in ([0.0, 0.0, 0.99999], [0.0, 0.99999, 0.0], [0.0, 0.0, 0.0]):
        tok = np.zeros(d, np.int32)
        tok[d - 3:] = tail["tokens"]
        c = np.zeros(d)
        c[d - 3:] = coins
        o = ge.spec.verify_chains(target, tok, [d - 3, d], c, tail["u"], draft=draft)
        assert o.tolist() == [(rr.chain(p, q, tail["tokens"], coins, tail["u"][0])[0], None)]


def test_same_answers_for_a_row_whatever_else_the_call_holds(ge, gpu):
    """A request's answer does not depend on the batch around it, nor on the run."""
    rng = np.random.default_rng(13)
    b, p, q = _batch(rng, [3, 1, 4, 0, 2], 50257, "f32", "bf16", gpu)
    first = ge.spec.verify_chains(**b)
    for _ in range(3):
        again = ge.spec.verify_chains(**b)
        assert torch.equal(first.tokens, again.tokens) and torch.equal(first.probs, again.probs)
    for r in range(5):
        s, e = b["begin"][r], b["begin"][r + 1]
        one = dict(target=b["target"][s + r:e + r + 1], tokens=b["tokens"][s:e], begin=[0, e - s], coins=b["coins"][s:e],
                   u=b["u"][r:r + 1], draft=b["draft"][s:e])
        assert ge.spec.verify_chains(**one).tolist() == [first.tolist()[r]]


def test_in_a_graph(ge, gpu):
    """A captured call replayed over new inputs, with eager calls of the same handle's stream in between."""
    rng = np.random.default_rng(14)
    lens = [3, 0, 2, 5]
    sets = [_batch(rng, lens, 20011, "f32", "f32", gpu) for _ in range(3)]
    dev = {k: torch.from_numpy(np.asarray(x)).to(gpu) if not isinstance(x, torch.Tensor) else x.clone()
           for k, x in sets[0][0].items()}
    dev["begin"] = dev["begin"].int()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        ge.spec.verify_chains(**dev, max_drafts=5)  # (opens the stream's handle)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o = ge.spec.verify_chains(**dev, max_drafts=5)
        for k in (0, 1, 2, 1, 0, 2):
            for name, x in sets[k][0].items():
                dev[name].copy_(x if isinstance(x, torch.Tensor) else torch.from_numpy(np.asarray(x)))
            o.tokens.fill_(-9)
            o.emit_len.fill_(-9)
            g.replay()
            s.synchronize()
            want = rr.chains(sets[k][1], sets[k][2], *(sets[k][0][n] for n in ("tokens", "begin", "coins", "u")))
            assert o.tolist() == [(w[0], None) for w in want]
            eager = ge.spec.verify_chains(**dev, max_drafts=5)
            assert eager.tolist() == o.tolist()


def test_two_graphs_of_one_handle(ge, gpu):
    """Two captured calls that share a stream's workspace, replayed in turn on it."""
    rng = np.random.default_rng(20)
    sets = [_batch(rng, lens, v, "bf16", "f32", gpu) for lens, v in (([2, 4, 0], 30011), ([1] * 40, 7001))]
    want = [[(w[0], None) for w in rr.chains(p, q, *(b[n] for n in ("tokens", "begin", "coins", "u")))] for b, p, q in sets]
    devs = []
    for b, _, _ in sets:
        d = {k: torch.from_numpy(np.asarray(x)).to(gpu) if not isinstance(x, torch.Tensor) else x for k, x in b.items()}
        devs.append(dict(d, begin=d["begin"].int()))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graphs, outs = [], []
        for d in devs:
            ge.spec.verify_chains(**d, max_drafts=4)  # (opens the stream's handle, at this vocabulary)
        s.synchronize()
        for d in devs:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                outs.append(ge.spec.verify_chains(**d, max_drafts=4))
        for k in (0, 1, 1, 0, 0, 1):
            outs[k].tokens.fill_(-9)
            graphs[k].replay()
            assert outs[k].tolist() == want[k]
            assert ge.spec.verify_chains(**devs[1 - k], max_drafts=4).tolist() == want[1 - k]


def test_two_threads_on_one_stream(ge, gpu):
    """Calls of two threads on the same stream share its handle: one after the other on the device."""
    rng = np.random.default_rng(21)
    sets = [_batch(rng, [3, 1, 0, 5], 20001, "f32", "f32", gpu) for _ in range(2)]
    want = [[(w[0], None) for w in rr.chains(p, q, *(b[n] for n in ("tokens", "begin", "coins", "u")))] for b, p, q in sets]
    bad = []

    def work(k):
        for _ in range(30):
            if ge.spec.verify_chains(**sets[k][0]).tolist() != want[k]:
                bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_streams(ge, gpu):
    """Calls on two streams at once: a handle each."""
    rng = np.random.default_rng(15)
    sets = [_batch(rng, [3] * 16, 50257, "f32", "f32", gpu) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(6):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                outs[k].append(ge.spec.verify_chains(**sets[k][0]))
    torch.cuda.synchronize()
    for k in range(2):
        want = [(w[0], None) for w in rr.chains(sets[k][1], sets[k][2], *(sets[k][0][n] for n in ("tokens", "begin", "coins", "u")))]
        assert all(o.tolist() == want for o in outs[k])


def test_draws_follow_the_residual(ge, gpu):
    """dist, qprob, verify_chains in a row against the verify round over logits (gse_verify_tree) with the same random
    numbers: a strict chain's emitted tokens and path."""
    S = ge.sampling.SamplingParams
    rng = np.random.default_rng(16)
    v, lens, nout = 32003, [4, 1, 0, 3, 5, 2], 11
    begin = np.concatenate([[0], np.cumsum(lens)])
    d, r = int(begin[-1]), len(lens)
    g = torch.Generator(device=gpu).manual_seed(5)
    x = torch.randn((d + r, v), generator=g, device=gpu) * 2
    row = torch.from_numpy(np.arange(d) + np.repeat(np.arange(r), lens)).to(gpu)
    y = x[row] + 0.4 * torch.randn((d, v), generator=g, device=gpu)
    q = ge.spec.qprob(y, 0.9)
    tok = [ge.sampling.draw(q[i], float(rng.random())) for i in range(d)]
    params = [S(temperature=0.9, accept="rejection", top_p=1.0 if k % 2 else 0.97) for k in range(r)]
    per_row = [params[k] for k in range(r) for _ in range(lens[k] + 1)]
    p = ge.sampling.dist_batch(x, per_row)
    seeds = [int(s) for s in rng.integers(0, 2 ** 63, r)]
    reqs = [dict(target=x[begin[k] + k:begin[k + 1] + k + 1], tokens=tok[begin[k]:begin[k + 1]], parents=list(range(lens[k])),
                 params=params[k], seed=seeds[k], nout=nout, q=[q[i] for i in range(begin[k], begin[k + 1])] or None)
            for k in range(r)]
    tree = ge.spec.verify_tree(reqs)
    coins = [ora.uniform(ora.mix(seeds[k], spo.SALT_ACC), nout + i) for k in range(r) for i in range(lens[k])]
    u = [ora.uniform(ora.mix(seeds[k], spo.SALT_RES), nout + i) for k in range(r) for i in range(lens[k] + 1)]  # per row
    got = ge.spec.verify_chains(p, tok, begin, coins, u, draft=q)
    for k in range(r):
        toks, path, _ = tree[k]
        mine = got.tolist()[k][0]
        a = len(toks) - 1
        assert len(mine) == len(toks) and mine[:a] == toks[:a]
        if a < lens[k]:  # (a leaf samples in descending order of probability, a chain's last row in vocabulary order)
            assert mine == toks, k
