"""Timing cases of the operators over a paged cache of keys and values, and of beam search over it.

A case is a dict of plain values; "kind" says which operator one pass calls:

  write    kv.write: the keys and values of new tokens to their cache slots, as they are or in 8 bits with a scale per token
           and head
  read     kv.read: cached tokens of many requests as contiguous rows, out of 8 bits or as they are
  attend   kv.attend: each request's new tokens (one, a chain, a draft tree) against its cached keys and values
  beam     beam.select: the best continuations over a request's beams and the vocabulary
  reorder  kv.reorder: the cached tokens of beams moved to the beams that continue them

The plain forms below compute the same from elementary tensor operations. Inputs are drawn on the GPU from the seed.
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8,
         "u8": torch.uint8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "i8": 1, "u8": 1}
MOST = {"e4m3": 448.0, "i8": 127.0}  # the largest value that 8 bits hold
TINY = 2.0 ** -126                   # the smallest scale: a row of zeros has it


def listed():
    return [
        # a serving batch's decode step: one token a request, into an 8-bit cache
        dict(name="write_decode_64", kind="write", tokens=64, heads=8, dim=128, page=16, source="bf16", cache="e4m3",
             heads_first=False, pool=1024),
        # a chunk of prompts, an 8-bit integer cache with the heads ahead of the page's tokens, odd head counts and sizes
        dict(name="write_prompts_16384", kind="write", tokens=16384, heads=5, dim=80, page=24, source="f16", cache="i8",
             heads_first=True, pool=1000),
        # a few short requests read back (a prefix that a library's kernel then attends to)
        dict(name="read_4", kind="read", requests=4, context=512, heads=8, dim=128, page=16, cache="e4m3", out="bf16",
             heads_first=False),
        # a batch of contexts moved out of the cache
        dict(name="read_heads_32", kind="read", requests=32, context=8192, heads=5, dim=80, page=24, cache="i8", out="f16",
             heads_first=True),
        # one user's decode step over a long chat
        dict(name="attend_chat_1", kind="attend", requests=1, context=8192, new=1, tree=False, group=4, heads=8, dim=128,
             page=16, cache="bf16", query="bf16", heads_first=False),
        # a round of tree verification: nine nodes a request, two chains of four from the anchor
        dict(name="attend_tree_96", kind="attend", requests=96, context=4096, new=9, tree=True, group=4, heads=8, dim=128,
             page=32, cache="bf16", query="bf16", heads_first=False),
        # chains of drafts, ragged, over an 8-bit integer cache with odd sizes; requests without a token
        dict(name="attend_chain_24", kind="attend", requests=24, context=3000, new=6, tree=False, group=3, heads=5, dim=80,
             page=24, cache="i8", query="f16", heads_first=True),
        # a large decode batch over long 8-bit contexts
        dict(name="attend_batch_128", kind="attend", requests=128, context=16384, new=1, tree=False, group=8, heads=8,
             dim=128, page=64, cache="e4m3", query="bf16", heads_first=False),
        # one user's beams
        dict(name="beam_1x4", kind="beam", requests=1, beams=4, keep=8, vocab=128256, logits="f32"),
        # a batch of beam searches over half-precision logits
        dict(name="beam_64x8", kind="beam", requests=64, beams=8, keep=16, vocab=151936, logits="bf16"),
        # the beams' first tokens, every layer's keys and values
        dict(name="reorder_1x4", kind="reorder", requests=1, beams=4, tokens=16, caches=64, heads=8, dim=128, page=16,
             cache="bf16", heads_first=False),
        # a batch of beams deep in their answers, an 8-bit cache
        dict(name="reorder_8x8", kind="reorder", requests=8, beams=8, tokens=256, caches=48, heads=5, dim=80, page=24,
             cache="u8", heads_first=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "beam", "reorder"])
    heads, dim = rng.randint(1, 8), rng.choice([64, 72, 80, 96, 128])
    page, first = rng.choice([1, 8, 16, 24, 32, 64, 128]), rng.random() < 0.4
    half = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice(["e4m3", "i8", half])
    if kind == "write":
        tokens = _log_int(rng, 1, 16384)
        return dict(kind=kind, tokens=tokens, heads=heads, dim=dim, page=page, source=rng.choice([half, "f32"]), cache=cache,
                    heads_first=first, pool=(tokens + 4096) // page + 3)
    if kind == "read":
        return dict(kind=kind, requests=_log_int(rng, 1, 32), context=_log_int(rng, 64, 8192), heads=heads, dim=dim, page=page,
                    cache=cache, out=half, heads_first=first)
    if kind == "attend":
        requests = _log_int(rng, 1, 128)
        context = _log_int(rng, 128, 131072 if requests == 1 else 16384 if requests < 8 else 8192)
        tree = rng.random() < 0.3
        new = 9 if tree else rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 40)])
        group = rng.choice([1, 2, 3, 4, 8])
        context = max(128, min(context, (1 << 33) // (requests * new * group * heads * dim)))
        return dict(kind=kind, requests=requests, context=context, new=new, tree=tree, group=group, heads=heads, dim=dim,
                    page=page, cache=cache, query=half, heads_first=first)
    if kind == "beam":
        beams, requests = rng.randint(2, 8), _log_int(rng, 1, 64)
        vocab = rng.choice([32000, 50257, 128256, 151936]) if rng.random() < 0.4 else _log_int(rng, 4000, 151936)
        return dict(kind=kind, requests=requests, beams=beams, keep=rng.choice([beams, 2 * beams]), vocab=vocab,
                    logits=rng.choice(["f32", "bf16"]) if requests <= 32 else "bf16")
    return dict(kind=kind, requests=_log_int(rng, 1, 8), beams=rng.randint(2, 8), tokens=_log_int(rng, 1, 256),
                caches=2 * rng.randint(4, 24), heads=rng.randint(1, 5), dim=rng.choice([64, 72, 80]), page=page,
                cache=rng.choice(["bf16", "u8"]), heads_first=first)


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _rand(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def _kv_values(g, heads, dim, shape):
    """Keys or values: channels of different sizes, some tokens larger than others."""
    channel = torch.exp(0.5 * _rand(g, heads, dim))
    return _rand(g, *shape, heads, dim).mul_(channel).mul_(torch.exp(0.3 * _rand(g, *shape, 1, 1)))


def _quantise(x, kind):
    """Rows in 8 bits: scale = max |x| / most, at least TINY; the values x / scale, rounded to nearest, ties to even."""
    scale = (x.abs().amax(-1) * np.float32(1 / MOST[kind])).clamp(min=TINY)
    x = x * (torch.ones_like(scale) / scale)[..., None]
    return (x.round().to(torch.int8) if kind == "i8" else x.to(torch.float8_e4m3fn)), scale


def _first(t, heads_first):
    """[pages, page, heads, ...] with the heads ahead of the page's tokens, where the case has them so."""
    return t.transpose(1, 2).contiguous() if heads_first else t


def _cache(g, case, pages, page):
    """Keys, values and, in 8 bits, their scales, of `pages` pages."""
    def one():
        parts, scales = [], []
        for p in range(0, pages, 1 + (1 << 28) // (page * case["heads"] * case["dim"])):  # (a billion bytes of fp32 at a time)
            n = min(pages, p + 1 + (1 << 28) // (page * case["heads"] * case["dim"])) - p
            x = _kv_values(g, case["heads"], case["dim"], (n, page))
            if case["cache"] in MOST:
                x, s = _quantise(x, case["cache"])
                scales.append(_first(s, case["heads_first"]))
            parts.append(_first(x.to(DTYPE[case["cache"]]), case["heads_first"]))
        return torch.cat(parts), torch.cat(scales) if scales else None
    (k, ks), (v, vs) = one(), one()
    return k, v, (ks, vs) if ks is not None else None


def _table(g, case, lengths, page, most):
    """Each request's pages, drawn from a pool that is a little larger than they need; -1 past them."""
    width = (most + page - 1) // page + 1
    held = (lengths + page - 1) // page
    used = int(held.sum())
    ids = torch.randperm(used + 3, generator=g, device=g.device).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=g.device)
    table[torch.arange(width, device=g.device) < held[:, None]] = ids[:used]
    return table, used + 3


def _between(g, lo, hi, n):
    """n whole numbers spread over lo .. hi, hi among them, in an order of the seed's (so that sums are the case's alone)."""
    x = hi - (hi - lo) * torch.arange(n, device=g.device) // max(n - 1, 1)
    return x[torch.randperm(n, generator=g, device=g.device)]


def _prepare_write(case, g):
    n, page, pool = case["tokens"], case["page"], case["pool"]
    state = dict(kind="write", cache=case["cache"], heads_first=case["heads_first"])
    for name in "kv":
        state[name] = _kv_values(g, case["heads"], case["dim"], (n,)).to(DTYPE[case["source"]])
    slot = torch.randperm(pool * page, generator=g, device=g.device)[:n]
    if n >= 32:  # (a batch of fixed size: its last places are empty)
        slot[-(n // 32):] = -1
    shape = (pool, case["heads"], page) if case["heads_first"] else (pool, page, case["heads"])
    for name in ("keys", "values"):
        state[name] = torch.zeros((*shape, case["dim"]), device=g.device).to(DTYPE[case["cache"]])
    state["scales"] = tuple(torch.zeros(shape, device=g.device) for _ in range(2)) if case["cache"] in MOST else None
    return dict(state, slot=slot)


def _prepare_read(case, g):
    r, page = case["requests"], case["page"]
    n = _between(g, case["context"] // 2, case["context"], r)
    first = torch.where(n % 2 == 0, 0, n // 4)
    begin = torch.zeros(r + 1, dtype=torch.int64, device=g.device)
    begin[1:] = (n - first).cumsum(0)
    table, pages = _table(g, case, n, page, case["context"])
    k, v, scales = _cache(g, case, pages, page)
    return dict(kind="read", keys=k, values=v, scales=scales, table=table, begin=begin.int(), first=first.int(),
                rows=int(begin[-1]), out=case["out"], heads_first=case["heads_first"])


def _prepare_attend(case, g):
    r, page, new = case["requests"], case["page"], case["new"]
    context = _between(g, case["context"] // 4, case["context"], r)
    n = torch.full((r,), new, device=g.device) if case["tree"] or new == 1 else _between(g, 1, new, r)
    if r >= 8 and not case["tree"]:  # a place of the batch without a request
        n[-1], n[-2], context[-1] = 0, new, 0
        n[:-2] = new if new == 1 else _between(g, 1, new, r - 2)
    length = context + n
    begin = torch.zeros(r + 1, dtype=torch.int64, device=g.device)
    begin[1:] = n.cumsum(0)
    rows = int(begin[-1])
    table, pages = _table(g, case, length, page, case["context"] + new)
    k, v, scales = _cache(g, case, pages, page)
    q = _rand(g, rows, case["group"] * case["heads"], case["dim"]).to(DTYPE[case["query"]])
    parents = None
    if case["tree"]:  # chains of four from the anchor
        node = torch.arange(new, device=g.device)
        node = torch.where(node % 4 == 1, 0, node - 1)
        parents = torch.where(node < 0, -1, node + begin[:-1, None]).reshape(-1).int()
    return dict(kind="attend", q=q, keys=k, values=v, scales=scales, table=table, begin=begin.int(), seq_len=length.int(),
                parents=parents, new=new, heads_first=case["heads_first"])


def _prepare_beam(case, g):
    rows, v = case["requests"] * case["beams"], case["vocab"]
    slope = torch.empty(v, device=g.device)  # rows like a trained model's: a Zipf slope over the row's own ranking of the tokens
    slope[torch.randperm(v, generator=g, device=g.device)] = -1.1 * torch.log1p(torch.arange(v, device=g.device).float())
    turn = torch.randint(0, v, (rows,), generator=g, device=g.device)
    x = torch.cat([slope, slope[:-1]]).unfold(0, v, 1)[turn].add_(_rand(g, rows, v).mul_(2.5))
    scores = -30 * torch.rand((case["requests"], 1), generator=g, device=g.device) \
        - torch.rand((case["requests"], case["beams"]), generator=g, device=g.device).mul_(3).cumsum(1)
    return dict(kind="beam", logits=x.to(DTYPE[case["logits"]]), scores=scores, keep=case["keep"])


def _prepare_reorder(case, g):
    r, b, page = case["requests"], case["beams"], case["page"]
    prompt = _between(g, 1, 256, r)
    length = (prompt + case["tokens"]).repeat_interleave(b)
    table, pages = _table(g, case, length, page, 256 + case["tokens"])
    shape = (case["heads"], page) if case["heads_first"] else (page, case["heads"])
    bits = torch.randint(-128, 128, (case["caches"], pages, *shape, case["dim"]), generator=g, device=g.device, dtype=torch.int8)
    parents = torch.randint(0, b, (r, b), generator=g, device=g.device)
    parents[0, 0] = b - 1
    return dict(kind="reorder", caches=bits.view(torch.uint8) if case["cache"] == "u8" else bits.to(DTYPE[case["cache"]]),
                table=table, seq_len=length.int(), first=prompt.int(), parents=parents.int(), page=page, most=case["tokens"],
                heads_first=case["heads_first"])


def prepare(case, seed):
    g = torch.Generator(device=torch.device("cuda", torch.cuda.current_device())).manual_seed(seed & 0x7FFFFFFF)
    return dict(write=_prepare_write, read=_prepare_read, attend=_prepare_attend, beam=_prepare_beam,
                reorder=_prepare_reorder)[case["kind"]](case, g)


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _put(cache, slot, rows, heads_first):
    page = cache.shape[2 if heads_first else 1]
    if heads_first:
        cache[slot // page, :, slot % page] = rows
    else:
        cache[slot // page, slot % page] = rows


def _get(cache, scale, ids, offset, heads_first):
    """The cached rows at pages `ids` and places `offset`, in fp32."""
    at = (ids, slice(None), offset) if heads_first else (ids, offset)
    x = cache[at].float()
    return x if scale is None else x * scale[at][..., None]


def _write(s):
    real = s["slot"] >= 0
    slot = s["slot"][real]
    for i, (name, cache) in enumerate((("k", s["keys"]), ("v", s["values"]))):
        x = s[name][real].float()
        if s["scales"] is None:
            _put(cache, slot, x.to(cache.dtype), s["heads_first"])
            continue
        x, scale = _quantise(x, s["cache"])
        if s["cache"] == "e4m3":  # (torch stores 8-bit floats by index as bytes)
            cache, x = cache.view(torch.uint8), x.view(torch.uint8)
        _put(cache, slot, x, s["heads_first"])
        _put(s["scales"][i], slot, scale, s["heads_first"])
    return dict(keys=s["keys"], values=s["values"], scales=s["scales"])


def _read(s):
    page = s["keys"].shape[2 if s["heads_first"] else 1]
    row = torch.arange(s["rows"], device=s["begin"].device)
    req = torch.searchsorted(s["begin"][1:].long(), row, right=True)
    at = row - s["begin"][req] + s["first"][req]
    ids = s["table"][req, at // page]
    ks, vs = s["scales"] or (None, None)
    return dict(k=_get(s["keys"], ks, ids, at % page, s["heads_first"]).to(DTYPE[s["out"]]),
                v=_get(s["values"], vs, ids, at % page, s["heads_first"]).to(DTYPE[s["out"]]))


def _attend(s):
    """softmax(q k / sqrt(dim)) v over what each new token sees: the tokens before its request's new ones, and of those itself
    and the earlier ones, with `parents` its ancestors alone."""
    q, begin, length, dev = s["q"], s["begin"].long(), s["seq_len"].long(), s["q"].device
    page = s["keys"].shape[2 if s["heads_first"] else 1]
    heads, dim = s["keys"].shape[1 if s["heads_first"] else 2], q.shape[2]
    r, n, group = len(length), s["new"], q.shape[1] // heads
    first, count = begin[:-1], begin[1:] - begin[:-1]
    i = torch.arange(n, device=dev)
    row = (first[:, None] + i).clamp(max=len(q) - 1)
    sees = i[:, None] >= i
    if s["parents"] is None:
        sees = sees.expand(r, n, n)
    else:
        sees = torch.zeros((r, n, n), dtype=torch.bool, device=dev)
        at = i.expand(r, n)
        for _ in range(n):  # (a node, its parent, ...)
            sees = sees | ((at[..., None] == i) & (at[..., None] >= 0))
            up = s["parents"].long()[(first[:, None] + at.clamp(min=0)).clamp(max=len(q) - 1)]
            at = torch.where((at < 0) | (up < 0), -1, up - first[:, None])
    most = s["table"].shape[1] * page
    t = torch.arange(most, device=dev)
    ids = s["table"].long().clamp(min=0)[:, t // page]
    new = t - (length - count)[:, None]                                   # a cached token's index among the new ones
    mask = (new[:, None] < 0) | (sees.gather(2, new.clamp(0, n - 1)[:, None].expand(r, n, most)) & (new[:, None] < n))
    mask = mask & (t < length[:, None])[:, None] & (i < count[:, None])[..., None]      # [r, n, most]
    out = torch.zeros(q.shape, dtype=torch.float32, device=dev)
    ks, vs = s["scales"] or (None, None)
    wide = q[row].float().reshape(r, n, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(r * heads, n * group, dim)
    k = _get(s["keys"], ks, ids, (t % page).expand(r, most), s["heads_first"])           # [r, most, heads, dim]
    w = torch.matmul(wide, k.permute(0, 2, 3, 1).reshape(r * heads, dim, most)) * dim ** -0.5
    del k
    w = w.reshape(r, heads, n, group, most).masked_fill_(~mask[:, None, :, None], -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True).clamp(min=-3e38)))
    w = w.div_(w.sum(-1, keepdim=True).clamp(min=1e-38)).reshape(r * heads, n * group, most)
    v = _get(s["values"], vs, ids, (t % page).expand(r, most), s["heads_first"])
    v = v.masked_fill_((t >= length[:, None])[..., None, None], 0)
    o = torch.matmul(w, v.permute(0, 2, 1, 3).reshape(r * heads, most, dim))
    o = o.reshape(r, heads, n, group, dim).permute(0, 2, 1, 3, 4).reshape(r, n, heads * group, dim)
    real = i < count[:, None]
    out[row[real]] = o[real]
    return out.to(q.dtype)


def _beam(s):
    """score + log softmax(logits), its `keep` largest over beams and vocabulary; ties to the lower beam, then token."""
    scores, v = s["scores"].double(), s["logits"].shape[1]
    x = s["logits"].double().reshape(*scores.shape, v)
    x = x - x.amax(-1, keepdim=True)
    total = x.sub_(x.exp().sum(-1, keepdim=True).log_()).add_(scores[..., None]).reshape(len(scores), -1)
    place = torch.arange(total.shape[1], device=total.device)
    at, best = [], []
    for _ in range(s["keep"]):
        best.append(total.amax(1))
        at.append(torch.where(total == best[-1][:, None], place, total.shape[1]).amin(1))
        total.scatter_(1, at[-1][:, None], -math.inf)
    at = torch.stack(at, 1)
    return dict(tokens=(at % v).int(), parents=(at // v).int(), scores=torch.stack(best, 1).float())


def _reorder(s):
    """Beam b of a request takes the cached tokens from `first` on of its beam parents[b]."""
    r, b = s["parents"].shape
    page, caches = s["page"], s["caches"]
    t = s["first"].long()[:, None] + torch.arange(s["most"], device=caches.device)                  # [r, most]
    inside = (t < s["seq_len"].reshape(r, b)[:, :1])[:, None].expand(r, b, s["most"])
    t = t.clamp(max=s["table"].shape[1] * page - 1)[:, None].expand(r, b, s["most"])
    ids = s["table"].long().reshape(r, b, -1).gather(2, t // page)
    src = torch.where(inside, ids.gather(1, s["parents"].long()[..., None].expand(r, b, s["most"])), ids)
    at, dst, src = (t % page)[inside], ids[inside], src[inside]
    if s["heads_first"]:
        caches[:, dst, :, at] = caches[:, src, :, at]
    else:
        caches[:, dst, at] = caches[:, src, at]
    return caches


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _own(s):
    ge = importlib.import_module("goethe-engine_amd")
    kind = s["kind"]
    if kind == "write":
        ge.kv.write(s["slot"], s["k"], s["v"], s["keys"], s["values"], scales=s["scales"], heads_first=s["heads_first"])
        return dict(keys=s["keys"], values=s["values"], scales=s["scales"])
    if kind == "read":
        k, v = ge.kv.read(s["keys"], s["values"], s["table"], s["begin"], first=s["first"], max_tokens=s["rows"],
                          scales=s["scales"], dtype=DTYPE[s["out"]], heads_first=s["heads_first"])
        return dict(k=k, v=v)
    if kind == "attend":
        return ge.kv.attend(s["q"], s["keys"], s["values"], s["table"], s["seq_len"], begin=s["begin"], parents=s["parents"],
                            max_new=s["new"], scales=s["scales"], heads_first=s["heads_first"])
    if kind == "beam":
        o = ge.beam.select(s["logits"], s["scores"], s["keep"])
        return dict(tokens=o.tokens, parents=o.parents, scores=o.scores)
    ge.kv.reorder(s["caches"], s["table"], s["seq_len"], s["parents"], first=s["first"], heads_first=s["heads_first"])
    return s["caches"]


def run(state):
    if own:
        return _own(state)
    return dict(write=_write, read=_read, attend=_attend, beam=_beam, reorder=_reorder)[state["kind"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _host(t):
    if t is None or isinstance(t, tuple):
        return t and tuple(_host(x) for x in t)
    return (t.float() if t.dtype == torch.float8_e4m3fn else t).double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _to_8(x, kind):
    """Rows in 8 bits, by the definition: the values held and the scales (in fp32, as they are stored)."""
    s = np.maximum(np.abs(x).max(-1).astype(np.float32) * np.float32(1 / MOST[kind]), np.float32(TINY))
    x = (x * (np.float32(1) / s).astype(np.float64)[..., None]).astype(np.float32).astype(np.float64)
    step = 1.0 if kind == "i8" else 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), -6) - 3)
    return np.rint(x / step) * step, s


def _exact_write(case, s):
    out, slot = {k: _host(s[k]) for k in ("keys", "values", "scales")}, _host(s["slot"])
    p, o = np.divmod(slot[slot >= 0], case["page"])
    for i, (name, cache) in enumerate((("k", out["keys"]), ("v", out["values"]))):
        x = _host(s[name])[slot >= 0]
        x, scale = _to_8(x, case["cache"]) if case["cache"] in MOST else (x, None)
        for h in range(case["heads"]):
            at = (p, h, o) if case["heads_first"] else (p, o, h)
            cache[at] = x[:, h]
            if scale is not None:
                out["scales"][i][at] = scale[:, h]
    if case["cache"] == "i8":
        out["keys"] = out["values"] = None
    return out


def _row(cache, scale, page_ids, n, first, heads_first, double):
    """Tokens first .. n - 1 of one request's pages, [tokens, heads, dim] in 64 bits."""
    x = double(cache[page_ids])
    x = x.swapaxes(1, 2) if heads_first else x
    if scale is not None:
        f = double(scale[page_ids])
        x = x * (f.swapaxes(1, 2) if heads_first else f)[..., None]
    return x.reshape(-1, *x.shape[2:])[first:n]


def _exact_read(case, s):
    if case["requests"] * case["context"] * case["heads"] * case["dim"] > 1 << 27:
        return None
    begin, first, table = (_host(s[k]).tolist() for k in ("begin", "first", "table"))
    scales, out = s["scales"] or (None, None), []
    for cache, scale in zip((s["keys"], s["values"]), scales):
        rows = [_row(cache, scale, [p for p in table[r] if p >= 0], first[r] + begin[r + 1] - begin[r], first[r],
                     s["heads_first"], _host) for r in range(case["requests"])]
        out.append(np.concatenate(rows))
    return dict(k=out[0], v=out[1])


def _exact_attend(case, s):
    begin, length, table = (_host(s[k]).tolist() for k in ("begin", "seq_len", "table"))
    parents = _host(s["parents"]).tolist() if case["tree"] else None
    scales = s["scales"] or (None, None)
    double = lambda t: t.float().double()  # noqa: E731
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for r in range(case["requests"]):
        b, n, ctx = begin[r], begin[r + 1] - begin[r], length[r] - (begin[r + 1] - begin[r])
        if n == 0:
            continue
        hidden = torch.zeros((n, length[r]), dtype=torch.bool)
        for i in range(n):
            path = list(range(i + 1))
            if parents is not None:
                path, at = [], b + i
                while at >= 0:
                    path.append(at - b)
                    at = parents[at]
            hidden[i, ctx:] = True
            hidden[i, [ctx + j for j in path]] = False
        hidden = hidden.to(out.device).repeat_interleave(case["group"], 0)
        ids = [p for p in table[r] if p >= 0]
        k, v = (_row(c, f, ids, length[r], 0, s["heads_first"], double) for c, f in zip((s["keys"], s["values"]), scales))
        for h in range(case["heads"]):
            at = slice(h * case["group"], (h + 1) * case["group"])
            x = s["q"][b:b + n, at].double().reshape(n * case["group"], -1) @ k[:, h].T.contiguous() / math.sqrt(case["dim"])
            x = torch.softmax(x.masked_fill(hidden, -math.inf), 1)
            out[b:b + n, at] = (x @ v[:, h].contiguous()).reshape(n, case["group"], -1)
    return out


def _exact_beam(case, s):
    x, scores = _host(s["logits"]), _host(s["scores"])
    best = []
    for r in range(case["requests"]):
        every = []
        for b in range(case["beams"]):
            row = x[r * case["beams"] + b]
            every.append(scores[r, b] + row - (row.max() + math.log(np.exp(row - row.max()).sum())))
        every = np.concatenate(every)
        best.append(-np.sort(-np.partition(every, len(every) - case["keep"])[-case["keep"]:]))
    return dict(tokens=None, parents=None, scores=np.array(best))


def _exact_reorder(case, s):
    if case["cache"] == "u8" or case["requests"] * case["beams"] * case["tokens"] > 500 or s["caches"].numel() > 1 << 27:
        return None
    c, table, parents, length, first = (_host(s[k]) for k in ("caches", "table", "parents", "seq_len", "first"))
    was = c.copy()
    for r in range(case["requests"]):
        for b in range(case["beams"]):
            for t in range(first[r], length[r * case["beams"]]):
                to, frm = (table[r * case["beams"] + k, t // case["page"]] for k in (b, parents[r, b]))
                at = (slice(None), t % case["page"]) if case["heads_first"] else (t % case["page"],)
                c[(slice(None), to, *at)] = was[(slice(None), frm, *at)]
    return c


def exact(case, seed):
    """What the definitions give, token by token and request by request."""
    return dict(write=_exact_write, read=_exact_read, attend=_exact_attend, beam=_exact_beam,
                reorder=_exact_reorder)[case["kind"]](case, prepare(case, seed))


def work(case):
    kind, d = case["kind"], case.get("heads", 0) * case.get("dim", 0)
    scale = 4 * case.get("heads", 0) if case.get("cache") in MOST else 0
    if kind == "write":
        n = case["tokens"]
        return {"bytes": n * (8 + 2 * (d * (SIZE[case["source"]] + SIZE[case["cache"]]) + scale)), "flops": n * d * 6}
    if kind == "read":
        n = case["requests"] * case["context"] * 0.75 * 0.875
        return {"bytes": n * 2 * (d * (SIZE[case["cache"]] + SIZE[case["out"]]) + scale), "flops": n * d * 2}
    if kind == "attend":
        r, some = case["requests"], case["tree"] or case["new"] == 1
        n = case["new"] if some else (case["new"] + 1) / 2
        cached = (0.375 + 0.625 * r) * case["context"] + r * n
        rows = r * n * case["group"]
        return {"bytes": cached * 2 * (d * SIZE[case["cache"]] + scale) + 2 * rows * d * SIZE[case["query"]],
                "flops": 4 * cached * n * case["group"] * d}
    if kind == "beam":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": n * SIZE[case["logits"]] + case["requests"] * (4 * case["beams"] + 12 * case["keep"]), "flops": 3 * n}
    moved = case["requests"] * case["beams"] * (1 - 1 / case["beams"]) * case["tokens"] * case["caches"]
    return {"bytes": 2 * moved * d * SIZE[case["cache"]], "flops": 0}
