"""Timing cases of the operators around a verify round whose numbers stay on the device.

A case is a dict of plain values; "kind" says which operator one pass calls:

  chain   spec.verify_chains: every request's drafted chain against the target's probability rows, with the acceptance
          coins and the draw's uniform given
  pages   paged.PageTable.step: tokens kept and added per request -> pages taken and released, the block table, the new
          tokens' cache slots and positions
  path    paged.keep_path: the accepted path of each request's draft tree moved to consecutive cache slots

The plain forms below compute the same from elementary tensor operations. Inputs are drawn on the GPU from the seed.
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPE = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8}
NOISE = 0.5    # the drafter's logits are the target's plus NOISE times a normal:
ACCEPT = 0.8   # a draft is then accepted about this often


def listed():
    return [
        # one user's chat with a small drafter: the latency of one short chain
        dict(name="chain_chat_1", kind="chain", requests=1, drafts=4, ragged=False, vocab=128256, target="f32",
             draft="f32", cut=1.0),
        # prompt-lookup drafts (no draft distribution), ragged chains, some requests without a draft, an odd vocabulary
        dict(name="chain_lookup_24", kind="chain", requests=24, drafts=6, ragged=True, vocab=50257, target="bf16",
             draft="none", cut=1.0),
        # the target's rows as gse_dist gives them: fp64, a nucleus, zero elsewhere
        dict(name="chain_nucleus_16", kind="chain", requests=16, drafts=4, ragged=True, vocab=151936, target="f64",
             draft="f32", cut=0.95),
        # a serving batch with softmax rows of both models
        dict(name="chain_64", kind="chain", requests=64, drafts=7, ragged=False, vocab=128256, target="f32", draft="f32",
             cut=1.0),
        # the largest batch and vocabulary, half-precision rows
        dict(name="chain_512", kind="chain", requests=512, drafts=3, ragged=False, vocab=262144, target="bf16",
             draft="bf16", cut=1.0),
        # one user's decode step
        dict(name="pages_decode_1", kind="pages", requests=1, page=16, context=8192, before=1, add=1, prompts=0.0,
             room=1, tree=False),
        # the step between two tree rounds of a batch: 1 to 9 tokens kept, nine nodes added at their depths
        dict(name="pages_tree_96", kind="pages", requests=96, page=32, context=8192, before=9, add=9, prompts=0.0,
             room=864, tree=True),
        # continuous batching: chains, requests that end, prompts that start in their place; pages of an odd size
        dict(name="pages_mixed_512", kind="pages", requests=512, page=24, context=4096, before=5, add=5, prompts=0.1,
             room=32768, tree=False),
        # a batch of prompts and long chunks
        dict(name="pages_prompt_1024", kind="pages", requests=1024, page=64, context=16384, before=1, add=512, prompts=0.5,
             room=1048576, tree=False),
        # one request, two chains of four from the anchor, every layer's keys and values
        dict(name="path_1", kind="path", requests=1, chains=2, depth=4, caches=32, heads=8, dim=128, page=16,
             dtype="bf16", heads_first=False),
        # a serving batch
        dict(name="path_64", kind="path", requests=64, chains=2, depth=4, caches=64, heads=8, dim=128, page=16,
             dtype="bf16", heads_first=False),
        # deeper trees over an 8-bit cache with the heads ahead of the page's tokens, odd head counts and sizes
        dict(name="path_heads_100", kind="path", requests=100, chains=4, depth=6, caches=48, heads=5, dim=80, page=32,
             dtype="u8", heads_first=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chain", "chain", "pages", "path"])
    if kind == "chain":
        target = rng.choice(["f32", "f32", "bf16", "f16", "f64"])
        draft = rng.choice(["none", "f32", target])
        requests = _log_int(rng, 1, 512)
        drafts = rng.randint(1, 8 if requests <= 128 else 3)
        top = min(262144, 512 * 262144 * 2 // (requests * (8 if target == "f64" else 4)))
        vocab = rng.choice([v for v in (32000, 50257, 128256, 151936) if v <= top]) if rng.random() < 0.3 and top >= 32000 \
            else _log_int(rng, 4000, top)
        return dict(kind=kind, requests=requests, drafts=drafts, ragged=rng.random() < 0.5, vocab=vocab, target=target,
                    draft=draft, cut=rng.choice([1.0, 1.0, 0.95]))
    if kind == "pages":
        requests = _log_int(rng, 1, 1024)
        add = rng.choice([1, rng.randint(2, 9), _log_int(rng, 10, 512)])
        tree = 2 <= add <= 9 and rng.random() < 0.5
        prompts = 0.0 if tree else rng.choice([0.0, 0.1, 0.3])
        room = requests * add if prompts == 0.0 else min(1048576, requests * (add + 300))
        return dict(kind=kind, requests=requests, page=rng.choice([1, 8, 16, 24, 32, 64, 128]),
                    context=_log_int(rng, 256, 16384), before=rng.randint(1, 9), add=add, prompts=prompts, room=room, tree=tree)
    caches = 2 * rng.randint(4, 32)
    return dict(kind=kind, requests=_log_int(rng, 1, 100), chains=rng.randint(2, 4), depth=rng.randint(1, 6), caches=caches,
                heads=rng.randint(1, 8), dim=rng.choice([64, 72, 80, 96, 128]), page=rng.choice([8, 16, 24, 32]),
                dtype=rng.choice(["bf16", "bf16", "f16", "u8"]), heads_first=rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _logits(g, rows, vocab, dev):
    """Rows like a trained model's: a Zipf slope over a ranking of the tokens that is the row's own, plus a normal."""
    slope = torch.empty(vocab, device=dev)
    slope[torch.randperm(vocab, generator=g, device=dev)] = -1.1 * torch.log1p(torch.arange(vocab, device=dev).float())
    turn = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    x = torch.cat([slope, slope[:-1]]).unfold(0, vocab, 1)[turn]
    return x.add_(torch.randn((rows, vocab), generator=g, device=dev).mul_(2.5))


def _sampled(g, x):
    """A token of each row of logits, drawn from their softmax."""
    n = torch.rand(x.shape, generator=g, device=x.device).clamp_(1e-9, 1 - 6e-8).log_().neg_().log_()
    return (x - n).argmax(1)


def _nucleus(p, cut):
    """p's smallest set of most likely tokens that holds `cut` of the mass, scaled to one; zero elsewhere."""
    s = p.sort(dim=1, descending=True).values
    k = (s.cumsum(1) < cut).sum(1, keepdim=True).clamp_(max=p.shape[1] - 1)
    p = torch.where(p >= s.gather(1, k), p, torch.zeros_like(p))
    return p / p.sum(1, keepdim=True)


def _prepare_chain(case, g, dev):
    r, k, v = case["requests"], case["drafts"], case["vocab"]
    n = torch.randint(0, k + 1, (r,), generator=g, device=dev) if case["ragged"] else torch.full((r,), k, device=dev)
    n[0] = k
    begin = torch.zeros(r + 1, dtype=torch.int32, device=dev)
    begin[1:] = n.cumsum(0)
    drafts = int(begin[-1])
    z = _logits(g, drafts + r, v, dev)
    owner = torch.repeat_interleave(torch.arange(r, device=dev), n)
    row = torch.arange(drafts, device=dev) + owner            # the target row of each draft
    draft = None
    if case["draft"] == "none":  # copied from the prompt: confident rows, the copied token mostly their best
        z.mul_(2.5)
        token = _sampled(g, 1.5 * z[row])
    else:
        zq = z[row].add_(torch.randn((drafts, v), generator=g, device=dev), alpha=NOISE)
        token = _sampled(g, zq)
        draft = torch.softmax(zq, 1).to(DTYPE[case["draft"]])
        del zq
    target = torch.softmax(z.double() if case["target"] == "f64" else z, 1)
    del z
    if case["cut"] < 1.0:
        target = _nucleus(target, case["cut"])
    return dict(kind="chain", target=target.to(DTYPE[case["target"]]), draft=draft, token=token.int(), begin=begin, most=k,
                coin=torch.rand(drafts, generator=g, device=dev, dtype=torch.float64),
                u=torch.rand(r, generator=g, device=dev, dtype=torch.float64))


def _prepare_pages(case, g, dev):
    r, page = case["requests"], case["page"]
    between = lambda lo, hi: torch.randint(lo, hi + 1, (r,), generator=g, device=dev)  # noqa: E731
    length = between(case["context"] // 4, case["context"])
    held = (length + case["before"] + page - 1) // page
    keep = between(1, case["before"])
    add = torch.full((r,), case["add"], device=dev) if case["tree"] or case["add"] == 1 else between(1, case["add"])
    chance = torch.rand(r, generator=g, device=dev)
    ends = chance < case["prompts"]
    keep = torch.where(ends, -1, keep)
    add = torch.where(ends, torch.where(chance < 0.7 * case["prompts"], between(16, 1024), 0), add)
    add = torch.where(add.cumsum(0) <= case["room"], add, 0)
    width = (case["context"] + case["before"] + max(1024, case["add"]) + page) // page + 1
    used = int(held.sum())
    pool = r * ((case["context"] + case["before"]) // page + 3) + case["room"] // page + 7
    ids = torch.randperm(pool, generator=g, device=dev).int()
    table = torch.full((r, width), -1, dtype=torch.int32, device=dev)
    have = torch.arange(width, device=dev) < held[:, None]
    table[have] = ids[:used]
    head = int(torch.randint(0, pool, (1,), generator=g, device=dev))
    ring = torch.full((pool,), -1, dtype=torch.int32, device=dev)
    ring[(head + torch.arange(pool - used, device=dev)) % pool] = ids[used:]
    counters = torch.cat([torch.tensor([head, pool - used], device=dev), length, held]).int()
    depth = None
    if case["tree"]:  # chains of four from the anchor
        node = torch.arange(case["add"], device=dev)
        depth = torch.where(node > 0, (node - 1) % 4 + 1, 0).repeat(r).int()
    return dict(kind="pages", table=table, ring=ring, counters=counters, after=torch.zeros_like(counters), page=page,
                keep=keep.int(), add=add.int(), depth=depth, room=case["room"])


def _prepare_path(case, g, dev):
    r, page, n = case["requests"], case["page"], 1 + case["chains"] * case["depth"]
    context = torch.randint(1, 256, (r,), generator=g, device=dev)
    width = (256 + n) // page + 1
    pages = r * width
    table = torch.randperm(pages, generator=g, device=dev).reshape(r, width)
    at = context[:, None] + torch.arange(n, device=dev)
    slot = (table.gather(1, at // page) * page + at % page).reshape(-1)
    # the accepted chain and how much of it: the anchor, then the chain's first nodes
    chain = torch.randint(0, case["chains"], (r,), generator=g, device=dev)
    emit_len = torch.randint(1, case["depth"] + 2, (r,), generator=g, device=dev)
    chain[0], emit_len[0] = case["chains"] - 1, case["depth"] + 1
    step = torch.arange(case["depth"] + 1, device=dev)
    anchor = n * torch.arange(r, device=dev)
    nodes = torch.where(step > 0, 1 + chain[:, None] * case["depth"] + step - 1, 0)
    nodes = torch.where(step < emit_len[:, None], anchor[:, None] + nodes, -1)
    shape = (case["heads"], page) if case["heads_first"] else (page, case["heads"])
    bits = torch.randint(-128, 128, (case["caches"], pages, *shape, case["dim"]), generator=g, device=dev, dtype=torch.int8)
    cache = bits.view(torch.uint8) if case["dtype"] == "u8" else bits.to(DTYPE[case["dtype"]])
    return dict(kind="path", cache=cache, heads_first=case["heads_first"], page=page, slot=slot, anchor=anchor.int(),
                emit_len=emit_len.int(), emit_nodes=nodes.int())


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed & 0x7FFFFFFF)
    return dict(chain=_prepare_chain, pages=_prepare_pages, path=_prepare_path)[case["kind"]](case, g, dev)


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _chain(s):
    """Accept x_i while coin_i q_i(x_i) < p_i(x_i); at the first draft that is not, draw from max(p - q, 0) (a draft without
    a distribution: p without its token; where that leaves nothing: p), after the last one from the next row of p."""
    target, draft, begin, most = s["target"], s["draft"], s["begin"].long(), s["most"]
    r, v = len(begin) - 1, target.shape[1]
    dev = target.device
    first, count, i = begin[:-1], begin[1:] - begin[:-1], torch.arange(most, device=dev)
    top = max(len(s["token"]) - 1, 0)
    at = (first[:, None] + i).clamp(max=top)
    req = torch.arange(r, device=dev)
    row = (first + req)[:, None] + torch.minimum(i, count[:, None])
    x = s["token"].long()[at]
    real = (i < count[:, None]) & (x >= 0) & (x < v)
    x = x.clamp(0, v - 1)
    px = target[row, x].double()
    qx = draft[at, x].double() if draft is not None else torch.ones_like(px)
    took = (real & (qx > 0) & (s["coin"][at] * qx < px)).long().cumprod(1)
    a = took.sum(1)
    failed = (a < most) & real.gather(1, a.clamp(max=most - 1)[:, None])[:, 0]
    at_a = at.gather(1, a.clamp(max=most - 1)[:, None])[:, 0]
    x_a = x.gather(1, a.clamp(max=most - 1)[:, None])[:, 0]
    p = target[first + req + a].double()
    if draft is not None:
        w = p - torch.where(failed[:, None], draft[at_a].double(), torch.zeros((), dtype=torch.float64, device=dev))
    else:
        w = p.clone()
        w[req, x_a] = torch.where(failed, 0.0, w[req, x_a])
    w = w.clamp_(min=0)
    c = w.cumsum(1)
    empty = failed & (c[:, -1] == 0)
    p = p.clamp_(min=0)
    w, c = torch.where(empty[:, None], p, w), torch.where(empty[:, None], p.cumsum(1), c)
    total = c[:, -1]
    fine = torch.isfinite(total) & (total > 0)
    last = v - 1 - (w > 0).flip(1).to(torch.uint8).argmax(1)
    j = torch.minimum(torch.searchsorted(c, (s["u"] * total)[:, None])[:, 0], last)
    step = torch.arange(most + 1, device=dev)
    emit = torch.where(step < a[:, None], torch.nn.functional.pad(x, (0, 1)), j[:, None])
    emit_len = a + fine.long()
    inside = step < emit_len[:, None]
    at_row = (first + req)[:, None] + torch.minimum(step, count[:, None])
    return dict(len=emit_len.int(), tokens=torch.where(inside, emit, -1).int(),
                probs=torch.where(inside, target[at_row, emit], 0).float(), status=(~fine).int())


def _pages(s):
    """Per request: length' = length + keep (keep < 0: 0), need = ceil((length' + add) / page) pages; what it lacks comes
    from the head of the ring of free pages, what it has too many of goes to its tail, in the order of the requests."""
    table, ring, page = s["table"], s["ring"], s["page"]
    r, width, pool = table.shape[0], table.shape[1], len(ring)
    dev = table.device
    head, free = s["counters"][0].long(), s["counters"][1].long()
    length, held = s["counters"][2:2 + r].long(), s["counters"][2 + r:].long()
    keep, add = s["keep"].long(), s["add"].long()
    kept = torch.where(keep < 0, 0, length + keep)
    total = kept + add
    need = (total + page - 1) // page
    more = (need - held).clamp(min=0)
    begin = torch.nn.functional.pad(add.cumsum(0), (1, 0))
    took_before = more.cumsum(0) - more
    served = (need <= width) & ((more == 0) | (took_before + more <= free)) & (begin[1:] <= s["room"])
    less = torch.where(served, (held - need).clamp(min=0), 0)
    less_to = less.cumsum(0)
    col = torch.arange(width, device=dev)
    fresh = served[:, None] & (col >= held[:, None]) & (col < need[:, None])
    table.copy_(torch.where(fresh, ring[(head + took_before[:, None] + col - held[:, None]) % pool], table))
    k = (torch.arange(pool, device=dev) - head - free) % pool
    who = torch.searchsorted(less_to, k, right=True).clamp(max=r - 1)
    back = table[who, (need[who] + k - less_to[who] + less[who]).clamp(0, width - 1)]
    ring.copy_(torch.where(k < less_to[-1], back, ring))
    t = torch.arange(s["room"], device=dev)
    req = torch.searchsorted(begin[1:], t, right=True).clamp(max=r - 1)
    real = t < begin[-1]
    at = kept[req] + t - begin[req]
    slot = table[req, (at // page).clamp(max=width - 1)].long() * page + at % page
    pos = at if s["depth"] is None else kept[req] + s["depth"].long()[:s["room"]]
    took = torch.where(served, more, 0).sum()
    now = torch.where(served, need, held)
    s["after"].copy_(torch.cat([((head + took) % pool)[None], (free - took + less_to[-1])[None], kept, now]))
    return dict(table=table, ring=ring, counters=s["after"], begin=begin.int(),
                slot=torch.where(real & served[req], slot, -1), pos=torch.where(real, pos, 0).int(),
                req=torch.where(real, req, -1).int(), seq=torch.where(served, total, kept).int(), status=(~served).int())


def _path(s):
    """The cache rows of an accepted path's nodes moved to the slots that follow the anchor's."""
    cache, page, slot = s["cache"], s["page"], s["slot"]
    step = torch.arange(1, s["emit_nodes"].shape[1], device=cache.device)
    anchor = s["anchor"].long()[:, None]
    inside = step < s["emit_len"][:, None]
    src = slot[torch.where(inside, s["emit_nodes"][:, 1:].long(), anchor)].reshape(-1)  # (the others: the anchor onto itself)
    dst = slot[torch.where(inside, anchor + step, anchor)].reshape(-1)
    if s["heads_first"]:
        cache[:, dst // page, :, dst % page] = cache[:, src // page, :, src % page]
    else:
        cache[:, dst // page, dst % page] = cache[:, src // page, src % page]
    return cache


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _own(s):
    ge = importlib.import_module("goethe-engine_amd")
    if s["kind"] == "chain":
        o = ge.spec.verify_chains(s["target"], s["token"], s["begin"], s["coin"], s["u"], draft=s["draft"],
                                  max_drafts=s["most"])
        return dict(len=o.emit_len, tokens=o.tokens, probs=o.probs, status=o.status)
    if s["kind"] == "pages":
        pages = ge.paged.PageTable.of(s["table"], s["ring"], s["counters"], s["page"])
        m = pages.step(s["add"], keep=s["keep"], depth=s["depth"], max_tokens=s["room"], into=s["after"])
        return dict(table=pages.table, ring=pages.ring, counters=m.counters, begin=m.begin, slot=m.slot, pos=m.pos, req=m.req,
                    seq=m.seq_len, status=m.status)
    ge.paged.keep_path(s["cache"], s["slot"], s["anchor"], s["emit_len"], s["emit_nodes"], heads_first=s["heads_first"])
    return s["cache"]


def run(state):
    if own:
        return _own(state)
    return dict(chain=_chain, pages=_pages, path=_path)[state["kind"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    """The probabilities of a chain's emitted tokens, and the moved cache, request by request on the host."""
    if case["kind"] == "pages":
        return None  # (whole numbers only)
    s = prepare(case, seed)
    h = {k: t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy() for k, t in s.items()
         if isinstance(t, torch.Tensor) and t.numel() <= 1 << 27}
    if case["kind"] == "path":
        if case["requests"] > 8 or case["dtype"] == "u8" or "cache" not in h:
            return None
        c = h["cache"]
        for r in range(case["requests"]):
            for i in range(1, h["emit_len"][r]):
                src, dst = (divmod(int(h["slot"][k]), case["page"]) for k in (h["emit_nodes"][r, i], h["anchor"][r] + i))
                if case["heads_first"]:
                    c[:, dst[0], :, dst[1]] = c[:, src[0], :, src[1]]
                else:
                    c[:, dst[0], dst[1]] = c[:, src[0], src[1]]
        return c
    if "target" not in h or (s["draft"] is not None and "draft" not in h):
        return None
    out = np.zeros((case["requests"], case["drafts"] + 1))
    for r in range(case["requests"]):
        b, e = int(h["begin"][r]), int(h["begin"][r + 1])
        q, p, x = None, h["target"][b + r], None
        for i in range(b, e):
            p, x = h["target"][i + r], int(h["token"][i])
            q = h["draft"][i] if s["draft"] is not None else (np.arange(case["vocab"]) == x).astype(np.float64)
            if not h["coin"][i] * q[x] < p[x]:
                break
            out[r, i - b] = p[x]
            q, p = None, h["target"][i + 1 + r]
        else:
            i = e
        w = p if q is None else np.where(np.arange(case["vocab"]) == x, 0.0, p) if s["draft"] is None else np.maximum(p - q, 0.0)
        w = w if w.sum() > 0 else p
        c = np.cumsum(w)
        out[r, i - b] = p[min(int((c < h["u"][r] * c[-1]).sum()), int(np.flatnonzero(w)[-1]))]
    return dict(len=None, tokens=None, probs=out, status=None)


def work(case):
    r = case["requests"]
    size = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2, "u8": 1}
    if case["kind"] == "chain":
        v, n = case["vocab"], case["drafts"] / 2 if case["ragged"] else case["drafts"]
        failed = 1 - ACCEPT ** n
        q = 0 if case["draft"] == "none" else failed * size[case["draft"]]
        small = n * (4 + 8 + 2 * size[case["target"]]) + 12 + (case["drafts"] + 1) * 8 + 8
        return {"bytes": r * (v * (size[case["target"]] + q) + small), "flops": r * v * 3}
    if case["kind"] == "pages":
        return {"bytes": case["room"] * (16 + (4 if case["tree"] else 0)) + r * 40 + case["room"] / case["page"] * 8,
                "flops": case["room"] * 4}
    row = case["heads"] * case["dim"] * size[case["dtype"]] * case["caches"]
    moved = (r - 1) * (case["chains"] - 1) / case["chains"] * case["depth"] / 2 + case["depth"]
    return {"bytes": moved * row * 2 + r * 16, "flops": 0}
