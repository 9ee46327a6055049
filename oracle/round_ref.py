"""Oracle: numpy statements, in 64 bits and request by request, of what happens around a verify round (test infrastructure,
never product code).

  chain / chains  drafted chains against rows of probabilities with given random numbers: draft i accepted iff q_i(x_i) > 0
                  and coin_i q_i(x_i) < p_i(x_i); at the first that is not, the token is drawn from max(p - q, 0) (a draft
                  without a distribution: p without its token; where nothing is left: p), after the last one from the row
                  that follows. With one draft it is spec_ref.mss with one kid (spec.py:88-103).
  Pages           a paged cache's bookkeeping with a queue of free pages and a list of pages per request
  keep_path       a path's entries moved one after the other

chains is pinned in tests/test_round_host.py by its law (the emitted token's is the target's, counted over a grid of coins and
draws) and by spec_ref.mss; Pages by its invariant (every page is in one place) and known answers.
"""
from collections import deque

import numpy as np


def draw(w, u):
    """The first index with a positive weight whose inclusive sum reaches u * sum(w), the last positive one where rounding
    leaves none; -1 when a weight is not finite or none is positive (negative weights count as 0)."""
    if not np.isfinite(w).all():
        return -1
    w = np.maximum(w, 0.0)
    c = np.cumsum(w)
    if not (c[-1] > 0 and np.isfinite(c[-1])):
        return -1
    pos = np.flatnonzero(w > 0)
    hit = pos[~(c[pos] < u * c[-1])]
    return int(hit[0] if len(hit) else pos[-1])


def chain(p, q, tokens, coins, u):
    """p [n + 1, V], q [n, V] or None, of one request (u: one draw, or one per row): (emitted tokens, target weights of them,
    error)."""
    p = np.asarray(p, np.float64)
    v = p.shape[1]
    out, i, w = [], 0, None
    while i < len(tokens) and 0 <= tokens[i] < v:
        x = int(tokens[i])
        qx = 1.0 if q is None else float(q[i][x])
        if not (qx > 0 and coins[i] * qx < p[i][x]):
            with np.errstate(invalid="ignore"):
                w = p[i] - (np.asarray(q[i], np.float64) if q is not None else 0.0)
            if q is None:
                w[x] = 0.0
            if np.isfinite(w).all() and not (w > 0).any():
                w = p[i]
            break
        out.append(x)
        i += 1
    t = draw(p[i] if w is None else w, u[i] if np.ndim(u) else u)
    probs = [float(p[k][x]) for k, x in enumerate(out)]
    if t >= 0:
        out.append(t)
        probs.append(float(p[i][t]))
    return out, probs, t < 0


def chains(target, draft, tokens, begin, coins, u):
    """Per request chain()'s answer; begin as verify_chains takes it, u per request or per target row."""
    res = []
    per_row = len(u) > len(begin) - 1
    for r in range(len(begin) - 1):
        b, e = int(begin[r]), int(begin[r + 1])
        if per_row:
            u_r = np.asarray(u, np.float64)[b + r:e + r + 1]
        res.append(chain(target[b + r:e + r + 1], draft[b:e] if draft is not None else None, [int(x) for x in tokens[b:e]],
                         coins[b:e], u_r if per_row else u[r]))
    return res


class Pages:
    def __init__(self, requests, pool, page, max_pages):
        self.page, self.max_pages, self.pool = page, max_pages, pool
        self.free = deque(range(pool))
        self.length = [0] * requests
        self.pages = [[] for _ in range(requests)]

    def step(self, add, keep=None, depth=None, max_tokens=None, laid=None):
        """dict(begin, slot, pos, req, seq, status) after one step; laid: the status of the step that added what keep counts."""
        n = len(self.length)
        max_tokens = sum(max(int(a), 0) for a in add) if max_tokens is None else max_tokens
        keep = [0] * n if keep is None else keep
        if laid is not None:
            keep = [min(int(k), 0) if s != 0 else k for k, s in zip(keep, laid)]
        begin, seq, status = [0], [], []
        slot, pos, req = [-1] * max_tokens, [0] * max_tokens, [-1] * max_tokens
        short, back = False, []
        for r in range(n):
            a, k = int(add[r]), int(keep[r])
            held = len(self.pages[r])
            kept = 0 if k < 0 else self.length[r] + k
            at, begin_r = begin[-1], begin[-1] + max(a, 0)
            begin.append(begin_r)
            st = 0
            if a < 0 or kept > held * self.page:
                st = 2
                kept = self.length[r]
            else:
                need = -(-(kept + a) // self.page)
                more = max(need - held, 0)
                if need > self.max_pages or (a > 0 and begin_r > max_tokens):
                    st = 1
                    # (what it would have taken still counts ahead of the requests after it)
                    short = short or (need <= self.max_pages and more > 0)
                elif more and (short or more > len(self.free)):
                    st, short = 1, True
            self.length[r] = kept
            if st == 0:
                for _ in range(more):
                    self.pages[r].append(self.free.popleft())
                back += self.pages[r][need:]
                del self.pages[r][need:]
            elif st == 1 and k < 0:  # (it ended: its pages are free, though what was to start in its place did not fit)
                back += self.pages[r]
                self.pages[r] = []
            for i in range(max(a, 0)):
                if at + i >= max_tokens:
                    break
                req[at + i] = r
                pos[at + i] = kept + (i if depth is None else int(depth[at + i]))
                if st == 0:
                    w = kept + i
                    slot[at + i] = self.pages[r][w // self.page] * self.page + w % self.page
            seq.append(kept + (a if st == 0 else 0))
            status.append(st)
        self.free.extend(back)  # (free from the next step on)
        return dict(begin=begin, slot=slot, pos=pos, req=req, seq=seq, status=status)

    def check(self):
        """Every page is in one place."""
        every = sorted(list(self.free) + [p for ps in self.pages for p in ps])
        assert every == list(range(self.pool))


def keep_path(read, write, slot, anchor, emit_len, emit_nodes):
    """read(slot) -> data, write(slot, data): entry i of each path to the slot i after the anchor's."""
    for r in range(len(anchor)):
        for i in range(1, int(emit_len[r])):
            write(int(slot[anchor[r] + i]), read(int(slot[emit_nodes[r][i]])))
