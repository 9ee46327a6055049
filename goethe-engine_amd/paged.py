"""The paged cache around a verify round, with its numbers on the device: what goethe_engine/kv.py:287-303 and
engine.py:299-305 commit on the host from lengths copied back.

  PageTable   which pages each request holds and which are free; step() keeps what a round accepted, adds the next tokens,
              takes and gives back pages and maps the new tokens to cache slots and positions (gsp_pages_step)
  StepMap     what a step returns: the slot map of its new tokens
  keep_path   the accepted path of each request's draft tree moved to consecutive slots (gsp_keep_path)
  Caches      equal-shaped cache tensors (keys and values of every layer) as one argument of keep_path

A round of tree verification, nothing of which waits for the host:

    step = pages.step(add=prompts)                       # the first tokens; then, round by round:
    ...                                                  # the model writes its keys and values to step.slot
    call.launch()                                        # spec.VerifyCall over the target's logits
    step = call.commit(step, pages, caches, add=nodes, depth=depth, max_tokens=n)

commit is keep_path, the accepted path moved behind its anchor, and the step that keeps it and adds the next round's nodes. A
round of chains needs no move: its accepted drafts are already consecutive (spec.verify_chains(...).commit). Both commits
keep nothing of a request that the round's step did not serve.
"""
import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from .sampling import _device
from .spec import _count, _vec


class StepMap:
    """A step's new tokens: request r's are entries begin[r] .. begin[r + 1] - 1 (int32 [R + 1]) of slot (int64: page *
    tokens per page + offset), pos and req (int32); entries past the last token are -1, 0 and -1. seq_len int32 [R]: each
    request's tokens with the new ones; status int32 [R]: _lib.STEP_OK, STEP_FULL (nothing added: no page left for it, a full
    table row, or past max_tokens) or STEP_BAD (numbers out of range: left as it was), its slots then -1. counters: the
    state after the step."""

    def __init__(self, begin, slot, pos, req, seq_len, status, counters):
        self.begin, self.slot, self.pos, self.req = begin, slot, pos, req
        self.seq_len, self.status, self.counters = seq_len, status, counters


def _state(t, what, dev, dims):
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != dims or t.device != dev:
        raise ValueError(f"{what} must be an int32 tensor of {dims} dimension(s) on {dev}")
    if not t.is_contiguous() and t.stride(-1) != 1:
        raise ValueError(f"{what} must have unit stride")
    return t


class PageTable:
    """The pages of `requests` requests over a cache of `pool` pages of `page` tokens, at most max_pages each; a page belongs to
    one request (pages of a shared prefix are kept outside). Steps of one table follow one another on the device. State there:
    table int32 [requests, max_pages] (a request's pages in order), ring int32 [pool] (the free pages, a queue), counters int32
    [2 + 2 requests]: the queue's head and length, then length and held (pages) of each request."""

    def __init__(self, requests, pool, page, max_pages, device=None):
        requests, pool, page, max_pages = int(requests), int(pool), int(page), int(max_pages)
        if requests < 1 or pool < 1 or page < 1 or max_pages < 1:
            raise ValueError("requests, pool, page and max_pages must be > 0")
        dev = torch.device(device) if device is not None else _device()
        table = torch.full((requests, max_pages), -1, dtype=torch.int32, device=dev)
        counters = torch.zeros(2 + 2 * requests, dtype=torch.int32, device=dev)
        counters[1] = pool
        self._set(table, torch.arange(pool, dtype=torch.int32, device=dev), counters, page)

    @classmethod
    def of(cls, table, ring, counters, page):
        """A PageTable over existing state tensors (used in place)."""
        self = cls.__new__(cls)
        self._set(table, ring, counters, int(page))
        return self

    def _set(self, table, ring, counters, page):
        dev = table.device
        self.table, self.ring = _state(table, "table", dev, 2), _state(ring, "ring", dev, 1)
        self.requests, self.max_pages = table.shape
        if self.requests < 1 or self.max_pages < 1 or ring.numel() < 1 or page < 1:
            raise ValueError("requests, pool, page and max_pages must be > 0")
        if self.requests > 1 and table.stride(0) < self.max_pages:
            raise ValueError("table rows overlap")
        self.table_ld = table.stride(0) if self.requests > 1 else self.max_pages
        self.counters, self.page, self.device = self._counters(counters), page, dev

    def _counters(self, t):
        if _state(t, "counters", self.table.device, 1).numel() != 2 + 2 * self.requests:
            raise ValueError(f"counters must have {2 + 2 * self.requests} entries")
        return t

    @property
    def length(self):
        """int32 [requests] tokens of each request (a view of the state)."""
        return self.counters[2:2 + self.requests]

    @property
    def held(self):
        """int32 [requests] pages of each request."""
        return self.counters[2 + self.requests:]

    @property
    def free(self):
        """int32 [1]: the number of free pages."""
        return self.counters[1:2]

    def step(self, add, keep=None, depth=None, max_tokens=None, into=None, of=None):
        """One step on the current stream, asynchronously (a graph can capture it): request r's length grows by keep[r]
        tokens that an earlier step added (keep[r] < 0: it ends and gives back its pages, also where its new tokens then
        do not fit), then add[r] new tokens get pages and slots. Pages are taken in request order; those given back are free
        from the next step on. depth [max_tokens]:
        each new token's distance from its request's first (a tree node's depth; default: its index). max_tokens: entries of
        the map (default: the sum of add, which then has to be on the host). into: counters of the same size that receive
        the new state; this table's own then stay as they were (pages taken are the same if the step is made again).
        of: the StepMap that added the tokens which keep counts; nothing was written for a request that it did not serve, so
        that one's keep > 0 counts as 0 (without it, the caller sees to that). Returns a StepMap."""
        return self._step(*self._ready(add, keep, depth, max_tokens, into, of))

    def _ready(self, add, keep, depth, max_tokens, into=None, of=None):
        """step's arguments as _step takes them, on the device; what is not in order is refused here."""
        r, dev = self.requests, self.device
        if _count(add) != r or (keep is not None and _count(keep) != r):
            raise ValueError(f"add and keep must have {r} entries")
        if max_tokens is None:
            if isinstance(add, torch.Tensor) and add.device.type != "cpu":
                raise ValueError("add is on the device: max_tokens is required")
            max_tokens = sum(max(int(k), 0) for k in add)
        n = int(max_tokens)
        if not 0 <= n <= 1 << 30:
            raise ValueError(f"max_tokens {n} is not in [0, 2^30]")
        if depth is not None and _count(depth) < n:
            raise ValueError(f"depth must have {n} entries")
        if into is None:
            into = self.counters
        elif into is not self.counters:
            self._counters(into)
            if 0 < abs(into.data_ptr() - self.counters.data_ptr()) < 4 * into.numel():
                raise ValueError("into overlaps the table's counters")
        if of is not None and of.status.shape[0] != r:
            raise ValueError(f"a step of {of.status.shape[0]} requests for a table of {r}")
        if dev.type != "cuda":
            raise RuntimeError("goethe-engine_amd needs a HIP device (the table's state is on the host)")
        if of is not None and of.status.device != dev:
            raise ValueError(f"a step on {of.status.device}, the table on {dev}")
        i32 = torch.int32
        add = _vec(add, i32, dev)
        keep = _vec(keep, i32, dev) if keep is not None else None
        depth = _vec(depth, i32, dev) if depth is not None else None
        return add, keep, depth, n, into, of

    def _step(self, add, keep, depth, n, into, of):
        r, dev, i32 = self.requests, self.device, torch.int32
        slot = torch.empty(n, dtype=torch.int64, device=dev)
        ints = torch.empty(2 * n + 3 * r + 1, dtype=i32, device=dev)
        pos, req, begin, seq, status = ints.split_with_sizes((n, n, r + 1, r, r))
        p = _lib.Pages(_PAGES, r, self.page, self.ring.shape[0], self.max_pages, 0, self.table.data_ptr(), self.table_ld,
                       self.ring.data_ptr(), self.counters.data_ptr(), into.data_ptr())
        t = _lib.Step(_STEP, n, keep.data_ptr() if keep is not None else None, add.data_ptr(),
                      depth.data_ptr() if depth is not None else None, begin.data_ptr(), slot.data_ptr(), pos.data_ptr(),
                      req.data_ptr(), seq.data_ptr(), status.data_ptr(), _lib.raw_stream(dev.index),
                      of.status.data_ptr() if of is not None else None)
        _lib.device_handle(dev.index).call("gsp_pages_step", C.byref(p), C.byref(t))
        return StepMap(begin, slot, pos, req, seq, status, into)


_PAGES, _STEP, _PATH = C.sizeof(_lib.Pages), C.sizeof(_lib.Step), C.sizeof(_lib.Path)


def _layout(shape, stride, size, heads_first, dense=False):
    """(pages, page, chunks, chunk bytes, page / token / chunk strides in bytes) of one cache's [pages, page, ...] or, heads
    first, [pages, heads, page, ...]: a token's data as equal contiguous chunks. dense: the tensor has no gaps."""
    need = 4 if heads_first else 3
    if len(shape) < need or 0 in shape:
        raise ValueError(f"a cache of shape {tuple(shape)}: [pages, {'heads, page' if heads_first else 'page, ...'}] is wanted")
    if dense:  # (sizes from the shape: a dimension of one may have any stride)
        token = math.prod(shape[need - 1:]) * size
        if heads_first:
            return shape[0], shape[2], shape[1], token, shape[1] * shape[2] * token, token, shape[2] * token
        return shape[0], shape[1], 1, token, shape[1] * token, token, 0
    if any(s == 0 and k > 1 for k, s in zip(shape, stride)):
        raise ValueError("a cache must not be an expanded tensor")

    def run(i):  # elements of the dimensions from i on, when they lie together
        n = 1
        for k, s in zip(reversed(shape[i:]), reversed(stride[i:])):
            if k > 1 and s != n:
                return None
            n *= k
        return n

    at = 2 if heads_first else 1
    token = stride[at] * size
    if heads_first:
        chunks, cs, n = shape[1], stride[1], run(3)
    else:
        chunks, cs, n = 1, 0, run(2)
        if n is None and len(shape) > 3:
            chunks, cs, n = shape[2], stride[2], run(3)
    if n is None:
        raise ValueError("a token's data must lie in equal contiguous pieces")
    return shape[0], shape[at], chunks, n * size, stride[0] * size, token, cs * size


class Caches:
    """Cache tensors of one shape and one layout (keys and values of every layer), each [pages, page, ...] or, heads first,
    [pages, heads, page, ...], as one argument of keep_path: their addresses go to the device once. The tensors are kept
    alive and used in place; they must not share memory."""

    def __init__(self, tensors, heads_first=False):
        self.tensors, self.heads_first = list(tensors), bool(heads_first)
        if not self.tensors:
            raise ValueError("no caches")
        t0 = self.tensors[0]
        for t in self.tensors:
            if t.shape != t0.shape or t.stride() != t0.stride() or t.dtype != t0.dtype or t.device != t0.device:
                raise ValueError("caches must have one shape, layout, type and device")
        self.layout = _layout(t0.shape, t0.stride(), t0.element_size(), self.heads_first, t0.is_contiguous())
        ptrs = [t.data_ptr() for t in self.tensors]
        if len(set(ptrs)) < len(ptrs):
            raise ValueError("the same cache twice")
        self.align = min(16, *[k & -k for k in ptrs])
        self.device = t0.device
        self.ptrs = torch.from_numpy(np.array(ptrs, np.int64)).to(self.device)


def keep_path(caches, slot, anchor, emit_len, emit_nodes, heads_first=False):
    """Moves the accepted paths of a round's draft trees in the caches, in place, in one gsp_keep_path call on the current
    stream: entry i = 1 .. emit_len[r] - 1 of request r's path goes from slot[emit_nodes[r, i]] to slot[anchor[r] + i].
    caches: a Caches, or one stacked tensor [n, pages, page, ...] (heads_first: [n, pages, heads, page, ...]); slot: StepMap.slot
    of the round; anchor, emit_len int32 [R], emit_nodes int32 [R, ld]: gse_verify_tree's (VerifyCall.keep_path passes
    them). Nodes ascend along a path and requests share no slots; entries out of range, negative slots and requests
    with a negative anchor (padded ones) are skipped."""
    stacked = not isinstance(caches, Caches)
    if not stacked:
        n, layout, dev = len(caches.tensors), caches.layout, caches.device
    else:
        if not isinstance(caches, torch.Tensor) or caches.dim() < 4:
            raise ValueError("caches must be a Caches or a stacked tensor [n, pages, page, ...]")
        if caches.shape[0] > 1 and caches.stride(0) == 0:
            raise ValueError("a cache must not be an expanded tensor")
        n, dev = caches.shape[0], caches.device
        layout = _layout(caches.shape[1:], caches.stride()[1:], caches.element_size(), heads_first, caches.is_contiguous())
    r = _count(anchor)
    if _count(emit_len) != r or emit_nodes.dim() != 2 or emit_nodes.shape[0] != r:
        raise ValueError(f"anchor, emit_len and emit_nodes must have one entry per request ({r})")
    if not isinstance(slot, torch.Tensor) or slot.dtype != torch.int64 or slot.dim() != 1:
        raise ValueError("slot must be an int64 tensor of one dimension")
    if dev.type != "cuda":
        raise RuntimeError("goethe-engine_amd needs a HIP device (the caches are on the host)")
    if slot.device != dev:
        raise ValueError(f"slot on {slot.device}, the caches on {dev}")
    ld = emit_nodes.shape[1]
    if r == 0 or n == 0 or ld == 0:
        return
    slot = slot.contiguous()
    i32 = torch.int32
    anchor, emit_len, emit_nodes = _vec(anchor, i32, dev), _vec(emit_len, i32, dev), _vec(emit_nodes, i32, dev)
    pages, page, chunks, size, page_stride, token_stride, chunk_stride = layout
    if stacked:
        base, stride, ptrs, align = caches.data_ptr(), caches.stride(0) * caches.element_size(), None, 0
    else:
        base, stride, ptrs, align = None, 0, caches.ptrs.data_ptr(), caches.align
    p = _lib.Path(_PATH, r, slot.shape[0], n, slot.data_ptr(), anchor.data_ptr(), emit_len.data_ptr(), emit_nodes.data_ptr(), ld,
                  base, stride, ptrs, align, page, pages, chunks, size, 0, page_stride, token_stride, chunk_stride,
                  _lib.raw_stream(dev.index))
    _lib.device_handle(dev.index).call("gsp_keep_path", C.byref(p))
