"""The keys and values of a paged cache (paged.PageTable keeps its books): written, read back, attended to, and moved between
beams, on the device and on the current stream (include/gsk.h).

  write    a step's new keys and values to their slots, as they are or in 8 bits with a scale per token and head
  read     cached tokens as contiguous rows
  attend   attention of a step's new tokens (one a request, a chain, a draft tree) over the cache
  reorder  the cached tokens of beams moved to the beams that continue them (beam.select's parents)

A layer of a model's step over the cache, then the round's end:

    step = pages.step(add=nodes, depth=depth, max_tokens=n)
    kv.write(step.slot, k, v, keys, values, scales=scales)
    o = kv.attend(q, keys, values, pages.table, step.seq_len, begin=step.begin, status=step.status, parents=parents,
                  max_new=most, scales=scales)
    ...
    step = call.commit(step, pages, caches, ...)          # spec.VerifyCall; 8-bit scales move as caches of their own

keys and values are one layer's: tensors [pages, page, heads, dim] or, heads first, [pages, heads, page, dim], of one shape and
layout, bfloat16, float16, float8_e4m3fn or int8; dim is a multiple of 8 up to 256. In 8 bits scales is a pair of float32 tensors
[pages, page, heads] ([pages, heads, page]): an element stands for its value times its token's and head's scale. No call computes
gradients. Calls on one stream follow one another; none waits for the host, and a graph can capture them (attend once its
stream's handle is open: after one call on it).
"""
import functools
import math
import struct

import torch

from . import _lib
from .paged import Caches, _layout
from .spec import _count, _vec

_TYPES = {torch.bfloat16: _lib.K_BF16, torch.float16: _lib.K_F16, torch.float8_e4m3fn: _lib.K_E4M3, torch.int8: _lib.K_I8}
_ROWS = {torch.bfloat16: _lib.K_BF16, torch.float16: _lib.K_F16, torch.float32: _lib.K_F32}
# the structs of gsk.h, packed (a third of the time that ctypes takes to fill one)
_CACHE, _WRITE, _READ = struct.Struct("6I2Q3q2Q3q"), struct.Struct("4I2Q4q2Q"), struct.Struct("4I3Qq2I3Q")
_ATTEND, _REORDER = struct.Struct("6IQ2q2QqIf5QqQ"), struct.Struct("4IQq2I4QqQ4I3qQ")


@functools.lru_cache(maxsize=1024)
def _layout_of(shape, stride, dtype, heads_first, scale_shape, scale_stride, writes):
    """gsk_cache's numbers of a cache's shape and strides: (size, type, pages, page, heads, dim), (page, token, head strides), the
    same of the scales, and what the addresses have to be multiples of. Refuses what is not in order."""
    if dtype not in _TYPES:
        raise ValueError(f"a cache of {dtype}: bfloat16, float16, float8_e4m3fn or int8 is wanted")
    if len(shape) != 4 or 0 in shape:
        raise ValueError(f"a cache of shape {tuple(shape)}: [pages, page, heads, dim] (heads first: [pages, heads, page, dim]) is wanted")
    kind, dim = _TYPES[dtype], shape[3]
    pages, (heads, page) = shape[0], shape[1:3] if heads_first else shape[2:0:-1]

    def strides(t):
        ps, (hs, ts) = t[0], t[1:3] if heads_first else t[2:0:-1]
        if writes and ((ps == 0 and pages > 1) or (ts == 0 and page > 1) or (hs == 0 and heads > 1)):
            raise ValueError("the cache written to, and its scales, must not be expanded")
        return ps, ts, hs

    if dim % 8 or dim > _lib.MAX_DIM:
        raise ValueError(f"dim {dim} is no multiple of 8 up to {_lib.MAX_DIM}")
    at = strides(stride)
    if stride[3] != 1 or (at[0] | at[1] | at[2]) % 8:
        raise ValueError("a token's head must lie together, at a multiple of 8 elements")
    if pages * page >= 1 << 32 or heads > 1 << 12:
        raise ValueError(f"{pages} pages of {page} tokens, {heads} heads: at most 2^32 - 1 slots and 2^12 heads")
    if kind < _lib.K_E4M3:
        if scale_shape is not None:
            raise ValueError(f"a cache of {dtype} has no scales")
        return (_CACHE.size, kind, pages, page, heads, dim), at, (0, 0, 0), 16
    if scale_shape is None:
        raise ValueError("an 8-bit cache needs its scales")
    if scale_shape != shape[:3]:
        raise ValueError(f"scales must be of shape {tuple(shape[:3])}")
    return (_CACHE.size, kind, pages, page, heads, dim), at, strides(scale_stride), 8


def _cache(keys, values, scales, heads_first, writes=False):
    """The cache as the library takes it, its (size, type, pages, page, heads, dim), its strides and its device; what is not in
    order is refused here."""
    shape, stride, dtype, dev = keys.shape, keys.stride(), keys.dtype, keys.device
    if values.shape != shape or values.stride() != stride or values.dtype is not dtype or values.device != dev:
        raise ValueError("keys and values must have one shape, layout, type and device")
    k, v, ks, vs = keys.data_ptr(), values.data_ptr(), 0, 0
    if scales is None:
        size, at, s_at, align = _layout_of(shape, stride, dtype, heads_first, None, None, writes)
    else:
        a, b = scales
        s_shape, s_stride = a.shape, a.stride()
        if a.dtype is not torch.float32 or b.dtype is not torch.float32 or b.shape != s_shape or b.stride() != s_stride:
            raise ValueError("scales must be two float32 tensors of one shape and layout")
        if a.device != dev or b.device != dev:
            raise ValueError(f"scales on {a.device} and {b.device}, the cache on {dev}")
        size, at, s_at, align = _layout_of(shape, stride, dtype, heads_first, s_shape, s_stride, writes)
        ks, vs = a.data_ptr(), b.data_ptr()
        if writes and ks == vs:
            raise ValueError("the scales written to must not be the keys' and the values' at once")
    if (k | v) % align:
        raise ValueError("a token's head must lie together, at a multiple of 8 elements")
    if writes and k == v:
        raise ValueError("the cache written to must not be keys and values at once")
    return _CACHE.pack(*size, k, v, *at, ks, vs, *s_at), size, at, dev


def _same_device(dev, name, t):
    if t.device != dev:
        raise ValueError(f"{name} on {t.device}, the cache on {dev}")


def _on_device(dev):
    if dev.type != "cuda":
        raise RuntimeError("goethe-engine_amd needs a HIP device (the cache is on the host)")


@functools.lru_cache(maxsize=1024)
def _rows_in_order(shape, stride, name, heads, dim):
    if len(shape) != 3 or (heads and shape[1] != heads) or shape[2] != dim:
        raise ValueError(f"{name} must be a tensor [tokens, {heads or 'heads'}, {dim}]")
    return stride[2] == 1 and stride[0] % 8 == 0 and stride[1] % 8 == 0


def _rows(t, name, heads, dim):
    """[tokens, heads, dim] rows as the kernels read them (rows that do not start at 16 bytes are copied): the tensor, its
    address, shape and strides."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor [tokens, {heads or 'heads'}, {dim}]")
    shape, stride, at = t.shape, t.stride(), t.data_ptr()
    if not _rows_in_order(shape, stride, name, heads, dim) or at % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        stride, at = t.stride(), t.data_ptr()
    return t, at, shape, stride


@functools.lru_cache(maxsize=1024)
def _work_bytes(device, handle_rows, size, at, call):
    """gsk_attention_work for sizes alone: (size .. dim) and strides of gsk_cache, call: (requests .. max_new, max_pages)."""
    c = _CACHE.pack(*size, 0, 0, *at, *[0] * 5)
    a = _ATTEND.pack(_ATTEND.size, *call[:-1], *[0] * 6, call[-1], 0.0, *[0] * 7)
    return _lib.handle(device, 1, 1).call("gsk_attention_work", c, a)


def _table(table):
    """A table's requests, pages each and row stride."""
    if not isinstance(table, torch.Tensor) or table.dtype is not torch.int32 or table.dim() != 2 or 0 in table.shape:
        raise ValueError("table must be an int32 tensor [requests, pages]")
    (r, width), (ld, one) = table.shape, table.stride()
    if one != 1 and width > 1:
        raise ValueError("table must have unit stride")
    return r, width, ld


def write(slot, k, v, keys, values, scales=None, heads_first=False):
    """Writes the rows k, v [tokens, heads, dim] (bfloat16, float16, float32) to the cache slots slot (int64 [tokens], page * tokens
    per page + offset: paged.StepMap.slot), in place; negative slots and those past the cache are skipped, a slot belongs to one
    token of the call. In 8 bits, in fp32: scale = max(max |row| * (1 / M), 2^-126), M = 448 (float8_e4m3fn) or 127 (int8), the
    elements row * (1 / scale) rounded to nearest even; a row with a NaN or an infinity then reads as NaN."""
    c, (_, _, _, _, heads, dim), _, dev = _cache(keys, values, scales, heads_first, writes=True)
    k, k_at, shape, k_stride = _rows(k, "k", heads, dim)
    v, v_at, v_shape, v_stride = _rows(v, "v", heads, dim)
    kind, n = _ROWS.get(k.dtype), shape[0]
    if kind is None or v.dtype is not k.dtype:
        raise ValueError(f"k of {k.dtype} and v of {v.dtype}: both bfloat16, float16 or float32 are wanted")
    if v_shape != shape or not isinstance(slot, torch.Tensor) or slot.dtype is not torch.int64 or slot.shape != shape[:1]:
        raise ValueError("k, v and slot (int64) must have one entry per token")
    if n * heads > 1 << 26:
        raise ValueError(f"{n} tokens of {heads} heads: at most 2^26 in all")
    _on_device(dev)
    _same_device(dev, "k", k)
    _same_device(dev, "v", v)
    _same_device(dev, "slot", slot)
    if n == 0:
        return
    if not slot.is_contiguous():
        slot = slot.contiguous()
    index = dev.index
    a = _WRITE.pack(_WRITE.size, n, kind, 0, k_at, v_at, k_stride[0], k_stride[1], v_stride[0], v_stride[1], slot.data_ptr(),
                    _lib.raw_stream(index))
    _lib.device_handle(index).call("gsk_write", c, a)


def read(keys, values, table, begin, first=None, max_tokens=None, scales=None, dtype=torch.bfloat16, heads_first=False, out=None):
    """Cached tokens as rows: (k, v), [max_tokens, heads, dim] of dtype. Rows begin[r] .. begin[r + 1] - 1 are request r's tokens
    first[r], first[r] + 1, ... (first: 0). table int32 [requests, pages]: each request's pages (PageTable.table). max_tokens:
    the rows (default: the last of begin, which then has to be on the host). out: the two tensors to write to (contiguous).
    Rows from begin[requests] on are left as they were (without out: not set); a row whose token or page is out of range is 0."""
    c, (_, _, _, page, heads, dim), _, dev = _cache(keys, values, scales, heads_first)
    r, width, ld = _table(table)
    if _count(begin) != r + 1 or (first is not None and _count(first) != r):
        raise ValueError(f"begin must have {r + 1} entries, first {r}")
    if max_tokens is None:
        if isinstance(begin, torch.Tensor) and begin.device.type != "cpu":
            raise ValueError("begin is on the device: max_tokens is required")
        max_tokens = max(int(begin[r]), 0)
    n, kind = int(max_tokens), _ROWS.get(dtype)
    if kind is None:
        raise ValueError(f"rows of {dtype}: bfloat16, float16 or float32 is wanted")
    if n < 0 or n * heads > 1 << 26:
        raise ValueError(f"{n} rows of {heads} heads: 0 to 2^26 in all")
    if width * page >= 1 << 31:
        raise ValueError(f"{width} pages of {page} tokens a request: at most 2^31 - 1 tokens")
    shape = (n, heads, dim)
    if out is not None:
        k, v = out
        for t in out:
            if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"out must be two contiguous {dtype} tensors of shape {shape}, at multiples of 16 bytes")
            _same_device(dev, "out", t)
        if n and k.data_ptr() == v.data_ptr():
            raise ValueError("out must be two tensors")
    _on_device(dev)
    _same_device(dev, "table", table)
    if out is None:
        k, v = torch.empty((2, *shape), dtype=dtype, device=dev).unbind()
    if n == 0:
        return k, v
    begin = _vec(begin, torch.int32, dev)
    first = _vec(first, torch.int32, dev) if first is not None else None
    index = dev.index
    a = _READ.pack(_READ.size, r, n, kind, k.data_ptr(), v.data_ptr(), table.data_ptr(), ld, width, 0, begin.data_ptr(),
                   first.data_ptr() if first is not None else 0, _lib.raw_stream(index))
    _lib.device_handle(index).call("gsk_read", c, a)
    return k, v


def attend(q, keys, values, table, seq_len, begin=None, status=None, parents=None, max_new=None, scale=None, scales=None,
           heads_first=False, out=None):
    """Attention of a step's new tokens: softmax(scale * q k) v, [tokens, query heads, dim] of q's type. Request r's new tokens are
    rows begin[r] .. begin[r + 1] - 1 of q (paged.StepMap.begin; without begin: row r alone), the last of its seq_len[r] cached
    tokens, written to the cache already. Each sees the tokens before its request's new ones, and of those itself and the earlier
    ones; with parents (int32 [tokens], gse_tree.parent: a node's parent row, -1 an anchor) itself and its ancestors alone.

    q [tokens, query heads, dim], bfloat16 or float16 (the cache's type, where that is not 8 bits); query head h reads the cache's
    head h // (query heads / heads). table int32 [requests, pages]. max_new: the most new tokens of a request (default: from begin,
    which then has to be on the host; with parents at most 64), later ones are left out. status: the step's (a request that it did
    not serve gives zeros). scale: default dim ** -0.5. out: a contiguous tensor to write to. What sees nothing is 0; rows from
    begin[requests] on are left as they were (without out: not set); numbers out of range give zeros, cached tokens whose page
    is out of range are not seen."""
    c, size, at, dev = _cache(keys, values, scales, heads_first)
    _, cache_kind, _, page, heads, dim = size
    q, q_at, (n, hq, _), q_stride = _rows(q, "q", None, dim)
    kind = _TYPES.get(q.dtype, _lib.K_F32)
    if kind > _lib.K_F16 or (cache_kind <= _lib.K_F16 and cache_kind != kind):
        raise ValueError(f"q of {q.dtype} over a cache of {keys.dtype}")
    if hq == 0 or hq % heads:
        raise ValueError(f"{hq} query heads over {heads} heads of the cache")
    r, width, ld = _table(table)
    if width * page >= 1 << 31 or r * (16 + width * page // 32) >= 1 << 32:
        raise ValueError(f"{width} pages of {page} tokens for {r} requests: at most 2^31 - 1 tokens each, 2^37 in all")
    if _count(seq_len) != r or (begin is not None and _count(begin) != r + 1) or (status is not None and _count(status) != r):
        raise ValueError(f"seq_len and status must have {r} entries, begin {r + 1}")
    if begin is None:
        if n != r or parents is not None or (max_new is not None and int(max_new) != 1):
            raise ValueError(f"without begin: one new token for each of the {r} requests, got {n}")
        max_new = 1
    elif max_new is None:
        if isinstance(begin, torch.Tensor) and begin.device.type != "cpu":
            raise ValueError("begin is on the device: max_new is required")
        b = [int(x) for x in begin]
        max_new = max([1, *(y - x for x, y in zip(b, b[1:]))])
    max_new = int(max_new)
    if not 0 < max_new <= 1 << 24:
        raise ValueError(f"max_new {max_new} is not in [1, 2^24]")
    rows = min(max_new, n) * (hq // heads)
    tiles = -(-rows // (16 if rows <= 16 else 32 if rows <= 32 or dim > 128 else 48))
    if rows >= (1 << 32) - 48 or r * (16 + width * page // 32) * max(tiles, 1) >= 1 << 32:
        raise ValueError(f"{r} requests of up to {min(max_new, n)} new tokens over up to {width * page}: fewer new ones a call")
    if parents is not None and (_count(parents) < n or max_new > _lib.MAX_TREE):
        raise ValueError(f"parents must have {n} entries, for trees of at most {_lib.MAX_TREE} new tokens")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 2.0 ** 127:
        raise ValueError(f"scale {scale} is not in [-2^127, 2^127]")
    if out is not None:
        if out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be a contiguous tensor like q, at a multiple of 16 bytes")
        _same_device(dev, "out", out)
    _on_device(dev)
    _same_device(dev, "q", q)
    _same_device(dev, "table", table)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if n == 0:
        return out
    i32, index = torch.int32, dev.index
    seq_len = _vec(seq_len, i32, dev)
    begin = _vec(begin, i32, dev) if begin is not None else None
    parents = _vec(parents, i32, dev) if parents is not None else None
    status = _vec(status, i32, dev) if status is not None else None
    h, work = _lib.handle(index, 1, 1), None
    need = _work_bytes(index, h.rows, size, at, (r, n, hq, kind, max_new, width))
    if need:
        work = torch.empty(need, dtype=torch.uint8, device=dev)
    a = _ATTEND.pack(_ATTEND.size, r, n, hq, kind, max_new, q_at, q_stride[0], q_stride[1], out.data_ptr(), table.data_ptr(), ld,
                     width, scale, begin.data_ptr() if begin is not None else 0, seq_len.data_ptr(),
                     status.data_ptr() if status is not None else 0, parents.data_ptr() if parents is not None else 0,
                     work.data_ptr() if need else 0, need, _lib.raw_stream(index))
    h.call("gsk_attend", c, a)
    return out


@functools.lru_cache(maxsize=1024)
def _stacked(shape, stride, size, heads_first, dense):
    """Caches, bytes between them and the layout of each (paged._layout) of a stacked tensor."""
    if len(shape) < 4:
        raise ValueError("caches must be a Caches or a stacked tensor [n, pages, page, ...]")
    if shape[0] > 1 and stride[0] == 0:
        raise ValueError("a cache must not be an expanded tensor")
    return shape[0], stride[0] * size, _layout(shape[1:], stride[1:], size, heads_first, dense)


def reorder(caches, table, seq_len, parents, first=None, heads_first=False):
    """Moves the cached tokens of beams, in place: with parents int32 [groups, beams], beam b of group g is row g * beams + b of
    table and seq_len, and gets the tokens first[g] <= t < seq_len of beam parents[g, b] as they were before the call (first: 0;
    what comes before it, a prompt, is alike in a group's beams). caches: a paged.Caches, or one stacked tensor [n, pages, page,
    ...] (heads_first: [n, pages, heads, page, ...]), of any type. table int32 [groups * beams, pages] (PageTable.table), a page in
    one row. At most 32 beams; a parent out of range leaves its beam as it is, a negative first its group, and tokens past either
    beam's length stay."""
    stacked = not isinstance(caches, Caches)
    if not stacked:
        n, layout, dev = len(caches.tensors), caches.layout, caches.device
    else:
        if not isinstance(caches, torch.Tensor):
            raise ValueError("caches must be a Caches or a stacked tensor [n, pages, page, ...]")
        n, each, layout = _stacked(caches.shape, caches.stride(), caches.element_size(), bool(heads_first), caches.is_contiguous())
        dev = caches.device
    if not isinstance(parents, torch.Tensor) or parents.dim() != 2:
        raise ValueError("parents must be a tensor [groups, beams]")
    groups, beams = parents.shape
    if groups == 0 or n == 0:
        return
    if not 1 <= beams <= _lib.MAX_BEAMS:
        raise ValueError(f"{beams} beams: 1 to {_lib.MAX_BEAMS}")
    rows, width, ld = _table(table)
    if rows != groups * beams or _count(seq_len) != groups * beams or (first is not None and _count(first) != groups):
        raise ValueError(f"table and seq_len must have {groups * beams} rows, first {groups} entries")
    pages, page, chunks, size, page_stride, token_stride, chunk_stride = layout
    if n * chunks * size > 1 << 25:
        raise ValueError(f"{n} caches of {chunks * size} bytes a token: at most 2^25 bytes in all")
    if width * page >= 1 << 31 or pages * page >= 1 << 32:
        raise ValueError(f"{width} of {pages} pages of {page} tokens: at most 2^31 - 1 tokens of 2^32 - 1")
    _on_device(dev)
    _same_device(dev, "table", table)
    i32 = torch.int32
    parents, seq_len = _vec(parents, i32, dev), _vec(seq_len, i32, dev)
    first = _vec(first, i32, dev) if first is not None else None
    if stacked:
        base, stride, ptrs, align = caches.data_ptr(), each, 0, 0
    else:
        base, stride, ptrs, align = 0, 0, caches.ptrs.data_ptr(), caches.align
    a = _REORDER.pack(_REORDER.size, groups, beams, n, table.data_ptr(), ld, width, page, seq_len.data_ptr(), parents.data_ptr(),
                      first.data_ptr() if first is not None else 0, base, stride, ptrs, align, pages, chunks, size, page_stride,
                      token_stride, chunk_stride, _lib.raw_stream(dev.index))
    _lib.device_handle(dev.index).call("gsk_reorder", a)
