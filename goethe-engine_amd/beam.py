"""Beam search's selection on the device (include/gsk.h): the best continuations over a request's beams and the vocabulary. The
paged cache then follows with kv.reorder.

    best = beam.select(logits, scores, 2 * beams)       # logits [requests * beams, V], scores [requests, beams]
    ...                                                 # a caller sets aside those that end; of the others the first `beams`
    kv.reorder(caches, pages.table, step.seq_len, parents, first=prompt)
    step = pages.step(add=ones, keep=ones)
"""
import functools
import struct

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.K_BF16, torch.float16: _lib.K_F16, torch.float32: _lib.K_F32}
_BEAMS = struct.Struct("6IQq5QqQ")  # gsk_beams


class Choice:
    """The continuations of each request, best first: tokens and parents (the beam continued) int32 [requests, n], scores
    float32 [requests, n]; -1, -1 and -inf where there are fewer than n."""

    def __init__(self, tokens, parents, scores):
        self.tokens, self.parents, self.scores = tokens, parents, scores


def select(logits, scores, n):
    """The n best continuations of each request's beams, on the current stream, asynchronously: the largest scores[r, b] +
    log_softmax(logits[r * beams + b])[token], ties to the lower beam, then to the lower token. logits: a device tensor
    [requests * beams, V], float32, bfloat16 or float16, used in place at any row stride; scores [requests, beams], taken as
    float32 (-inf: a beam that is not continued, as in a first step's all but one). At most 32 beams and n <= 64. A NaN logit
    counts as -inf, and tokens of -inf are not taken; a beam whose score is not finite, or whose logits hold +inf or nothing above
    -inf, gives none. Returns a Choice."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _TYPES:
        raise ValueError("logits must be a float32, bfloat16 or float16 tensor [requests * beams, V]")
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2 or not scores.is_floating_point():
        raise ValueError("scores must be a floating-point tensor [requests, beams]")
    (requests, beams), vocab, n = scores.shape, logits.shape[1], int(n)
    if logits.shape[0] != requests * beams:
        raise ValueError(f"{logits.shape[0]} rows of logits for {requests} requests of {beams} beams")
    if not 1 <= beams <= _lib.MAX_BEAMS or not 1 <= n <= _lib.MAX_KEEP:
        raise ValueError(f"{beams} beams, {n} kept: 1 to {_lib.MAX_BEAMS} and 1 to {_lib.MAX_KEEP}")
    if not 1 <= vocab <= 1 << 30 or requests > 1 << 24:
        raise ValueError(f"V = {vocab}, {requests} requests: 1 to 2^30 and at most 2^24")
    dev = logits.device
    if dev.type != "cuda":
        raise RuntimeError("goethe-engine_amd needs a HIP device (the logits are on the host)")
    if scores.device != dev:
        raise ValueError(f"scores on {scores.device}, the logits on {dev}")
    if (logits.stride(1) != 1 and vocab > 1) or (logits.shape[0] > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    if scores.dtype is not torch.float32 or not scores.is_contiguous():
        scores = scores.to(torch.float32).contiguous()
    tokens, parents = torch.empty((2, requests, n), dtype=torch.int32, device=dev).unbind()
    best = torch.empty((requests, n), dtype=torch.float32, device=dev)
    if requests:
        h = _lib.handle(dev.index, 1, 1)
        kind, ld = _TYPES[logits.dtype], logits.stride(0) if logits.shape[0] > 1 else vocab
        need = _work_bytes(dev.index, requests, beams, n, vocab, kind)
        work = torch.empty(need, dtype=torch.uint8, device=dev)
        h.call("gsk_beam", _BEAMS.pack(_BEAMS.size, requests, beams, n, vocab, kind, logits.data_ptr(), ld, scores.data_ptr(),
                                       tokens.data_ptr(), parents.data_ptr(), best.data_ptr(), work.data_ptr(), need,
                                       _lib.raw_stream(dev.index)))
    return Choice(tokens, parents, best)


@functools.lru_cache(maxsize=1024)
def _work_bytes(device, *sizes):
    return _lib.handle(device, 1, 1).call("gsk_beams_work", _BEAMS.pack(_BEAMS.size, *sizes, *[0] * 9))
