"""Beam search over the int4 KV cache: choosing the next beams from the logits, and
the step of a cache's sequences to them.

The reference samples one continuation of a sequence
(``engine/gemma4_multilayer.cpp:519-527``).  Here a group of ``beams`` sequences of
one cache holds a request's best ones: :func:`beam_select` chooses among their
continuations and ``reorder`` of :class:`gemma4metal_amd.paged.PagedInt4KVCache` and
:class:`gemma4metal_amd.turboquant.Int4KVCache` moves the cached rows;
:func:`beam_step` is both.

As in ``turboquant.py``, torch holds device memory and streams; every computation
runs in ``libturboquant_hip.so``.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from ._lib import call
from .paged import _fits_int, _placed, _workspace
from .turboquant import _DT, _need, _ptr, _stream


@functools.lru_cache(maxsize=64)
def _select_ws_size(B: int, W: int, V: int) -> int:
    return _lib.load().tq_beam_select_workspace_size(B, W, V)


@_placed
def beam_select(logits: torch.Tensor, scores: torch.Tensor, num_out: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None, pad_token: int = 0,
                workspace: Optional[torch.Tensor] = None):
    """The next beams of every group.  logits (B, W, V) f32|f16|bf16, of any strides
    but the last's, which is 1; scores (B, W) f32, the beams' sums of log-probabilities
    so far.  Of a group's totals ``scores[w] + log_softmax(logits[w])[t]`` the
    ``num_out`` (W by default) largest, the lowest (w, t) first among equals; totals of
    two beams that differ by less than 7.2e-7 may change places (6e-8 as a rule).
    A beam with finished[b, w] (bool or uint8) has one candidate: itself, with
    ``pad_token``.  A score of -inf or NaN gives its beam none (the first step of a
    request: all beams but one), nor does a logit of -inf or NaN.

    Returns (scores, parents, tokens), each (B, num_out), best first: f32 totals, the
    int32 number b * W + w of the beam that is continued (what ``reorder`` takes, where
    num_out is W) and the int32 token; -inf, -1 and -1 where there are fewer candidates.
    1 <= W, num_out <= 64, V <= 2^24."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be on a GPU device")
    _need(logits.dim() == 3 and logits.dtype in _DT, "logits must be (B, W, V) float32, float16 or bfloat16")
    B, W, V = logits.shape
    _need(V == 1 or logits.stride(2) == 1, "logits must be contiguous along the vocabulary")
    dev = logits.device
    if not (isinstance(scores, torch.Tensor) and scores.dtype is torch.float32 and scores.shape == (B, W)
            and scores.device == dev and scores.is_contiguous()):
        raise ValueError(f"scores must be contiguous float32 ({B}, {W}) on {dev}")
    if finished is not None and not (isinstance(finished, torch.Tensor) and finished.dtype in (torch.bool, torch.uint8)
                                     and finished.shape == (B, W) and finished.device == dev
                                     and finished.is_contiguous()):
        raise ValueError(f"finished must be contiguous bool or uint8 ({B}, {W}) on {dev}")
    K, pad = W if num_out is None else int(num_out), int(pad_token)
    _need(K >= 1, "num_out must be at least 1")
    _fits_int(num_out=K, pad_token=pad)
    out = (torch.empty((B, K), dtype=torch.float32, device=dev), torch.empty((B, K), dtype=torch.int32, device=dev),
           torch.empty((B, K), dtype=torch.int32, device=dev))
    nbytes = _select_ws_size(B, W, V)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if workspace is None else _workspace(workspace, nbytes, dev, 0)
    call("tq_beam_select", logits.data_ptr(), _DT[logits.dtype], logits.stride(0), logits.stride(1), scores.data_ptr(),
         _ptr(finished), B, W, V, K, pad, *[t.data_ptr() for t in out], ws.data_ptr(), ws.numel(),
         _stream(None))
    return out


def _check_caches(caches, sequences: int, device) -> dict:
    """What a step needs of its caches, before any of them moves.  Returns the number
    of the last cache with each lengths tensor."""
    last, held = {}, {}
    for i, cache in enumerate(caches):
        n = cache.lengths
        _need(n.shape == (sequences,) and n.device == device and n.dtype is torch.int32 and n.is_contiguous(),
              "every cache must hold a sequence for each beam, on the logits' device, in contiguous int32 lengths")
        paged = hasattr(cache, "block_tables")
        for t in (cache.tensors()[0], cache.block_tables) if paged else cache.tensors()[:1]:
            _need(t.data_ptr() not in held, "a cache (its rows, or its block_tables) is given twice")
            held[t.data_ptr()] = True
        at = n.data_ptr()
        for other, j in last.items():
            _need(abs(other - at) >= 4 * sequences
                  or other == at and not paged and not hasattr(caches[j], "block_tables"),
                  "lengths may be shared by Int4KVCaches only, and whole")
        last[at] = i
    return last


def beam_step(caches, logits: torch.Tensor, scores: torch.Tensor, *, finished: Optional[torch.Tensor] = None,
              pad_token: int = 0):
    """:func:`beam_select` of as many beams, and ``reorder`` of the cache (or each of a
    list of caches), whose sequences are the B * W beams: sequence b * W + w then holds
    the rows of its new beam, whose token comes next.  Int4KVCaches may share one
    ``lengths`` tensor.  Returns beam_select's results; a beam for which a paged cache had
    no page has ended and has a score of -inf."""
    caches = caches if isinstance(caches, (list, tuple)) else (caches,)
    out = beam_select(logits, scores, finished=finished, pad_token=pad_token)
    parents = out[1].flatten()
    last = _check_caches(caches, parents.shape[0], parents.device)
    for i, cache in enumerate(caches):
        if hasattr(cache, "block_tables"):
            out[0].masked_fill_(cache.reorder(parents).view(out[0].shape) == 0, float("-inf"))
        else:
            cache.reorder(parents, set_lengths=last[cache.lengths.data_ptr()] == i)
    return out
