"""Paged int4 KV cache: a pool of pages shared by the sequences of a batch.

A page holds ``page_size`` rows (a power of two, 32 to 1024) of every kv head;
the pool's tensors are ``(num_pages, num_kv_heads, page_size, .)`` in the int4
layout of :mod:`gemma4metal_amd.turboquant`, and ``block_tables`` (int32,
``(sequences, max_pages)``) names the page of each ``page_size`` rows of a
sequence, -1 where there is none.  The reference has no paged cache: its cache
is one growing array per layer (``engine/gemma4_multilayer.cpp:230-249``).

As in ``turboquant.py``, torch holds device memory and streams; every
computation runs in ``libturboquant_hip.so``.  Tensors of one call lie on one
device, which need not be the current one.  Every function also takes
``stream=`` (a ``torch.cuda.Stream`` of that device; the current one by default).

Workspaces are cached per (device, stream).  Calls captured into HIP graphs
that may be replayed at the same time, or beside eager calls of the stream that
they were captured on, need a ``workspace=`` each (uint8, zero-filled, at least
the ``*_workspace_size`` bytes).

Attention is off by 0.2e-6 to 2e-6 of its result against 64 bits, as far as
products in 32 bits are.
"""
from __future__ import annotations

import ctypes
import functools
import inspect
from typing import Optional, Union

import torch

from . import _lib
from ._lib import call
from .turboquant import _DT, _MODES, _QUANT_DT, _check_cuda, _ptr, _sb_dtype, _size_caches, _stream
from .turboquant import workspace as _cached_workspace

# Buffers that a captured graph points to: kept for good, since the cached one
# of a stream is replaced when a larger call comes.
_captured: dict = {}


def _need(cond: bool, msg: str):
    if not cond:
        raise ValueError(msg)


def _workspace(ws: Optional[torch.Tensor], nbytes: int, device: torch.device, stream: int) -> torch.Tensor:
    if ws is None:
        ws = _cached_workspace(nbytes, device, stream)
        if torch.cuda.is_current_stream_capturing():
            _captured[ws.data_ptr()] = ws
        return ws
    _check_cuda("workspace", ws)
    if ws.dtype != torch.uint8 or ws.numel() < nbytes or ws.device != device:
        raise ValueError(f"workspace must be uint8 of at least {nbytes} bytes on {device}")
    return ws


def _placed(fn):
    """Runs fn with its first tensor's device, and ``stream=`` where given,
    current: launches, allocations and the capture state all go by those."""
    sig = inspect.signature(fn)
    name = next(iter(sig.parameters))

    @functools.wraps(fn)
    def run(*args, stream=None, **kw):
        first = args[0] if args else kw.get(name)
        t = first[0] if isinstance(first, (list, tuple)) and first else first
        if isinstance(t, torch.Tensor) and t.is_cuda:
            if stream is not None:
                _need(stream.device == t.device, "stream must be on the tensors' device")
                with torch.cuda.stream(stream):
                    return fn(*args, **kw)
            if t.device.index != torch.cuda.current_device():
                with torch.cuda.device(t.device):
                    return fn(*args, **kw)
        return fn(*args, **kw)
    extra = inspect.Parameter("stream", inspect.Parameter.KEYWORD_ONLY, default=None, annotation=Optional[torch.cuda.Stream])
    run.__signature__ = sig.replace(parameters=[*sig.parameters.values(), extra])
    return run


def _check_pages(pages, D: int, device, lead: int = 0):
    """(num_pages, Hkv, page_size, scale dtype) of six page tensors with
    ``lead`` leading axes."""
    names = ("k_quant", "k_scales", "k_biases", "v_quant", "v_scales", "v_biases")
    for n, t in zip(names, pages):
        _check_cuda(n, t)
        if t.device != device:
            raise ValueError(f"{n} must be on {device}")
    kq = pages[0]
    _need(kq.dim() == 4 + lead and kq.shape[-1] == D // 8 and D % 64 == 0,
          "k_quant must be (num_pages, Hkv, page_size, D/8) uint32")
    shape = kq.shape[:-1]
    sbt = _sb_dtype("k_scales", pages[1])
    for i, (n, t) in enumerate(zip(names, pages)):
        if i % 3 == 0:
            if t.shape != kq.shape or t.dtype not in _QUANT_DT:
                raise ValueError(f"{n} must be {tuple(kq.shape)} uint32")
        elif t.shape != shape + (D // 64,) or t.dtype != pages[1].dtype:
            raise ValueError(f"{n} must be {tuple(shape) + (D // 64,)} of one scale dtype")
    return shape[lead], shape[lead + 1], shape[lead + 2], sbt


def _pages_fine(pages, D: int, di: int) -> bool:
    """What _check_pages checks of pages without leading axes, as one expression:
    a decode call's host time is part of a short layer's."""
    kq, ks, kb, vq, vs, vb = pages
    try:
        shape, dt = kq.shape, ks.dtype
        rows = shape[:3] + (D // 64,)
        return (len(shape) == 4 and shape[3] == D // 8 and D % 64 == 0 and vq.shape == shape
                and ks.shape == rows and kb.shape == rows and vs.shape == rows and vb.shape == rows
                and dt is kb.dtype and dt is vs.dtype and dt is vb.dtype
                and (dt is torch.float16 or dt is torch.float32)
                and kq.dtype in _QUANT_DT and vq.dtype in _QUANT_DT
                and kq.get_device() == di and ks.get_device() == di and kb.get_device() == di
                and vq.get_device() == di and vs.get_device() == di and vb.get_device() == di
                and kq.is_contiguous() and ks.is_contiguous() and kb.is_contiguous()
                and vq.is_contiguous() and vs.is_contiguous() and vb.is_contiguous())
    except (AttributeError, IndexError):
        return False


def _ints_fine(t, shape, di: int) -> bool:
    return (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == shape and t.get_device() == di
            and t.is_contiguous())


def _check_ints(name: str, t: torch.Tensor, shape, device):
    _check_cuda(name, t)
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"{name} must be int32 {tuple(shape)} on {device}")


def _out(out, shape, device):
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=device)
    _check_cuda("out", out)
    if tuple(out.shape) != tuple(shape) or out.dtype != torch.float32 or out.device != device:
        raise ValueError(f"out must be {tuple(shape)} float32 on {device}")
    return out


# ---------------------------------------------------------------------------
# append and attention
# ---------------------------------------------------------------------------

@_placed
def kv_append_int4_paged(k_new: torch.Tensor, v_new: torch.Tensor,
                         k_quant: torch.Tensor, k_scales: torch.Tensor, k_biases: torch.Tensor,
                         v_quant: torch.Tensor, v_scales: torch.Tensor, v_biases: torch.Tensor,
                         block_tables: torch.Tensor, positions: torch.Tensor, *, mode: str = "mlx") -> None:
    """Quantize k_new / v_new (B, Hkv, T, D) into rows positions[b] ..
    positions[b]+T-1 of sequence b's pages.  Rows past the table, or whose entry
    names no page, are dropped."""
    for n, t in (("k_new", k_new), ("v_new", v_new)):
        _check_cuda(n, t)
    _need(k_new.dim() == 4 and k_new.shape == v_new.shape and k_new.dtype == v_new.dtype
          and k_new.device == v_new.device, "k_new / v_new must both be (B, Hkv, T, D) of one dtype")
    _need(k_new.dtype in _DT, "k_new must be float32, float16 or bfloat16")
    B, Hkv, T, D = k_new.shape
    pages = (k_quant, k_scales, k_biases, v_quant, v_scales, v_biases)
    dev = k_new.device
    di = dev.index
    if not _pages_fine(pages, D, di):
        _check_pages(pages, D, dev)
    N, H, page, _ = k_quant.shape
    _need(H == Hkv, "k_new and the pages must have the same kv heads")
    _need(block_tables.dim() == 2, "block_tables must be (B, max_pages)")
    P = block_tables.shape[1]
    if not _ints_fine(block_tables, (B, P), di):
        _check_ints("block_tables", block_tables, (B, P), dev)
    if not _ints_fine(positions, (B,), di):
        _check_ints("positions", positions, (B,), dev)
    call("tq_kv_append_int4_paged", k_new.data_ptr(), v_new.data_ptr(), _DT[k_new.dtype],
         *[t.data_ptr() for t in pages], _DT[k_scales.dtype], B, Hkv, D, page, N, block_tables.data_ptr(), P,
         positions.data_ptr(), T, _MODES[mode], _stream(None))


@functools.lru_cache(maxsize=256)
def _prefill_ws_size(*shape) -> int:
    return _lib.load().tq_sdpa_int4_paged_prefill_workspace_size(*shape)


@functools.lru_cache(maxsize=256)
def _paged_ws_size(*shape) -> int:
    return _lib.load().tq_sdpa_int4_paged_workspace_size(*shape)


_size_caches += [_paged_ws_size, _prefill_ws_size]


@_placed
def sdpa_int4_paged(queries: torch.Tensor,
                    k_quant: torch.Tensor, k_scales: torch.Tensor, k_biases: torch.Tensor,
                    v_quant: torch.Tensor, v_scales: torch.Tensor, v_biases: torch.Tensor,
                    block_tables: torch.Tensor, seq_lens: torch.Tensor, gqa_factor: int, scale: float = 1.0,
                    sliding_window: int = 0, num_sinks: int = 0, *, windows: Optional[torch.Tensor] = None,
                    shared_prefix: int = 0, prefix_table: Optional[torch.Tensor] = None,
                    max_kv_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Batched decode attention over pages.  queries (B, Hq, D) f32|f16|bf16;
    block_tables int32 (B, max_pages); seq_lens / windows int32 (B).  The query
    of sequence b attends key t < seq_lens[b] iff its window W is 0, t >=
    seq_lens[b] - W, or t < num_sinks (the first tokens stay visible); none: 0.

    ``shared_prefix`` (a multiple of the page size): the first rows of every
    sequence lie in the same pages, as after :func:`kv_pages_fork`, and are
    attended once for the whole batch.  They are those of sequence 0's table or,
    where it has been freed or evicted from, of ``prefix_table`` (int32
    (shared_prefix / page size,)), which must name every prefix page that a
    sequence attends (:meth:`PagedInt4KVCache.prefix_table`).
    ``max_kv_len`` bounds the lengths (longer ones are cut to it); the table's
    reach by default.  Returns (B, Hq, D) float32."""
    _check_cuda("queries", queries)
    _need(queries.dim() == 3 and queries.dtype in _DT, "queries must be (B, Hq, D) float32, float16 or bfloat16")
    B, Hq, D = queries.shape
    dev = queries.device
    di = dev.index
    pages = (k_quant, k_scales, k_biases, v_quant, v_scales, v_biases)
    if not _pages_fine(pages, D, di):
        _check_pages(pages, D, dev)
    N, Hkv, page, _ = k_quant.shape
    sbt = _DT[k_scales.dtype]
    _need(block_tables.dim() == 2, "block_tables must be (B, max_pages)")
    P = block_tables.shape[1]
    if not _ints_fine(block_tables, (B, P), di):
        _check_ints("block_tables", block_tables, (B, P), dev)
    if not _ints_fine(seq_lens, (B,), di):
        _check_ints("seq_lens", seq_lens, (B,), dev)
    if windows is not None:
        _check_ints("windows", windows, (B,), dev)
    mx = P * page if max_kv_len is None else int(max_kv_len)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    else:
        out = _out(out, (B, Hq, D), dev)
    sh = _stream(None)
    ws = _workspace(workspace, _paged_ws_size(B, Hq, Hkv, D, mx, int(shared_prefix)), dev, sh)
    if prefix_table is None:
        name, prefix = "tq_sdpa_int4_paged", ()
    else:
        _need(page > 0, "k_quant must have rows")
        _check_ints("prefix_table", prefix_table, (int(shared_prefix) // page,), dev)
        name, prefix = "tq_sdpa_int4_paged_prefix", (prefix_table.data_ptr(),)
    call(name, queries.data_ptr(), _DT[queries.dtype], *[t.data_ptr() for t in pages], sbt, out.data_ptr(), B, Hq, Hkv,
         D, page, N, block_tables.data_ptr(), P, seq_lens.data_ptr(), _ptr(windows), mx, int(gqa_factor), float(scale),
         int(sliding_window), int(num_sinks), *prefix, int(shared_prefix), ws.data_ptr(), ws.numel(), sh)
    return out


@_placed
def sdpa_int4_paged_prefill(queries: torch.Tensor,
                            k_quant: torch.Tensor, k_scales: torch.Tensor, k_biases: torch.Tensor,
                            v_quant: torch.Tensor, v_scales: torch.Tensor, v_biases: torch.Tensor,
                            block_table: torch.Tensor, n_prior: int, gqa_factor: int, scale: float = 1.0,
                            sliding_window: int = 0, num_sinks: int = 0, *, out: Optional[torch.Tensor] = None,
                            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Prompt (multi-query) attention of one sequence over its pages: queries
    (n_new, Hq, D) at positions n_prior .. n_prior+n_new-1, whose rows are
    already appended; block_table int32 (max_pages,).  Query i attends key t <=
    n_prior + i iff the window W is 0, n_prior + i - t < W, or t < num_sinks.
    Returns (n_new, Hq, D) float32."""
    _check_cuda("queries", queries)
    _need(queries.dim() == 3 and queries.dtype in _DT, "queries must be (n_new, Hq, D) float32, float16 or bfloat16")
    S, Hq, D = queries.shape
    dev = queries.device
    pages = (k_quant, k_scales, k_biases, v_quant, v_scales, v_biases)
    if not _pages_fine(pages, D, dev.index):
        _check_pages(pages, D, dev)
    N, Hkv, page, _ = k_quant.shape
    sbt = _DT[k_scales.dtype]
    _need(block_table.dim() == 1, "block_table must be (max_pages,)")
    _check_ints("block_table", block_table, block_table.shape, dev)
    out = _out(out, (S, Hq, D), dev)
    sh = _stream(None)
    ws = _workspace(workspace, _prefill_ws_size(Hq, Hkv, D, int(n_prior), S), dev, sh)
    call("tq_sdpa_int4_paged_prefill", queries.data_ptr(), _DT[queries.dtype], *[t.data_ptr() for t in pages], sbt,
         out.data_ptr(), Hq, Hkv, D, page, N, block_table.data_ptr(), block_table.shape[0], int(n_prior), S,
         int(gqa_factor), float(scale), int(sliding_window), int(num_sinks), ws.data_ptr(), ws.numel(), sh)
    return out


# ---------------------------------------------------------------------------
# page management
# ---------------------------------------------------------------------------

def _check_state(block_tables, refs, lengths=None):
    _check_cuda("block_tables", block_tables)
    _need(block_tables.dim() == 2, "block_tables must be (sequences, max_pages)")
    dev = block_tables.device
    S, P = block_tables.shape
    _check_ints("block_tables", block_tables, (S, P), dev)
    _need(isinstance(refs, torch.Tensor) and refs.dim() == 1, "refs must be int32 (num_pages,)")
    _check_ints("refs", refs, refs.shape, dev)
    if lengths is not None:
        _check_ints("lengths", lengths, (S,), dev)
    return S, P, refs.shape[0], dev


def _six(pages, refs, device):
    """Six page tensors, [layers,] num_pages first, as the C array, and what
    describes them."""
    _need(len(pages) == 6, "pages must be the six page tensors")
    kq = pages[0]
    _check_cuda("k_quant", kq)
    _need(kq.dim() in (4, 5), "page tensors must be ([layers,] num_pages, Hkv, page_size, .)")
    lead = kq.dim() - 4
    N, Hkv, page, sbt = _check_pages(pages, kq.shape[-1] * 8, device, lead)
    _need(refs is None or N == refs.shape[0], "refs must have one count a page")
    arr = (ctypes.c_void_p * 6)(*[t.data_ptr() for t in pages])
    return arr, sbt, (kq.shape[0] if lead else 1), Hkv, kq.shape[-1] * 8, N, page


@functools.lru_cache(maxsize=64)
def _pages_ws_size(S: int, N: int) -> int:
    return _lib.load().tq_kv_pages_workspace_size(S, N)


def _pages_ws(ws, S, N, device):
    nbytes = _pages_ws_size(S, N)
    if ws is None:
        # a buffer of the call's own: plans overwrite what attention keeps zeroed
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return _workspace(ws, nbytes, device, 0)


@_placed
def kv_pages_reserve(block_tables: torch.Tensor, refs: torch.Tensor, lengths: torch.Tensor, n_new: torch.Tensor,
                     page_size: int, *, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gives every sequence with n_new[s] > 0 the pages its next n_new[s] rows
    need, the lowest free ones first.  refs int32 (num_pages,) counts the table
    entries that name a page.  Returns int32 (sequences,): 1 where the request
    was carried out, 0 where there was none or pages ran out (in sequence
    order) or the table is too short."""
    S, P, N, dev = _check_state(block_tables, refs, lengths)
    _check_ints("n_new", n_new, (S,), dev)
    granted = torch.empty(S, dtype=torch.int32, device=dev)
    ws = _pages_ws(workspace, S, N, dev)
    call("tq_kv_pages_reserve", _ptr(block_tables), _ptr(refs), _ptr(lengths), _ptr(n_new), _ptr(granted), S, P, N,
         int(page_size), _ptr(ws), ws.numel(), _stream(None))
    return granted


@_placed
def kv_pages_advance(block_tables: torch.Tensor, refs: torch.Tensor, lengths: torch.Tensor, n_new: torch.Tensor,
                     page_size: int) -> torch.Tensor:
    """Counts appended rows: lengths[s] += n_new[s] where every one of those rows
    has a page, as after a granted :func:`kv_pages_reserve`.  Elsewhere the length
    stays: the append dropped rows, and a page that the sequence gets later holds
    what its last owner left there.  A negative n_new takes rows back (not into
    pages that other sequences share).  Returns int32 (sequences,): 1 where rows
    were counted."""
    S, P, N, dev = _check_state(block_tables, refs, lengths)
    _check_ints("n_new", n_new, (S,), dev)
    advanced = torch.empty(S, dtype=torch.int32, device=dev)
    call("tq_kv_pages_advance", _ptr(block_tables), _ptr(lengths), _ptr(n_new), _ptr(advanced), S, P, N,
         int(page_size), _stream(None))
    return advanced


@_placed
def kv_pages_fork(pages, block_tables: torch.Tensor, refs: torch.Tensor, lengths: torch.Tensor,
                  parents: torch.Tensor, *, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Makes every sequence s with parents[s] >= 0 a continuation of that
    sequence: full pages are shared, the partly filled last one is copied.
    ``pages``: the six page tensors, ([layers,] num_pages, Hkv, page_size, .).
    Returns int32 (sequences,): 1 where s was forked, 0 where it was not asked
    for or refused (s not empty, a parent that is s, out of range or itself
    forked into, no free page)."""
    S, P, N, dev = _check_state(block_tables, refs, lengths)
    arr, sbt, L, Hkv, D, _, page = _six(pages, refs, dev)
    _check_ints("parents", parents, (S,), dev)
    granted = torch.empty(S, dtype=torch.int32, device=dev)
    ws = _pages_ws(workspace, S, N, dev)
    call("tq_kv_pages_fork", arr, sbt, L, Hkv, D, _ptr(block_tables), _ptr(refs), _ptr(lengths), _ptr(parents),
         _ptr(granted), S, P, N, page, _ptr(ws), ws.numel(), _stream(None))
    return granted


@_placed
def kv_pages_free(block_tables: torch.Tensor, refs: torch.Tensor, lengths: torch.Tensor, which: torch.Tensor) -> None:
    """Ends the sequences with which[s] != 0: pages lose a reference, table rows
    become -1 and lengths 0.  See ``prefix_table`` of :func:`sdpa_int4_paged` where
    sequences share a prefix."""
    S, P, N, dev = _check_state(block_tables, refs, lengths)
    _check_ints("which", which, (S,), dev)
    call("tq_kv_pages_free", _ptr(block_tables), _ptr(refs), _ptr(lengths), _ptr(which), S, P, N, _stream(None))


@_placed
def kv_pages_evict(block_tables: torch.Tensor, refs: torch.Tensor, lengths: torch.Tensor, page_size: int,
                   sliding_window: int, num_sinks: int = 0, which: Optional[torch.Tensor] = None) -> None:
    """Gives up the pages that lie wholly between the first num_sinks rows and
    the window's last ``sliding_window`` ones, of the sequences with which[s]
    != 0 (all by default); their entries become -1.  The tables are every layer's:
    layers that see further back lose those keys too.  See ``prefix_table`` of
    :func:`sdpa_int4_paged` where sequences share a prefix."""
    S, P, N, dev = _check_state(block_tables, refs, lengths)
    if which is not None:
        _check_ints("which", which, (S,), dev)
    call("tq_kv_pages_evict", _ptr(block_tables), _ptr(refs), _ptr(lengths), _ptr(which), S, P, N, int(page_size),
         int(sliding_window), int(num_sinks), _stream(None))


@_placed
def kv_pages_compact(pages, block_tables: torch.Tensor, refs: torch.Tensor, *,
                     out: Optional[tuple] = None, workspace: Optional[torch.Tensor] = None):
    """Moves the pages in use to the front of the pool, in place.  Returns
    (block_tables, refs, live): the tables and counts of the new places, in new
    tensors or in ``out`` = (tables, refs), which may be the inputs, and the
    number of pages in use, int32 ()."""
    S, P, N, dev = _check_state(block_tables, refs)
    arr, sbt, L, Hkv, D, _, page = _six(pages, refs, dev)
    tables, counts = (torch.empty_like(block_tables), torch.empty_like(refs)) if out is None else out
    _check_ints("out tables", tables, (S, P), dev)
    _check_ints("out refs", counts, (N,), dev)
    live = torch.empty((), dtype=torch.int32, device=dev)
    ws = _pages_ws(workspace, S, N, dev)
    call("tq_kv_pages_compact", arr, sbt, L, Hkv, D, _ptr(block_tables), _ptr(refs), _ptr(tables), _ptr(counts),
         _ptr(live), S, P, N, page, _ptr(ws), ws.numel(), _stream(None))
    return tables, counts, live


@_placed
def kv_pages_copy(pages, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page src[i] to page dst[i] in all six tensors and every layer.
    Pairs out of range are skipped; no destination may occur twice or be
    another pair's source."""
    _need(len(pages) == 6, "pages must be the six page tensors")
    _check_cuda("k_quant", pages[0])
    dev = pages[0].device
    arr, sbt, L, Hkv, D, N, page = _six(pages, None, dev)
    _need(isinstance(src, torch.Tensor) and src.dim() == 1, "src must be int32 (n,)")
    _check_ints("src", src, src.shape, dev)
    _check_ints("dst", dst, src.shape, dev)
    call("tq_kv_pages_copy", arr, sbt, L, Hkv, D, N, page, _ptr(src), _ptr(dst), src.shape[0], _stream(None))


class PagedInt4KVCache:
    """A pool of int4 KV pages for the layers of a model, and the sequences in
    it: ``block_tables``, ``lengths`` and page reference counts on the device, so
    that a decode step with its bookkeeping can be captured into a HIP graph.
    Methods run on the current stream.

    The layers share the tables: those with a window and those that see everything
    need a cache each where ``evict`` is used.

    One step of a batch is ``reserve(n_new)``, ``append(layer, k, v)`` and
    ``attend(layer, q, ...)`` per layer, then ``advance(n_new)``; attention
    covers the rows appended since the last ``advance`` too.  A sequence that
    ``reserve`` refused (0 in what it returns) is left behind by the step: its
    rows are dropped, ``advance`` does not count them, and its attention is not
    that of the new token.  It asks for the same rows again."""

    def __init__(self, num_pages: int, page_size: int, sequences: int, max_pages: int, num_kv_heads: int,
                 head_dim: int, device, *, num_layers: int = 1, scale_dtype: torch.dtype = torch.float16):
        lead = (num_layers, num_pages, num_kv_heads, page_size)
        self.page_size, self.D, self.Hkv, self.num_layers = page_size, head_dim, num_kv_heads, num_layers
        self.kq = torch.zeros(lead + (head_dim // 8,), dtype=torch.uint32, device=device)
        self.vq = torch.zeros_like(self.kq)
        self.ks = torch.zeros(lead + (head_dim // 64,), dtype=scale_dtype, device=device)
        self.kb, self.vs, self.vb = (torch.zeros_like(self.ks) for _ in range(3))
        self.block_tables = torch.full((sequences, max_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)

    def tensors(self):
        return self.kq, self.ks, self.kb, self.vq, self.vs, self.vb

    def layer(self, i: int):
        return tuple(t[i] for t in self.tensors())

    def reserve(self, n_new: torch.Tensor) -> torch.Tensor:
        return kv_pages_reserve(self.block_tables, self.refs, self.lengths, n_new, self.page_size)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, *, mode: str = "mlx"):
        """k_new / v_new (sequences, Hkv, T, D) behind each sequence's rows."""
        kv_append_int4_paged(k_new, v_new, *self.layer(layer), self.block_tables, self.lengths, mode=mode)

    def append_one(self, layer: int, sequence: int, k_new: torch.Tensor, v_new: torch.Tensor, *, mode: str = "mlx"):
        """k_new / v_new (Hkv, T, D) behind one sequence's rows (a prompt)."""
        s = slice(sequence, sequence + 1)
        kv_append_int4_paged(k_new[None], v_new[None], *self.layer(layer), self.block_tables[s], self.lengths[s],
                             mode=mode)

    def advance(self, n_new: torch.Tensor) -> torch.Tensor:
        """Counts the rows appended in this step, of the sequences that have pages
        for them: a sequence that ``reserve`` refused keeps its length.  Returns
        int32 (sequences,): 1 where rows were counted."""
        if not _ints_fine(n_new, self.lengths.shape, self.lengths.get_device()):
            n_new = torch.zeros_like(self.lengths).add_(n_new)
        return kv_pages_advance(self.block_tables, self.refs, self.lengths, n_new, self.page_size)

    def attend(self, layer: int, queries: torch.Tensor, gqa_factor: int, scale: float = 1.0, sliding_window: int = 0,
               num_sinks: int = 0, *, new: Union[int, torch.Tensor] = 1, windows: Optional[torch.Tensor] = None,
               shared_prefix: int = 0, prefix_table: Optional[torch.Tensor] = None, max_kv_len: Optional[int] = None,
               out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Decode attention of (sequences, Hq, D) queries over the lengths plus
        the ``new`` rows appended in this step: one count for all, or int32
        (sequences,).  A sequence that appended fewer rows than that attends
        whatever its pages hold behind them; its result means nothing."""
        return sdpa_int4_paged(queries, *self.layer(layer), self.block_tables, self.lengths + new, gqa_factor, scale,
                               sliding_window, num_sinks, windows=windows, shared_prefix=shared_prefix,
                               prefix_table=prefix_table, max_kv_len=max_kv_len, out=out, workspace=workspace)

    def prefix_table(self, shared_prefix: int, sequences: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The pages of the first ``shared_prefix`` rows, which these sequences (an
        index tensor; all by default) share as far as they have not given them up:
        int32 (shared_prefix / page size,), for :meth:`attend`.  Good until pages
        move or are given up."""
        t = self.block_tables if sequences is None else self.block_tables[sequences]
        return t[:, :shared_prefix // self.page_size].amax(0)

    def prefill(self, layer: int, sequence: int, queries: torch.Tensor, n_prior: int, gqa_factor: int,
                scale: float = 1.0, sliding_window: int = 0, num_sinks: int = 0, *,
                out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Prompt attention of one sequence: queries (n_new, Hq, D) behind
        n_prior rows, theirs already appended."""
        return sdpa_int4_paged_prefill(queries, *self.layer(layer), self.block_tables[sequence], n_prior, gqa_factor,
                                       scale, sliding_window, num_sinks, out=out, workspace=workspace)

    def fork(self, parents: torch.Tensor) -> torch.Tensor:
        return kv_pages_fork(self.tensors(), self.block_tables, self.refs, self.lengths, parents)

    def free(self, which: torch.Tensor) -> None:
        kv_pages_free(self.block_tables, self.refs, self.lengths, which)

    def evict(self, sliding_window: int, num_sinks: int = 0, which: Optional[torch.Tensor] = None):
        kv_pages_evict(self.block_tables, self.refs, self.lengths, self.page_size, sliding_window, num_sinks, which)

    def compact(self) -> torch.Tensor:
        """Packs the pool in place; returns the number of pages in use."""
        return kv_pages_compact(self.tensors(), self.block_tables, self.refs, out=(self.block_tables, self.refs))[2]
