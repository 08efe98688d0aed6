"""The pages of a paged cache: dealing them to requests, reordering rows
(sharing, copying, freeing pages) and compacting the pool.

The state of a pool is a ``PageTable``: ``block_table`` [R, W] page ids (-1 =
none), ``seq_lens`` [R], ``ref`` [num_pages] how many rows hold a page (0 = free).
Each function returns a new state (into ``out`` if given, which must not overlap
the state: two states used in turn serve a captured graph) and moves page data in
place in every cache of ``caches``: any tensors whose first dimension is the page
(K, V, scales, index keys, summaries, of every layer), each page contiguous.

Free pages are taken lowest first, so results do not depend on the order of
execution.  No call waits for the GPU: counts come back as device tensors [1].
No counterpart in the reference, whose serving stack keeps this on the host.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import UnsupportedShape
from .ops import _i32, _require_cuda


class PageTable(NamedTuple):
    block_table: torch.Tensor
    seq_lens: torch.Tensor
    ref: torch.Tensor


_ENTRIES = {"reserve": 0, "reorder": 1, "compact": 2}


def _overlap(x, y):
    """Whether two tensors' memory ranges meet."""
    def span(t):
        n = sum((s - 1) * abs(d) for s, d in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    (a, b), (c, d) = span(x), span(y)
    return a < d and c < b


def _check(state, what):
    bt, sl, ref = state
    if bt.dim() != 2 or sl.shape != (bt.shape[0],) or ref.dim() != 1:
        raise ValueError(f"{what}: block_table {tuple(bt.shape)}, seq_lens {tuple(sl.shape)}, ref {tuple(ref.shape)}: "
                         "[R, W], [R], [num_pages] expected")
    for t in state:
        if t.dtype != torch.int32:
            raise UnsupportedShape(f"{what}: block_table, seq_lens and ref are int32")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise UnsupportedShape(f"{what}: block_table rows, seq_lens and ref must be contiguous")
    if bt.shape[0] == 0 or bt.shape[1] == 0 or ref.numel() == 0:
        raise ValueError(f"{what}: an empty block_table or pool")


def _run(entry, state, rows, caches, page_size, out):
    if out is None and _lib.host:
        got = _lib.host.pages(_ENTRIES[entry], *state, rows, caches, page_size)
        if got is not NotImplemented:
            return PageTable(*got[:3]), got[3]
    name = f"srswa_pages_{entry}"
    _require_cuda(*state, rows, *caches)
    _check(state, name)
    bt, sl, ref = state
    dev = bt.device
    (R, W), N = bt.shape, ref.numel()
    if out is None:
        out = PageTable(torch.empty(R, W, dtype=torch.int32, device=dev), torch.empty_like(sl), torch.empty_like(ref))
    else:
        _require_cuda(*out)
        _check(out, name)
        if any(x.shape != y.shape for x, y in zip(out, state)):
            raise ValueError(f"{name}: out's shapes differ from the state's")
        if any(_overlap(x, y) for x in out for y in state):
            raise ValueError(f"{name}: out overlaps the state")
    for t in (*state, rows, *caches, *out):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}: one GPU expected")
    if rows is not None:
        if rows.shape != (R,):
            raise ValueError(f"{name}: {tuple(rows.shape)} values for {R} rows")
        rows = _i32(rows).contiguous()
    table = (_lib.PageCache * max(1, len(caches)))()
    filled = 0
    for t in caches:
        if t.dim() < 1 or t.shape[0] != N:
            raise ValueError(f"{name}: cache {tuple(t.shape)} does not have {N} pages")
        n = t.numel() // N
        if n == 0:
            continue
        if not t[0].is_contiguous() or (N > 1 and t.stride(0) < n):
            raise UnsupportedShape(f"{name}: each page of a cache must be contiguous, pages apart")
        c, e = table[filled], t.element_size()
        c.base, c.stride, c.bytes = t.data_ptr(), (t.stride(0) if N > 1 else n) * e, n * e
        filled += 1
    count = torch.empty(1, dtype=torch.int32, device=dev)
    nt, ns, nr = out
    a = _lib.PagesArgs(block_table=bt.data_ptr(), bt_sr=bt.stride(0), seq_lens=sl.data_ptr(), ref=ref.data_ptr(),
                       rows=_lib.ptr(rows), block_table_out=nt.data_ptr(), bto_sr=nt.stride(0),
                       seq_lens_out=ns.data_ptr(), ref_out=nr.data_ptr(), count=count.data_ptr(),
                       caches=ctypes.addressof(table), ncaches=filled, R=R, W=W, num_pages=N,
                       page_size=int(page_size))
    L = _lib.lib()
    with _lib.on_device(dev):
        nws = L.srswa_pages_workspace(ctypes.byref(a))
        ws = _lib.scratch(dev, nws)
        _lib.check(getattr(L, name)(ctypes.byref(a), _lib.ptr(ws), nws, _lib.stream_ptr(dev)), name)
    return PageTable(nt, ns, nr), count


def pages_reserve(state, new_lens, *, page_size, out=None):
    """Give every row the pages that its first ``new_lens`` [R] keys need.

    Entries below ceil(new_lens / page_size) that hold no page take the lowest
    free ones, in row and block order; pages a row has beyond that stay.
    Returns (state with seq_lens = new_lens, missing): ``missing`` counts the
    entries that stayed -1 because the pool ran out (keys there are neither
    written nor seen)."""
    return _run("reserve", state, new_lens, (), page_size, out)


def pages_reorder(state, parents, caches, *, page_size, out=None):
    """Let row r continue row parents[r] (beam search, forking, freeing).

    parents [R]: r keeps a row, another row forks or replaces it, any value
    outside [0, R) frees it (length 0).  Full pages are shared; of the rows
    that continue one parent the first keeps its remaining pages, each other
    one gets a copy of the page the parent has begun, in every cache.  Pages
    nobody holds any more become free and may be dealt in the same call.
    Returns (state, missing): ``missing`` counts copies that found no free page
    (that entry is -1).  A shared page stays shared: a row's ``seq_lens`` must not
    be set back into one."""
    return _run("reorder", state, parents, tuple(caches), page_size, out)


def pages_compact(state, caches, *, out=None):
    """Move the held pages to the lowest ids: with n pages held, those at or past
    n go, in order, into the free ones below n, in every cache, and the table
    follows.  Returns (state, n)."""
    return _run("compact", state, None, tuple(caches), 1, out)
