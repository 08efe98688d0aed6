"""The scaled 8-bit paged K/V cache: writing it and attending to it.

A cache is four tensors: ``k_cache`` / ``v_cache`` [num_pages, page_size, HKV, D]
in float8_e4m3fn or int8, and ``k_scale`` / ``v_scale`` [num_pages, HKV] fp32; a
stored value stands for byte * scale of its page and kv head.  ``block_table``
[R, max_blocks] maps a request's logical pages to pages; an id outside the cache
(-1) is no page: its keys are not visible and nothing is written for them.

* ``cache8_append``   quantises new keys and values into the pages
* ``cache8_decode``   attends one or a few rows per request (split over the keys)
* ``cache8_prefill``  attends many rows per request

``unlimited_dash_ops.attend_triton.dash_sparse_attn_decode`` takes the scales for
the router's selected blocks.  Serving only: no gradients.  No counterpart in the
reference, whose fp8 caches have no scales.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import UnsupportedShape
from .ops import _i32, _require_cuda

_FORMATS = {torch.int8: _lib.SRSWA_I8, torch.float8_e4m3fn: _lib.FP8_CODES[torch.float8_e4m3fn]}
_MOST_KEYS = 1 << 30          # of a request (the kernels' positions are 32-bit)


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    """(format code, num_pages, page_size, HKV, D) of a cache, its shapes and types checked."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} {k_cache.dtype} / v_cache {tuple(v_cache.shape)} "
                         f"{v_cache.dtype}: [num_pages, page_size, HKV, D] of one dtype expected")
    code = _FORMATS.get(k_cache.dtype)
    if code is None:
        raise UnsupportedShape(f"a scaled 8-bit cache holds float8_e4m3fn or int8, not {k_cache.dtype}")
    npages, page, HKV, D = k_cache.shape
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s.dtype != torch.float32 or s.shape != (npages, HKV):
            raise ValueError(f"{name} {tuple(s.shape)} {s.dtype} != [{npages}, {HKV}] float32")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise UnsupportedShape("head dim must be contiguous")
    return code, npages, page, HKV, D


def _same_device(*ts):
    """Every tensor on the first one's GPU."""
    _require_cuda(*ts)
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}: one GPU expected")
    return dev


def _table(block_table, rows):
    if block_table.dim() != 2 or block_table.shape[0] < rows:
        raise ValueError(f"block_table {tuple(block_table.shape)} for {rows} requests")
    bt = _i32(block_table)
    return bt if bt.stride(1) == 1 else bt.contiguous()


def cache8_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, *, cu_seqlens=None,
                  max_new_len=None):
    """Write new keys and values into the cache, in place.

    k, v [total, HKV, D] bf16 / fp16, read through their strides; request r's
    rows are cu_seqlens[r] .. cu_seqlens[r + 1) (None: total / R each) and become
    its keys start[r], start[r] + 1, ...; ``max_new_len`` the longest run (sizes
    the grid; needed with cu_seqlens, later rows of a longer run are not written).

    Per page and head the scale becomes the smallest power of two (>= 2^-100)
    that holds the page's new finite values, or stays the old one if that is
    larger and the page holds older keys; those are rounded again when it grows
    (exact in e4m3 but for subnormals).  Round to nearest even, infinities
    saturate, NaN stays NaN in e4m3 and is 0 in int8.  Rows behind the last new
    key are left as they are.  A page that starts with a new key takes nothing
    from what it held before.  Two requests of one call must not write the same
    page (fork it first: ``cache_pages.pages_reorder``)."""
    if _lib.host and _lib.host.append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, cu_seqlens,
                                      max_new_len) is None:
        return
    dev = _same_device(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, cu_seqlens)
    code, npages, page, HKV, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if k.dim() != 3 or k.shape[1:] != (HKV, D) or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} / v {tuple(v.shape)} {v.dtype} != [total, {HKV}, {D}]")
    if k.dtype not in (torch.bfloat16, torch.float16):
        raise UnsupportedShape(f"new keys and values are bf16 / fp16, not {k.dtype}")
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise UnsupportedShape("head dim must be contiguous")
    total, R = k.shape[0], start.numel()
    bt = _table(block_table, R)
    st = _i32(start).contiguous()
    cu = None
    if cu_seqlens is None:
        if R == 0 or total % R:
            raise ValueError(f"{total} rows do not divide among {R} requests")
        n = total // R
        if max_new_len is not None and int(max_new_len) != n:
            raise ValueError(f"max_new_len {max_new_len} without cu_seqlens: {n} rows each")
    else:
        cu = _i32(cu_seqlens).contiguous()
        if cu.numel() != R + 1 or max_new_len is None or int(max_new_len) < 0:
            raise ValueError(f"cu_seqlens [{cu.numel()}] for {R} requests needs R + 1 entries and max_new_len")
        n = min(int(max_new_len), total)
    ks, vs, kc, vc = k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    a = _lib.Cache8AppendArgs(
        k=k.data_ptr(), k_sn=ks[0], k_sh=ks[1], v=v.data_ptr(), v_sn=vs[0], v_sh=vs[1],
        k_cache=k_cache.data_ptr(), kc_sp=kc[0], kc_st=kc[1], kc_sh=kc[2],
        v_cache=v_cache.data_ptr(), vc_sp=vc[0], vc_st=vc[1], vc_sh=vc[2],
        k_scale=k_scale.data_ptr(), ks_sp=k_scale.stride(0), ks_sh=k_scale.stride(1),
        v_scale=v_scale.data_ptr(), vs_sp=v_scale.stride(0), vs_sh=v_scale.stride(1),
        block_table=bt.data_ptr(), bt_sr=bt.stride(0), start=st.data_ptr(), cu_seqlens=_lib.ptr(cu),
        R=R, total=total, max_new_len=n, HKV=HKV, D=D, max_blocks=bt.shape[1], num_pages=npages, page_size=page,
        dtype=_lib.dtype_code(k.dtype), kv_dtype=code)
    if total == 0 or npages == 0 or bt.shape[1] == 0:
        return
    with _lib.on_device(dev):
        _lib.check(_lib.lib().srswa_cache8_append(ctypes.byref(a), _lib.stream_ptr(dev)), "srswa_cache8_append")


def _attend_args(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu, mql, scale, window, sinks, out,
                 return_lse):
    """The argument struct of either form; returns (args, tensors to keep, out, lse, device)."""
    dev = _same_device(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu, out)
    code, npages, page, HKV, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)} != [total_q, HQ, {D}]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise UnsupportedShape(f"scaled 8-bit caches take bf16 / fp16 queries, not {q.dtype}")
    if q.stride(2) != 1:
        raise UnsupportedShape("head dim must be contiguous")
    total, HQ, _ = q.shape
    R = seq_lens.numel()
    bt = _table(block_table, R)
    sl = _i32(seq_lens).contiguous()
    if out is None:
        out = torch.empty(total, HQ, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError(f"out {tuple(out.shape)} {out.dtype}: q's shape and dtype, contiguous head dim expected")
    lse = torch.empty(total, HQ, dtype=torch.float32, device=dev) if return_lse else None
    qs, ks, vs, os_ = q.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    a = _lib.Cache8AttendArgs(
        q=q.data_ptr(), q_sn=qs[0], q_sh=qs[1], k_cache=k_cache.data_ptr(), k_sp=ks[0], k_st=ks[1], k_sh=ks[2],
        v_cache=v_cache.data_ptr(), v_sp=vs[0], v_st=vs[1], v_sh=vs[2],
        k_scale=k_scale.data_ptr(), ks_sp=k_scale.stride(0), ks_sh=k_scale.stride(1),
        v_scale=v_scale.data_ptr(), vs_sp=v_scale.stride(0), vs_sh=v_scale.stride(1),
        block_table=bt.data_ptr(), bt_sr=bt.stride(0), seq_lens=sl.data_ptr(), cu_seqlens_q=_lib.ptr(cu),
        out=out.data_ptr(), o_sn=os_[0], o_sh=os_[1],
        R=R, total_q=total, max_query_len=int(mql), HQ=HQ, HKV=HKV, D=D, max_blocks=bt.shape[1], num_pages=npages,
        page_size=page, window=window, sinks=sinks, scale=float(scale), dtype=_lib.dtype_code(q.dtype), kv_dtype=code)
    if lse is not None:
        a.lse = lse.data_ptr()
        a.lse_sn, a.lse_sh = HQ, 1
    return a, (bt, sl, cu), out, lse, dev


def _window(window, sinks):
    """The kernels' (window, sinks): 0 is no window."""
    if window is None and sinks == 0:
        return 0, 0
    w, s = 0 if window is None else int(window), int(sinks)
    if (window is not None and w < 1) or s < 0:
        raise ValueError(f"window {window} (None, or at least the row's own key) / sinks {sinks}")
    return min(w, _MOST_KEYS), min(s, _MOST_KEYS)


def _launch(form, a, dev):
    L = _lib.lib()
    with _lib.on_device(dev):
        nws = getattr(L, f"srswa_cache8_{form}_workspace")(ctypes.byref(a))
        ws = _lib.scratch(dev, nws)
        _lib.check(getattr(L, f"srswa_cache8_{form}")(ctypes.byref(a), _lib.ptr(ws), nws, _lib.stream_ptr(dev)),
                   f"srswa_cache8_{form}")


def cache8_decode(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, *, scale, decode_query_len=1,
                  window=None, sinks=0, out=None, return_lse=False):
    """Attention of each request's last ``decode_query_len`` tokens to its keys.

    q [R * decode_query_len, HQ, D] bf16 / fp16; seq_lens [R] keys stored, the
    rows' own included: row t of request r sits at p = seq_lens[r] -
    decode_query_len + t and sees the keys j <= p, with a window only j > p -
    window and the first ``sinks`` keys.  Returns out [rows, HQ, D] in q's dtype
    (0 for a row that sees no key) and, if asked, lse [rows, HQ] (natural log,
    -inf there).  A stored NaN reaches the rows that see its key, in V its own dim
    only."""
    w, s = _window(window, sinks)
    if _lib.host:
        got = _lib.host.attend(0, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, None, decode_query_len,
                               scale, w, s, out, bool(return_lse), None, None)
        if got is not NotImplemented:
            return got
    dql = int(decode_query_len)
    if dql < 1 or q.dim() != 3 or q.shape[0] != seq_lens.numel() * dql:
        raise ValueError(f"q {tuple(q.shape)} != {seq_lens.numel()} requests x {dql} rows")
    a, keep, out, lse, dev = _attend_args(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, None, dql,
                                          scale, w, s, out, return_lse)
    if a.R and a.num_pages and a.max_blocks:
        _launch("decode", a, dev)
    else:
        _no_keys(out, lse)
    return (out, lse) if return_lse else out


def cache8_prefill(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seq_lens, max_query_len, *,
                   scale, window=None, sinks=0, out=None, return_lse=False):
    """Attention of each request's last tokens, any number of them, to its keys.

    q [total_q, HQ, D], request r's rows cu_seqlens_q[r] .. cu_seqlens_q[r + 1)
    at the end of its seq_lens[r] keys; ``max_query_len`` the longest request
    (sizes the grid: later rows of a longer one are not written).  Visibility
    and returns as ``cache8_decode``; rows of q behind the last request are left
    as they are in ``out`` (and unset where ``out`` is not given)."""
    w, s = _window(window, sinks)
    if _lib.host:
        got = _lib.host.attend(1, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q,
                               max_query_len, scale, w, s, out, bool(return_lse), None, None)
        if got is not NotImplemented:
            return got
    if q.dim() != 3 or int(max_query_len) < 0:
        raise ValueError(f"q {tuple(q.shape)} / max_query_len {max_query_len}")
    _same_device(q, cu_seqlens_q)
    cu = _i32(cu_seqlens_q).contiguous()
    if cu.numel() != seq_lens.numel() + 1:
        raise ValueError(f"cu_seqlens_q [{cu.numel()}] for {seq_lens.numel()} requests")
    a, keep, out, lse, dev = _attend_args(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu,
                                          min(int(max_query_len), q.shape[0]), scale, w, s, out, return_lse)
    if a.R and a.num_pages and a.max_blocks:
        _launch("prefill", a, dev)
    else:
        _no_keys(out, lse)
    return (out, lse) if return_lse else out


def _no_keys(out, lse):
    """A cache without pages or a table without columns: no row sees a key."""
    out.zero_()
    if lse is not None:
        lse.fill_(float("-inf"))


def decode_selected(q, k_cache, v_cache, k_scale, v_scale, topk_idx, blk_bias, block_table, seq_lens, *,
                    decode_query_len, local_blocks, scale, out=None):
    """Block-sparse decode (``ops.gather_decode_paged``) over a scaled cache:
    the window of local_blocks pages, and before it the keys of the listed
    blocks with their slot's bias."""
    if _lib.host:
        got = _lib.host.attend(0, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, None, decode_query_len,
                               scale, min(int(local_blocks) * k_cache.shape[1], _MOST_KEYS), 0, out, False, topk_idx,
                               blk_bias)
        if got is not NotImplemented:
            return got
    _same_device(q, topk_idx, blk_bias)
    dql, total = int(decode_query_len), q.shape[0]
    page, HKV = k_cache.shape[1], k_cache.shape[2]
    if dql < 1 or q.dim() != 3 or total != seq_lens.numel() * dql:
        raise ValueError(f"q {tuple(q.shape)} != {seq_lens.numel()} requests x {dql} rows")
    if topk_idx.dim() != 3 or topk_idx.shape[:2] != (HKV, total):
        raise ValueError(f"topk_idx {tuple(topk_idx.shape)} != ({HKV}, {total}, K)")
    if topk_idx.shape[2] > 1024 or int(local_blocks) < 0:
        raise UnsupportedShape("at most 1024 slots, local_blocks >= 0")
    ti = _i32(topk_idx)
    bias = None
    if blk_bias is not None:
        if blk_bias.shape != topk_idx.shape:
            raise ValueError(f"blk_bias {tuple(blk_bias.shape)} != topk_idx {tuple(topk_idx.shape)}")
        bias = blk_bias.to(torch.float32)
        if bias.stride() != ti.stride():
            ti, bias = ti.contiguous(), bias.contiguous()
    a, keep, out, _, dev = _attend_args(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, None, dql,
                                        scale, min(int(local_blocks) * page, _MOST_KEYS), 0, out, False)
    ts = ti.stride()
    a.topk, a.t_sh, a.t_sn, a.t_sk, a.topk_n = ti.data_ptr(), ts[0], ts[1], ts[2], ti.shape[2]
    a.bias = _lib.ptr(bias)
    if not (a.R and a.num_pages and a.max_blocks) or (a.topk_n == 0 and a.window == 0):
        _no_keys(out, None)
    else:
        if a.topk_n == 0:
            a.topk = q.data_ptr()              # no slot is read; only marks the form
        _launch("decode", a, dev)
    return out
