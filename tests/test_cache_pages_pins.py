"""The page pool on the CPU: invariants of the oracle and the refusals of the
entry points before any launch."""

import ctypes

import pytest
import torch

from oracle import cache8_oracle as O
from srswa import UnsupportedShape, _lib, cache_pages


def _pool(seed, R=6, W=7, N=60, page=16):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, W * page + 1, (R,), generator=g).tolist()
    perm, o, table = torch.randperm(N, generator=g).tolist(), 0, []
    for n in lens:
        m = -(-n // page)
        table.append(perm[o:o + m] + [-1] * (W - m))
        o += m
    ref = [0] * N
    for row in table:
        for x in row:
            if x >= 0:
                ref[x] += 1
    return table, lens, ref


def _count(table, N):
    ref = [0] * N
    for row in table:
        for x in row:
            if x >= 0:
                ref[x] += 1
    return ref


def test_references_count_the_rows_and_copies_are_private():
    for seed in range(8):
        table, lens, ref = _pool(seed)
        par = torch.randint(-1, 6, (6,), generator=torch.Generator().manual_seed(seed + 50)).tolist()
        new, nlen, nref, missing, copies = O.reorder(table, lens, ref, par, 16)
        assert missing == 0 and nref == _count(new, len(ref))
        dst = [d for _, d in copies]
        assert len(set(dst)) == len(dst) and not set(dst) & {s for s, _ in copies}
        for r, p in enumerate(par):
            if p >= 0 and nlen[r] % 16:
                assert nref[new[r][nlen[r] // 16]] == 1            # a begun page has one holder
        # keys found through either table agree once the copies are made
        moved = dict((d, s) for s, d in copies)
        for r, p in enumerate(par):
            for b in range(-(-nlen[r] // 16)):
                assert moved.get(new[r][b], new[r][b]) == table[p][b]
        c, cref, n, moves = O.compact(new, nref)
        assert cref == _count(c, len(ref)) and all(x > 0 for x in cref[:n]) and not any(cref[n:])


def test_reserve_takes_the_lowest_free_pages():
    table, ref, missing = O.reserve([[2, -1], [-1, -1]], [0, 0, 1, 0], [20, 40], 16)
    assert (table, ref, missing) == ([[2, 0], [1, 3]], [1, 1, 1, 1], 0)
    assert O.reserve([[2, -1], [-1, -1]], [0, 1, 1], [20, 40], 16) == ([[2, 0], [-1, -1]], [1, 1, 1], 2)


def test_refusals(monkeypatch):
    monkeypatch.setattr(cache_pages, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "lib", lambda: pytest.fail("reached the library"))
    i32 = dict(dtype=torch.int32)
    st = cache_pages.PageTable(torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(5, **i32))
    new = torch.zeros(2, **i32)
    with pytest.raises(UnsupportedShape, match="int32"):
        cache_pages.pages_reserve(st._replace(ref=st.ref.long()), new, page_size=16)
    with pytest.raises(ValueError, match="expected"):
        cache_pages.pages_reserve(st._replace(seq_lens=torch.zeros(3, **i32)), new, page_size=16)
    with pytest.raises(ValueError, match="values for 2 rows"):
        cache_pages.pages_reserve(st, new[:1], page_size=16)
    with pytest.raises(ValueError, match="empty"):
        cache_pages.pages_compact(st._replace(ref=torch.zeros(0, **i32)), [])
    with pytest.raises(ValueError, match="overlaps"):
        cache_pages.pages_reserve(st, new, page_size=16, out=st)
    with pytest.raises(ValueError, match="overlaps"):
        cache_pages.pages_compact(st, [], out=cache_pages.PageTable(torch.zeros(2, 3, **i32), st.seq_lens,
                                                                    torch.zeros(5, **i32)))
    with pytest.raises(ValueError, match="shapes differ"):
        cache_pages.pages_compact(st, [], out=cache_pages.PageTable(torch.zeros(2, 4, **i32), new.clone(),
                                                                    torch.zeros(5, **i32)))
    with pytest.raises(ValueError, match="5 pages"):
        cache_pages.pages_compact(st, [torch.zeros(4, 8)])
    with pytest.raises(UnsupportedShape, match="contiguous"):
        cache_pages.pages_compact(st, [torch.zeros(5, 8, 8).transpose(1, 2)])
    with pytest.raises(UnsupportedShape, match="apart"):
        cache_pages.pages_compact(st, [torch.zeros(1, 8).expand(5, 8)])


def test_host_tensors_are_refused():
    i32 = dict(dtype=torch.int32)
    st = cache_pages.PageTable(torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(5, **i32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache_pages.pages_compact(st, [])


def test_abi_refuses_before_any_launch():
    L = _lib.lib()
    a = _lib.PagesArgs()
    for fn in (L.srswa_pages_reserve, L.srswa_pages_reorder, L.srswa_pages_compact):
        assert fn(ctypes.byref(a), None, 0, None) == _lib.SRSWA_INVALID
    for i, n in enumerate(("block_table", "seq_lens", "ref", "rows", "block_table_out", "seq_lens_out", "ref_out",
                           "count")):
        setattr(a, n, 0x100000 * (i + 1))
    a.R, a.W, a.num_pages, a.page_size, a.bt_sr, a.bto_sr = 2, 3, 100, 16, 3, 3
    need = L.srswa_pages_workspace(ctypes.byref(a))
    assert need > 0
    for fn in (L.srswa_pages_reserve, L.srswa_pages_reorder, L.srswa_pages_compact):
        assert fn(ctypes.byref(a), ctypes.c_void_p(0x9000000), need - 1, None) == _lib.SRSWA_WORKSPACE
    a.R = 0
    assert L.srswa_pages_reorder(ctypes.byref(a), ctypes.c_void_p(0x9000000), need, None) == _lib.SRSWA_INVALID
