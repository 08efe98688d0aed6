"""The page pool on the GPU against the oracle's plain loops: state and page data
equal, nothing but the named pages written, the input state left as it was."""

import pytest
import torch

from oracle import cache8_oracle as O

pytestmark = pytest.mark.gpu


def _pool(seed, R, W, N, page, share=0):
    g = torch.Generator().manual_seed(seed)
    lens, left = [], N
    for r in range(R):
        n = int(torch.randint(0, min(W, max(left, 0)) * page + 1, (1,), generator=g)) if left > 0 else 0
        lens.append(n)
        left -= -(-n // page)
    perm, o, table = torch.randperm(N, generator=g).tolist(), 0, []
    for n in lens:
        m = -(-n // page)
        table.append(perm[o:o + m] + [-1] * (W - m))
        o += m
    for _ in range(share):                                # a full first page held twice
        a, b = torch.randint(0, R, (2,), generator=g).tolist()
        if lens[a] >= page and lens[b] >= page:
            table[b][0] = table[a][0]
    ref = [0] * N
    for row in table:
        for x in row:
            if x >= 0:
                ref[x] += 1
    return table, lens, ref, g


def _dev(dev, table, lens, ref):
    from srswa.cache_pages import PageTable
    return PageTable(*(torch.tensor(x, dtype=torch.int32).to(dev) for x in (table, lens, ref)))


def _caches(N, g, dev):
    """Page data of several kinds: 16-byte pages, rows of floats, odd bytes, pages of a wider allocation."""
    c = [torch.randint(0, 250, (N, 16, 2, 64), generator=g).to(torch.uint8), torch.randn(N, 3, generator=g),
         torch.randint(0, 250, (N, 7), generator=g).to(torch.uint8), torch.randn(2, N, 24, generator=g)[1],
         torch.randn(N, 2, 40, generator=g).to(torch.bfloat16)[:, 1], torch.zeros(N, 0)]
    d = [t.to(dev) for t in c]
    wide = torch.randn(N, 2, 40, generator=g)
    return c + [wide[:, 0].clone()], d + [wide.to(dev)[:, 0]]


def _equal(st, table, lens, ref):
    assert st.block_table.tolist() == table
    assert st.seq_lens.tolist() == lens
    assert st.ref.tolist() == ref


SIZES = [(1, 1, 1, 16), (3, 5, 16, 16), (6, 7, 60, 48), (40, 33, 900, 16), (300, 20, 5000, 64), (5, 700, 2048, 32),
         (4, 300, 4096, 16), (9, 40, 70, 16)]


@pytest.mark.parametrize("R,W,N,page", SIZES)
def test_reserve(dev, R, W, N, page):
    from srswa import cache_pages
    for seed in range(3):
        table, lens, ref, g = _pool(seed, R, W, N, page, share=2)
        grow = torch.randint(0, 4 * page, (R,), generator=g).tolist()
        new = [min(n + x, W * page + 5) if i % 3 else n for i, (n, x) in enumerate(zip(lens, grow))]
        if seed == 2:
            new = [W * page] * R                          # more than the pool may hold
        state = _dev(dev, table, lens, ref)
        st, missing = cache_pages.pages_reserve(state, torch.tensor(new).to(dev), page_size=page)
        t, rf, m = O.reserve(table, ref, new, page)
        _equal(st, t, new, rf)
        assert missing.tolist() == [m]
        _equal(state, table, lens, ref)


@pytest.mark.parametrize("R,W,N,page", SIZES)
def test_reorder(dev, R, W, N, page):
    from srswa import cache_pages
    for seed in range(4):
        table, lens, ref, g = _pool(seed + 20, R, W, N, page, share=2)
        par = torch.randint(-1, R + 1, (R,), generator=g).tolist()
        if seed == 1:
            par = list(range(R))                          # nothing moves
        if seed == 2:
            par = [R // 2] * R                            # one row for all
        if seed == 3:
            par = [-1] * R                                # every row is freed
        c, d = _caches(N, g, dev)
        state = _dev(dev, table, lens, ref)
        st, missing = cache_pages.pages_reorder(state, torch.tensor(par).to(dev), d, page_size=page)
        t, ln, rf, m, copies = O.reorder(table, lens, ref, par, page)
        _equal(st, t, ln, rf)
        assert missing.tolist() == [m]
        for x, y in zip(c, d):
            for s, e in copies:
                x[e] = x[s]
            assert torch.equal(y.cpu(), x)
        _equal(state, table, lens, ref)


@pytest.mark.parametrize("R,W,N,page", SIZES)
def test_compact(dev, R, W, N, page):
    from srswa import cache_pages
    for seed in range(3):
        table, lens, ref, g = _pool(seed + 40, R, W, N, page, share=3)
        if seed == 2:                                     # a full pool: nothing moves
            ref = [max(x, 1) for x in ref]
        c, d = _caches(N, g, dev)
        state = _dev(dev, table, lens, ref)
        st, live = cache_pages.pages_compact(state, d)
        t, rf, n, moves = O.compact(table, ref)
        _equal(st, t, lens, rf)
        assert live.tolist() == [n]
        for x, y in zip(c, d):
            for s, e in moves:
                x[e] = x[s]
            assert torch.equal(y.cpu(), x)
        _equal(state, table, lens, ref)


# rows and entries past a workgroup's width, pages past its tiles, tables past the one-workgroup plan
@pytest.mark.parametrize("R,W,N,page", [(1500, 3, 2500, 16), (300, 400, 9000, 16), (5, 8000, 36000, 16),
                                        (3, 300, 600000, 32)])
def test_larger_pools(dev, R, W, N, page):
    from srswa import cache_pages
    table, lens, ref, g = _pool(90, R, W, N, page, share=5)
    data = torch.randn(N, 3, generator=g)
    d = [data.to(dev)]
    state = _dev(dev, table, lens, ref)
    new = [min(n + 3 * page * (i % 4), W * page) for i, n in enumerate(lens)]
    st, missing = cache_pages.pages_reserve(state, torch.tensor(new).to(dev), page_size=page)
    table, ref, m = O.reserve(table, ref, new, page)
    _equal(st, table, new, ref)
    assert missing.tolist() == [m]
    par = torch.randint(-1, R, (R,), generator=g).tolist()
    st, missing = cache_pages.pages_reorder(st, torch.tensor(par).to(dev), d, page_size=page)
    table, lens, ref, m, copies = O.reorder(table, new, ref, par, page)
    _equal(st, table, lens, ref)
    assert missing.tolist() == [m]
    for s, e in copies:
        data[e] = data[s]
    st, live = cache_pages.pages_compact(st, d)
    table, ref, n, moves = O.compact(table, ref)
    _equal(st, table, lens, ref)
    assert live.tolist() == [n]
    for s, e in moves:
        data[e] = data[s]
    assert torch.equal(d[0].cpu(), data)


def test_pages_on_other_streams_at_once(dev):
    """The same state reordered on two streams, each with its own caches."""
    from srswa import cache_pages
    table, lens, ref, g = _pool(95, 40, 20, 700, 16)
    par = torch.randint(-1, 40, (40,), generator=g)
    t, ln, rf, m, copies = O.reorder(table, lens, ref, par.tolist(), 16)
    state, par = _dev(dev, table, lens, ref), par.to(torch.int32).to(dev)
    data = torch.randn(700, 2048, generator=g)
    d = [data.to(dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(cache_pages.pages_reorder(state, par, [d[i]], page_size=16))
    torch.cuda.synchronize()
    for s, e in copies:
        data[e] = data[s]
    for (st, missing), x in zip(got, d):
        _equal(st, t, ln, rf)
        assert missing.tolist() == [m] and torch.equal(x.cpu(), data)


def test_out_and_many_caches(dev):
    """More caches than one copy launch takes, and states written in turn."""
    from srswa import cache_pages
    table, lens, ref, g = _pool(70, 8, 9, 100, 16)
    state = _dev(dev, table, lens, ref)
    other = cache_pages.PageTable(*(torch.full_like(t, 77) for t in state))
    c = [torch.randn(100, 4, generator=g) for _ in range(150)]
    d = [t.to(dev) for t in c]
    par = [3, 3, 3, 0, 0, 7, -1, 7]
    st, _ = cache_pages.pages_reorder(state, torch.tensor(par).to(dev), d, page_size=16, out=other)
    assert all(a is b for a, b in zip(st, other))
    t, ln, rf, _, copies = O.reorder(table, lens, ref, par, 16)
    _equal(st, t, ln, rf)
    for x, y in zip(c, d):
        for s, e in copies:
            x[e] = x[s]
        assert torch.equal(y.cpu(), x)


def test_captured_calls_replay(dev):
    from srswa import cache_pages
    table, lens, ref, g = _pool(71, 6, 9, 80, 16)
    a = _dev(dev, table, lens, ref)
    b, c = (cache_pages.PageTable(*(torch.zeros_like(t) for t in a)) for _ in range(2))
    data = torch.randn(80, 32, generator=g).to(dev)
    new, par = torch.zeros(6, dtype=torch.int32, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)

    def step(x, y, z, d):
        _, m = cache_pages.pages_reserve(x, new, page_size=16, out=y)
        _, k = cache_pages.pages_reorder(y, par, [d], page_size=16, out=z)
        _, n = cache_pages.pages_compact(z, [d], out=y)
        return m, k, n

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, b, c, data.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        counts = step(a, b, c, data)
    for i in range(4):
        start = torch.randn(80, 32, generator=g)
        data.copy_(start)
        grown = [n + 5 * i for n in lens]
        new.copy_(torch.tensor(grown))
        p = torch.randint(-1, 6, (6,), generator=g).tolist()
        par.copy_(torch.tensor(p))
        graph.replay()
        torch.cuda.synchronize()
        t, rf, m = O.reserve(table, ref, grown, 16)
        t, ln, rf, k, copies = O.reorder(t, grown, rf, p, 16)
        for s, e in copies:
            start[e] = start[s]
        t, rf, n, moves = O.compact(t, rf)
        for s, e in moves:
            start[e] = start[s]
        _equal(b, t, ln, rf)
        assert [int(x) for x in counts] == [m, k, n] and torch.equal(data.cpu(), start), i
        torch.randn(1 << 16, device=dev).sum().item()
