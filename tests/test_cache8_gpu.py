"""The scaled 8-bit cache on the GPU against the 64-bit oracle: append (bytes and
scales equal, nothing else written), decode, selected blocks and prefill (within
the oracle's rounding bound), and a run of them together with the page pool."""

import math

import pytest
import torch

from oracle import cache8_oracle as O

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


def _table(g, lens, page, W, spare=2):
    """Pages dealt at random: (table lists, pages in all)."""
    n = sum(-(-x // page) for x in lens) + spare
    perm, o, table = torch.randperm(n, generator=g).tolist(), 0, []
    for x in lens:
        m = -(-x // page)
        table.append(perm[o:o + m] + [-1] * (W - m))
        o += m
    return table, n


def _cache(g, n, page, H, D, dt, pow2=True):
    """Random bytes (every format value but NaN) and scales."""
    b = torch.randint(-127, 127, (n, page, H, D), generator=g).to(torch.int8)
    e = torch.randint(-9, -4, (n, H), generator=g).float()
    if dt == E4M3:
        b = torch.randn(n, page, H, D, generator=g).mul(60).to(E4M3).view(torch.int8)
    s = torch.exp2(e)
    return b.view(dt) if dt == E4M3 else b, s if pow2 else s * (1 + torch.rand(n, H, generator=g))


def _same_bytes(got, ref, what):
    got = got.cpu()
    if got.dtype == E4M3:
        a, b = got.float(), ref.float()
        ok = (a == b) | (torch.isnan(a) & torch.isnan(b))
    else:
        ok = got == ref
    assert ok.all(), (what, int((~ok).sum()), ok.logical_not().nonzero()[:4].tolist())


# -------------------------------------------------------------------- append
APPEND = {
    # one token each: into an empty page, behind others, at a page's last row
    "step": dict(page=16, H=3, D=64, start=[0, 5, 15, 31, 40], runs=[1] * 5, W=4),
    "step_wide_page": dict(page=128, H=2, D=128, start=[0, 100, 127, 128], runs=[1] * 4, W=3),
    # runs over several pages, odd starts, an empty run in the middle, a run past the table
    "runs": dict(page=16, H=2, D=128, start=[3, 0, 17, 60], runs=[40, 16, 0, 9], W=4, cu=True),
    "runs_48": dict(page=48, H=1, D=64, start=[47, 0, 13], runs=[1, 97, 100], W=3, cu=True),
    "one_row": dict(page=64, H=1, D=128, start=[63], runs=[1], W=1),
    "wide": dict(page=1024, H=1, D=64, start=[1000, 3], runs=[30, 700], W=2, cu=True),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kv", [torch.int8, E4M3])
@pytest.mark.parametrize("name", list(APPEND))
def test_append_matches_oracle(dev, name, kv, dtype):
    from srswa import cache8
    c = APPEND[name]
    g = torch.Generator().manual_seed(list(APPEND).index(name) + 10)
    cap = c["W"] * c["page"]
    table, n = _table(g, [min(a + b, cap) for a, b in zip(c["start"], c["runs"])], c["page"], c["W"])
    kc, ks = _cache(g, n, c["page"], c["H"], c["D"], kv)
    vc, vs = _cache(g, n, c["page"], c["H"], c["D"], kv)
    total = sum(c["runs"])
    k, v = (torch.randn(total, c["H"], c["D"], generator=g).mul(m).to(dtype) for m in (3.0, 0.01))
    k[total // 2] *= 50                                   # one loud token: its pages' scales grow
    ref = [O.append(x, y, s, table, c["start"], c["runs"]) for x, y, s in ((k, kc, ks), (v, vc, vs))]
    d = [t.to(dev) for t in (k, v, kc, vc, ks, vs)]
    kw = {}
    if c.get("cu"):
        kw = dict(cu_seqlens=torch.tensor([0] + c["runs"]).cumsum(0).to(torch.int32).to(dev), max_new_len=max(c["runs"]))
    cache8.cache8_append(*d, torch.tensor(table, dtype=torch.int32).to(dev),
                         torch.tensor(c["start"], dtype=torch.int32).to(dev), **kw)
    for got, want, what in ((d[2], ref[0][0], "k"), (d[3], ref[1][0], "v")):
        _same_bytes(got, want, what)
    assert torch.equal(d[4].cpu(), ref[0][1]) and torch.equal(d[5].cpu(), ref[1][1])


@pytest.mark.parametrize("kv", [torch.int8, E4M3])
def test_append_values_that_do_not_fit(dev, kv):
    """NaN, infinities, zeros, subnormals and the type's largest value; a scale of
    the caller's own that is no power of two; missing and impossible pages."""
    from srswa import cache8
    for dtype in (BF, HF):
        g = torch.Generator().manual_seed(3)
        page, H, D = 16, 4, 64
        k = torch.randn(7, H, D, generator=g).to(dtype)
        k[0, 0, 3], k[0, 0, 4], k[0, 0, 5] = math.nan, math.inf, -math.inf
        k[1] = 0.0                                        # a page of zeros
        k[2, 1] = torch.finfo(dtype).smallest_normal / 4
        k[3, 2] = torch.finfo(dtype).max
        k[4] = math.nan                                   # nothing finite
        table = [[0], [1], [2], [3], [4], [-1], [9]]      # rows 5 and 6 have no page
        kc, ks = _cache(g, 6, page, H, D, kv)
        vc, vs = _cache(g, 6, page, H, D, kv)
        ks[:, 3] = 0.3
        start = [2, 0, 0, 1, 0, 0, 0]
        ref = O.append(k, kc, ks, table, start, [1] * 7)
        d = [t.to(dev) for t in (k, k, kc, vc, ks, vs)]
        cache8.cache8_append(*d, torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(start).to(dev))
        _same_bytes(d[2], ref[0], "k")
        assert torch.equal(d[4].cpu(), ref[1])


def test_append_reads_strides_and_writes_a_slice_of_a_cache(dev):
    from srswa import cache8
    g = torch.Generator().manual_seed(8)
    page, H, D = 32, 3, 64
    qkv = torch.randn(40, 3 * H, 2 * D, generator=g).to(BF)
    k, v = qkv[:, H:2 * H, :D], qkv[:, 2 * H:, D:]
    both = torch.randint(-100, 100, (5, page, 2 * H, D), generator=g).to(torch.int8)
    sc = torch.rand(5, 2 * H, generator=g) + 0.5
    table = [[4, 1, -1], [0, -1, -1]]
    ref = [O.append(x, both[:, :, s], sc[:, s], table, [5, 0], [35, 5])
           for x, s in ((k, slice(0, H)), (v, slice(H, 2 * H)))]
    both_d, sc_d, qkv_d = both.to(dev), sc.to(dev), qkv.to(dev)
    cache8.cache8_append(qkv_d[:, H:2 * H, :D], qkv_d[:, 2 * H:, D:], both_d[:, :, :H], both_d[:, :, H:], sc_d[:, :H],
                         sc_d[:, H:], torch.tensor(table).to(dev).t().contiguous().t(), torch.tensor([5, 0]).to(dev),
                         cu_seqlens=torch.tensor([0, 35, 40]).to(dev), max_new_len=35)
    assert torch.equal(both_d.cpu(), torch.cat([ref[0][0], ref[1][0]], 2))
    assert torch.equal(sc_d.cpu(), torch.cat([ref[0][1], ref[1][1]], 1))


def test_append_in_any_split_gives_one_scale(dev):
    """One call or token by token: the same scales; the same e4m3 bytes too where
    no value falls below the normal range."""
    from srswa import cache8
    g = torch.Generator().manual_seed(9)
    page, H, D, n = 32, 2, 128, 70
    k = (torch.rand(n, H, D, generator=g) + 0.25).to(BF)
    bt = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    state = []
    for step in (n, 1, 7):
        c = [torch.zeros(3, page, H, D, device=dev).to(E4M3) for _ in range(2)] + [torch.ones(3, H, device=dev)] * 1 + \
            [torch.ones(3, H, device=dev)]
        for s in range(0, n, step):
            x = k[s:s + step].to(dev)
            cache8.cache8_append(x, -x, *c, bt, torch.tensor([s], device=dev))
        state.append([t.float().cpu() for t in c])
    for other in state[1:]:
        assert all(torch.equal(a, b) for a, b in zip(state[0], other))


# -------------------------------------------------------------------- attend
def _check(got, lse, ref, what):
    o, l, tol = ref
    err = (got.cpu().double() - o).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, (err / tol.clamp(min=1e-300)).max().item(), (err > tol).sum().item())
    if lse is not None:
        lse = lse.cpu().double()
        none = torch.isinf(l)
        assert torch.equal(torch.isinf(lse), none), what
        assert ((lse - l).abs()[~none] <= 1e-4 * (1 + l[~none].abs())).all(), what


def _state(c, g, lens, spoil=True):
    table, n = _table(g, lens, c["page"], c["W"])
    kc, ks = _cache(g, n, c["page"], c["HKV"], c["D"], c["kv"], pow2=False)
    vc, vs = _cache(g, n, c["page"], c["HKV"], c["D"], c["kv"], pow2=False)
    if spoil:                                             # what no key holds: NaN bytes, NaN scales
        used = {x for row in table for x in row if x >= 0}
        for p in set(range(n)) - used:
            ks[p] = vs[p] = math.nan
            if c["kv"] == E4M3:
                kc.view(torch.int8)[p] = vc.view(torch.int8)[p] = 127
        for row, x in zip(table, lens):
            if x % c["page"] and c["kv"] == E4M3:
                p = row[x // c["page"]]
                kc.view(torch.int8)[p, x % c["page"]:] = vc.view(torch.int8)[p, x % c["page"]:] = 127
    return table, kc, vc, ks, vs


DECODE = {
    "short": dict(page=16, HQ=2, HKV=2, D=64, lens=[1, 15, 16, 17, 33], W=3, dql=1),
    "mha": dict(page=64, HQ=3, HKV=3, D=128, lens=[1, 64, 200, 129], W=4, dql=1),
    "gqa16": dict(page=32, HQ=16, HKV=1, D=128, lens=[70, 3], W=3, dql=1),
    "gqa_rows": dict(page=16, HQ=12, HKV=2, D=64, lens=[90, 31, 6], W=6, dql=5),       # 30 rows: two tiles
    "group_of_24": dict(page=32, HQ=24, HKV=1, D=64, lens=[50], W=2, dql=2),
    "before_the_first": dict(page=16, HQ=2, HKV=1, D=64, lens=[2, 0, 5], W=1, dql=4),   # rows without a key
    "window": dict(page=32, HQ=4, HKV=2, D=128, lens=[200, 5, 77, 33], W=7, dql=2, window=33),
    "window1": dict(page=16, HQ=2, HKV=2, D=64, lens=[40, 1], W=3, dql=3, window=1, sinks=1),
    "sinks": dict(page=48, HQ=4, HKV=4, D=64, lens=[300, 47, 49, 100], W=7, dql=1, window=20, sinks=37),
    "sinks_meet_window": dict(page=16, HQ=2, HKV=1, D=128, lens=[60, 64, 100], W=7, dql=3, window=40, sinks=25),
    "sinks_beyond": dict(page=16, HQ=2, HKV=1, D=128, lens=[60, 20], W=7, dql=1, window=4, sinks=5000),
    "window_beyond": dict(page=16, HQ=2, HKV=1, D=128, lens=[60, 20], W=7, dql=1, window=1 << 40),
    "chunks": dict(page=64, HQ=2, HKV=2, D=128, lens=[2500, 1, 700, 1300], W=40, dql=1),
    "chunks_rows": dict(page=16, HQ=6, HKV=2, D=64, lens=[1700, 900], W=110, dql=2),
    "page1024": dict(page=1024, HQ=1, HKV=1, D=64, lens=[1500], W=2, dql=1, window=300, sinks=3),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kv", [torch.int8, E4M3])
@pytest.mark.parametrize("name", list(DECODE))
def test_decode_and_prefill_match_oracle(dev, name, kv, dtype):
    from srswa import cache8
    c = dict(DECODE[name], kv=kv)
    g = torch.Generator().manual_seed(list(DECODE).index(name) + 30)
    lens, R, dql = c["lens"], len(c["lens"]), c["dql"]
    table, kc, vc, ks, vs = _state(c, g, lens)
    q = torch.randn(R * dql, c["HQ"], c["D"], generator=g).to(dtype)
    cu = [dql * r for r in range(R + 1)]
    win, sinks, scale = c.get("window"), c.get("sinks", 0), c["D"] ** -0.5
    ref = O.attend(q, kc, vc, ks, vs, table, cu, lens, scale, window=win, sinks=sinks)
    d = [t.to(dev) for t in (q, kc, vc, ks, vs)]
    bt, sl = torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(lens).to(dev)
    o, lse = cache8.cache8_decode(*d, bt, sl, scale=scale, decode_query_len=dql, window=win, sinks=sinks,
                                  return_lse=True)
    _check(o, lse, ref, "decode")
    o, lse = cache8.cache8_prefill(*d, bt, torch.tensor(cu).to(dev), sl, dql, scale=scale, window=win, sinks=sinks,
                                   return_lse=True)
    _check(o, lse, ref, "prefill")


PREFILL = {
    "one_each": dict(page=16, HQ=2, HKV=2, D=64, q=[1, 1], ctx=[0, 20], W=2),
    "ragged": dict(page=64, HQ=4, HKV=2, D=128, q=[70, 0, 1, 33, 130], ctx=[0, 10, 200, 63, 5], W=4),
    "first_rows_cut": dict(page=16, HQ=2, HKV=1, D=64, q=[40], ctx=[-9], W=3),          # 9 rows before key 0
    "window": dict(page=32, HQ=2, HKV=2, D=128, q=[150, 20], ctx=[100, 300], W=10, window=50, sinks=40),
    "window_small": dict(page=16, HQ=2, HKV=2, D=64, q=[130], ctx=[70], W=13, window=7, sinks=0),
    "sinks_only_far": dict(page=48, HQ=3, HKV=1, D=64, q=[65], ctx=[500], W=12, window=3, sinks=5),
    "wide_group": dict(page=32, HQ=16, HKV=2, D=64, q=[37, 9], ctx=[11, 0], W=2),
    "long_page": dict(page=1024, HQ=1, HKV=1, D=128, q=[100], ctx=[1000], W=2),
    "page48": dict(page=48, HQ=2, HKV=2, D=128, q=[129, 64], ctx=[31, 0], W=4),
    # few rows, long keys: the keys split over parts, as many as a request has chunks for
    "parts": dict(page=64, HQ=1, HKV=1, D=128, q=[40, 35], ctx=[2100, 300], W=34),
    "parts_window": dict(page=16, HQ=2, HKV=1, D=64, q=[33], ctx=[2500], W=160, window=1200, sinks=300),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kv", [torch.int8, E4M3])
@pytest.mark.parametrize("name", list(PREFILL))
def test_prefill_matches_oracle(dev, name, kv, dtype):
    from srswa import cache8
    c = dict(PREFILL[name], kv=kv)
    g = torch.Generator().manual_seed(list(PREFILL).index(name) + 60)
    lens = [a + b for a, b in zip(c["q"], c["ctx"])]
    table, kc, vc, ks, vs = _state(c, g, lens)
    cu = torch.tensor([0] + c["q"]).cumsum(0).tolist()
    total = cu[-1]
    q = torch.randn(total + 3, c["HQ"], c["D"], generator=g).to(dtype)
    win, sinks, scale = c.get("window"), c.get("sinks", 0), c["D"] ** -0.5
    o, l, tol = O.attend(q, kc, vc, ks, vs, table, cu, lens, scale, window=win, sinks=sinks)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    got, lse = cache8.cache8_prefill(*(t.to(dev) for t in (q, kc, vc, ks, vs)),
                                     torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(cu).to(dev),
                                     torch.tensor(lens).to(dev), max(c["q"]), scale=scale, window=win, sinks=sinks,
                                     out=out, return_lse=True)
    assert got is out and (out[total:] == 7.0).all()       # rows behind the last request
    _check(got[:total], lse[:total], (o[:total], l[:total], tol[:total]), name)


@pytest.mark.parametrize("kv", [torch.int8, E4M3])
def test_missing_pages_hide_their_keys(dev, kv):
    from srswa import cache8
    c = dict(page=16, HQ=2, HKV=1, D=64, W=6, kv=kv)
    g = torch.Generator().manual_seed(4)
    lens = [80, 90, 20]
    table, kc, vc, ks, vs = _state(c, g, lens)
    table[0][2], table[0][4], table[1][0], table[1][5], table[2][0], table[2][1] = -1, 1000, -5, 1 << 30, -1, -1
    q = torch.randn(3, 2, 64, generator=g).to(BF)
    over = [200, 90, 20]                                  # more keys than the table has pages for
    ref = O.attend(q, kc, vc, ks, vs, table, [0, 1, 2, 3], over, 0.2)
    assert math.isinf(ref[1][2, 0])
    args = [t.to(dev) for t in (q, kc, vc, ks, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev)]
    o, lse = cache8.cache8_decode(*args, torch.tensor(over).to(dev), scale=0.2, return_lse=True)
    _check(o, lse, ref, "decode")
    o, lse = cache8.cache8_prefill(*args, torch.arange(4).to(dev), torch.tensor(over).to(dev), 1, scale=0.2,
                                   return_lse=True)
    _check(o, lse, ref, "prefill")


def test_large_logits_and_scales(dev):
    """Logits of some thousands (one key takes all the weight) and scales far from 1."""
    from srswa import cache8
    for kv in (torch.int8, E4M3):
        c = dict(page=16, HQ=2, HKV=2, D=64, W=9, kv=kv)
        g = torch.Generator().manual_seed(14)
        lens = [130, 77]
        table, kc, vc, ks, vs = _state(c, g, lens)
        vs *= 2.0 ** -30
        q = (torch.randn(2, 2, 64, generator=g) * 40).to(BF)
        ref = O.attend(q, kc, vc, ks * 8, vs, table, [0, 1, 2], lens, 0.125)
        args = [t.to(dev) for t in (q, kc, vc, ks * 8, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev)]
        o, lse = cache8.cache8_decode(*args, torch.tensor(lens).to(dev), scale=0.125, return_lse=True)
        _check(o, lse, ref, "decode")


SELECTED = {
    "plain": dict(page=16, HQ=2, HKV=2, D=64, lens=[200, 17, 90], W=13, dql=1, K=4, LB=2),
    "rows": dict(page=32, HQ=8, HKV=2, D=128, lens=[250, 70], W=8, dql=2, K=3, LB=1, bias=True),
    "no_window": dict(page=16, HQ=2, HKV=1, D=64, lens=[100, 30], W=7, dql=2, K=5, LB=0, bias=True),
    "one_slot": dict(page=64, HQ=2, HKV=2, D=128, lens=[300], W=5, dql=1, K=1, LB=1),
    "no_slot": dict(page=16, HQ=2, HKV=2, D=64, lens=[100], W=7, dql=1, K=0, LB=3),
    "many_slots": dict(page=16, HQ=2, HKV=1, D=64, lens=[3000, 500], W=188, dql=1, K=200, LB=4, bias=True),
    "heads_20": dict(page=32, HQ=20, HKV=1, D=64, lens=[150], W=5, dql=2, K=3, LB=1, bias=True),
}


@pytest.mark.parametrize("kv", [torch.int8, E4M3])
@pytest.mark.parametrize("name", list(SELECTED))
def test_selected_blocks_match_oracle(dev, name, kv):
    from srswa.unlimited_dash_ops import dash_sparse_attn_decode
    c = dict(SELECTED[name], kv=kv)
    g = torch.Generator().manual_seed(list(SELECTED).index(name) + 80)
    lens, R, dql, K = c["lens"], len(c["lens"]), c["dql"], c["K"]
    table, kc, vc, ks, vs = _state(c, g, lens)
    ids = torch.randint(-1, c["W"] + 1, (c["HKV"], R * dql, K), generator=g).to(torch.int32)
    if K > 2:
        ids[:, 0, 2] = ids[:, 0, 0]                       # a repeated id
    bias = torch.randn(ids.shape, generator=g) if c.get("bias") else None
    if bias is not None:
        bias[0, 0, 1], bias[0, 0, 0] = -math.inf, torch.finfo(torch.float32).min
    q = torch.randn(R * dql, c["HQ"], c["D"], generator=g).to(BF)
    ref = O.attend(q, kc, vc, ks, vs, table, [dql * r for r in range(R + 1)], lens, 0.125,
                   window=c["LB"] * c["page"], topk=ids, bias=bias)
    ref = (torch.nan_to_num(ref[0]), ref[1], torch.nan_to_num(ref[2]))
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    b = None if bias is None else bias.to(dev)
    dash_sparse_attn_decode(q.to(dev), kc.to(dev), vc.to(dev), ids.to(dev), b,
                            torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(lens).to(dev), c["HKV"], 0.125,
                            out, dql, local_blocks=c["LB"], sparse_block_size=c["page"], k_scale=ks.to(dev),
                            v_scale=vs.to(dev))
    _check(out, None, ref, name)


def test_selected_takes_head_expanded_ids(dev):
    from srswa.unlimited_dash_ops import dash_sparse_attn_decode
    c = dict(page=16, HKV=3, D=64, W=13, kv=E4M3)
    g = torch.Generator().manual_seed(2)
    table, kc, vc, ks, vs = _state(c, g, [200, 90])
    ids = torch.randint(-1, 8, (1, 2, 4), generator=g).to(torch.int32).expand(3, 2, 4)
    bias = torch.randn(1, 2, 4, generator=g).expand(3, 2, 4)
    q = torch.randn(2, 3, 64, generator=g).to(HF).to(dev)
    outs = []
    for i, b in ((ids.to(dev), bias.to(dev)), (ids[:1].to(dev).expand(3, 2, 4), bias[:1].to(dev).expand(3, 2, 4))):
        outs.append(torch.empty_like(q))
        dash_sparse_attn_decode(q, kc.to(dev), vc.to(dev), i, b, torch.tensor(table, dtype=torch.int32).to(dev),
                                torch.tensor([200, 90]).to(dev), 3, 0.125, outs[-1], 1, local_blocks=1,
                                sparse_block_size=16, k_scale=ks.to(dev), v_scale=vs.to(dev))
    assert torch.equal(*outs)


def test_strided_queries_outputs_and_caches(dev):
    """Views: heads of a fused projection, K and V as halves of one page, layers of one allocation."""
    from srswa import cache8
    g = torch.Generator().manual_seed(21)
    lens, H, D, page = [70, 33], 2, 64, 16
    table, n = _table(g, lens, page, 5)
    kv = torch.randint(-100, 100, (n, 2, page, 2 * H, D), generator=g).to(torch.int8)
    sc = torch.rand(n, 2, 2 * H, generator=g) * 0.02
    qf = torch.randn(4, 6 * H, D, generator=g).to(BF)
    q = qf[:, 1:H + 1]
    kc, vc, ks, vs = kv[:, 0, :, H:], kv[:, 1, :, H:], sc[:, 0, :H], sc[:, 1, H:]
    ref = O.attend(q, kc, vc, ks, vs, table, [0, 2, 4], lens, 0.125)
    kvd, scd, qd = kv.to(dev), sc.to(dev), qf.to(dev)
    wide = torch.zeros(4, 3 * H, D, dtype=BF, device=dev)
    bt = torch.tensor(table, dtype=torch.int32).to(dev)
    args = (qd[:, 1:H + 1], kvd[:, 0, :, H:], kvd[:, 1, :, H:], scd[:, 0, :H], scd[:, 1, H:], bt)
    cache8.cache8_decode(*args, torch.tensor(lens).to(dev), scale=0.125, decode_query_len=2, out=wide[:, H:2 * H])
    _check(wide[:, H:2 * H], None, ref, "decode")
    assert not wide[:, :H].any() and not wide[:, 2 * H:].any()
    cache8.cache8_prefill(*args, torch.tensor([0, 2, 4]).to(dev), torch.tensor(lens).to(dev), 2, scale=0.125,
                          out=wide[:, 2 * H:])
    _check(wide[:, 2 * H:], None, ref, "prefill")


def test_ctypes_path_gives_the_same(dev, monkeypatch):
    """The native host path and the ctypes one (which also converts: 64-bit
    tables, unordered strides) launch the same work."""
    from srswa import _lib, cache8, cache_pages
    assert _lib.host is not None
    g = torch.Generator().manual_seed(61)
    page, H, D, lens = 16, 2, 64, [70, 33]
    table, n = _table(g, lens, page, 5, spare=6)
    kc, ks = _cache(g, n, page, H, D, E4M3)
    vc, vs = _cache(g, n, page, H, D, E4M3)
    q = torch.randn(4, 4, D, generator=g).to(BF).to(dev)
    x = torch.randn(4, H, D, generator=g).to(BF).to(dev)
    bt, sl = torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(lens, dtype=torch.int32).to(dev)
    ids = torch.randint(-1, 4, (H, 4, 3), generator=g).to(torch.int32).to(dev)
    ref = torch.zeros(n, dtype=torch.int32, device=dev)
    ref[bt[bt >= 0].long()] = 1
    got = []
    for native in (True, False):
        wide = not native                                # what only the ctypes path takes
        if not native:
            monkeypatch.setattr(_lib, "host", None)
        c = [t.to(dev).clone() for t in (kc, vc, ks, vs)]
        b, s = (bt.long(), sl.long()) if wide else (bt, sl)
        cu = torch.tensor([0, 2, 4], dtype=s.dtype, device=dev)
        res = [cache8.cache8_decode(q, *c, b, s, scale=0.1, decode_query_len=2, window=20, sinks=3),
               *cache8.cache8_prefill(q, *c, b, cu, s, 2, scale=0.1, return_lse=True),
               cache8.decode_selected(q, *c, ids, ids.float(), b, s, decode_query_len=2, local_blocks=1, scale=0.1)]
        cache8.cache8_append(x, x, *c, b, s - 2, cu_seqlens=cu, max_new_len=2)
        st, m = cache_pages.pages_reserve(cache_pages.PageTable(bt, sl, ref), s + 3, page_size=page)
        st, k = cache_pages.pages_reorder(st, torch.tensor([1, 1], device=dev, dtype=s.dtype), c, page_size=page)
        st, live = cache_pages.pages_compact(st, c)
        got.append(res + [t.view(torch.int8) for t in c] + list(st) + [m, k, live])
    assert len(got[0]) == len(got[1])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_arguments_of_other_kinds(dev):
    """Numbers that are not Python's own, truth values that are not bools, an output of a wider tensor."""
    import numpy as np
    from srswa import cache8
    g = torch.Generator().manual_seed(62)
    c = dict(page=16, HQ=4, HKV=2, D=64, W=4, kv=torch.int8)
    table, kc, vc, ks, vs = _state(c, g, [50, 20])
    q = torch.randn(4, 4, 64, generator=g).to(BF).to(dev)
    args = [t.to(dev) for t in (kc, vc, ks, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev)]
    sl, cu = torch.tensor([50, 20], dtype=torch.int32).to(dev), torch.tensor([0, 2, 4], dtype=torch.int32).to(dev)
    want = cache8.cache8_decode(q, *args, sl, scale=0.5, decode_query_len=2, window=9, sinks=2, return_lse=True)
    wide = torch.empty(4, 9, 64, dtype=BF, device=dev)
    for kw in (dict(return_lse=1), dict(return_lse=np.True_), dict(return_lse=True, out=wide[:, 3:7])):
        runs = [cache8.cache8_decode(q, *args, sl, scale=np.float32(0.5), decode_query_len=np.int64(2),
                                     window=np.int32(9), sinks=np.int64(2), **kw),
                cache8.cache8_decode(q, *args, sl, scale=0.5, decode_query_len=2, window=9, sinks=2, **kw),
                cache8.cache8_prefill(q, *args, cu, sl, 2, scale=0.5, window=9, sinks=2, **kw)]
        for got in runs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.is_tensor(cache8.cache8_decode(q, *args, sl, scale=0.5, decode_query_len=2, return_lse=0))


def test_empty_calls(dev):
    from srswa import cache8
    kc = torch.zeros(3, 16, 1, 64, dtype=torch.int8, device=dev)
    s = torch.ones(3, 1, device=dev)
    none = torch.zeros(0, 2, 64, dtype=BF, device=dev)
    bt, i0 = torch.zeros(0, 2, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    assert cache8.cache8_decode(none, kc, kc, s, s, bt, i0, scale=1.0).shape == (0, 2, 64)
    assert cache8.cache8_prefill(none, kc, kc, s, s, bt, torch.zeros(1, dtype=torch.int32, device=dev), i0, 0,
                                 scale=1.0).shape == (0, 2, 64)
    q = torch.ones(1, 2, 64, dtype=BF, device=dev)
    one = torch.ones(1, dtype=torch.int32, device=dev)
    o, lse = cache8.cache8_decode(q, kc, kc, s, s, torch.zeros(1, 0, dtype=torch.int32, device=dev), one, scale=1.0,
                                  return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    x = torch.zeros(0, 1, 64, dtype=BF, device=dev)
    cache8.cache8_append(x, x, kc, kc.clone(), s, s.clone(), torch.zeros(1, 2, dtype=torch.int32, device=dev), one,
                         cu_seqlens=torch.zeros(2, dtype=torch.int32, device=dev), max_new_len=4)
    assert not kc.any() and (s == 1).all()


# Small cases take the form by items of 16 rows; these run them through the 128-row tiles
# too, with a bound on the longest request that is far above it.
WIDE = 1 << 15


@pytest.fixture
def form(monkeypatch):
    def take(bound):
        monkeypatch.setenv("SRSWA_CACHE8_PREFILL", "tiles" if bound == WIDE else "items")
    return take


def _prefill(dev, c, g, bound, spoil=None, q=None):
    """(out, lse, oracle) of PREFILL-like case c; `spoil` may plant bytes in K and V."""
    from srswa import cache8
    lens = [a + b for a, b in zip(c["q"], c["ctx"])]
    table, kc, vc, ks, vs = _state(c, g, lens)
    if spoil:
        spoil(table, kc, vc, ks, vs)
    cu = torch.tensor([0] + c["q"]).cumsum(0).tolist()
    q = torch.randn(cu[-1], c["HQ"], c["D"], generator=g).to(BF) if q is None else q
    win, sinks, scale = c.get("window"), c.get("sinks", 0), c["D"] ** -0.5
    ref = O.attend(q, kc, vc, ks, vs, table, cu, lens, scale, window=win, sinks=sinks)
    got, lse = cache8.cache8_prefill(*(t.to(dev) for t in (q, kc, vc, ks, vs)),
                                     torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(cu).to(dev),
                                     torch.tensor(lens).to(dev), bound or max(c["q"]), scale=scale, window=win,
                                     sinks=sinks, return_lse=True)
    return got, lse, ref


@pytest.mark.parametrize("kv", [torch.int8, E4M3])
@pytest.mark.parametrize("name", list(PREFILL))
def test_prefill_tiles_match_oracle(dev, form, name, kv):
    form(WIDE)
    g = torch.Generator().manual_seed(list(PREFILL).index(name) + 160)
    got, lse, ref = _prefill(dev, dict(PREFILL[name], kv=kv), g, WIDE)
    _check(got, lse, ref, name)


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("bound", [1, 3, 50, 600])
def test_rows_past_the_bound_are_left(dev, form, bound, tiles):
    """Requests longer than max_query_len: their first rows are right, the others untouched."""
    from srswa import cache8
    form(WIDE if tiles else 0)
    g = torch.Generator().manual_seed(172)
    c = dict(page=64, HQ=8, HKV=2, D=64, W=60, kv=torch.int8)
    n, ctx = [70, 2, 650, 5], [3000, 10, 100, 2500]
    lens = [a + b for a, b in zip(n, ctx)]
    table, kc, vc, ks, vs = _state(c, g, lens)
    cu = [0, 70, 72, 722, 727]
    q = torch.randn(727, 8, 64, generator=g).to(BF)
    keep = [i for r in range(4) for i in range(cu[r], cu[r] + min(n[r], bound))]
    some = sorted(set(keep[:40] + keep[-40:]))            # (the oracle is slow)
    cuts = [sum(1 for i in some if i < x) for x in cu]
    out = torch.full(q.shape, 7.0, dtype=BF, device=dev)
    cache8.cache8_prefill(*(t.to(dev) for t in (q, kc, vc, ks, vs)), torch.tensor(table, dtype=torch.int32).to(dev),
                          torch.tensor(cu).to(dev), torch.tensor(lens).to(dev), bound, scale=0.125, out=out)
    rest = [i for i in range(727) if i not in set(keep)]
    assert (out[rest] == 7.0).all()
    for r in range(4):
        rows = some[cuts[r]:cuts[r + 1]]
        for i in rows:                                    # one row at a time: its own length
            o, _, tol = O.attend(q[i:i + 1], kc, vc, ks, vs, [table[r]], [0, 1], [lens[r] - (cu[r + 1] - 1 - i)], 0.125)
            assert ((out[i:i + 1].cpu().double() - o).abs() <= tol).all(), (bound, i)


@pytest.mark.parametrize("bound", [0, WIDE])
def test_prefill_of_many_requests(dev, form, bound):
    """More requests than a wave has lanes: each workgroup finds its own."""
    form(bound)
    g = torch.Generator().manual_seed(171)
    n = torch.randint(0, 9, (150,), generator=g).tolist()
    n[70], n[149] = 140, 33
    c = dict(page=16, HQ=4, HKV=2, D=64, kv=E4M3, q=n, ctx=torch.randint(0, 20, (150,), generator=g).tolist(), W=10)
    got, lse, ref = _prefill(dev, c, g, bound)
    _check(got, lse, ref, "150 requests")


def test_prefill_takes_either_form_by_itself(dev):
    """Shapes on both sides of the choice, the same requests cut into calls of few rows
    and in one of many: equal within the forms' roundings."""
    from srswa import cache8
    g = torch.Generator().manual_seed(173)
    page, HQ, HKV, D, R = 64, 16, 8, 64, 4
    n, ctx = 700, 300
    table, pages = _table(g, [n + ctx] * R, page, 16)
    kc, ks = _cache(g, pages, page, HKV, D, E4M3)
    vc, vs = _cache(g, pages, page, HKV, D, E4M3)
    q = torch.randn(R, n, HQ, D, generator=g).to(HF).to(dev)
    args = [t.to(dev) for t in (kc, vc, ks, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev)]

    def run(lo, hi):
        cu = torch.arange(R + 1, dtype=torch.int32, device=dev) * (hi - lo)
        sl = torch.full((R,), ctx + hi, dtype=torch.int32, device=dev)
        o, lse = cache8.cache8_prefill(q[:, lo:hi].reshape(-1, HQ, D), *args, cu, sl, hi - lo, scale=0.125,
                                       return_lse=True)
        return o.reshape(R, hi - lo, HQ, D).double(), lse.reshape(R, hi - lo, HQ).double()

    whole = run(0, n)
    parts = [run(lo, min(lo + 9, n)) for lo in range(0, n, 9)]
    o, lse = (torch.cat([p[i] for p in parts], 1) for i in range(2))
    # each form: weights within 2^-11 of a half step in fp16 and an output rounding of 2^-11, of values up to max |v|
    top = (vc.float().abs().amax((1, 3)) * vs).amax().item()
    assert ((whole[0] - o).abs() <= 4 * 2.0 ** -11 * top).all()
    assert ((whole[1] - lse).abs() <= 1e-4 * (1 + lse.abs())).all()


def _check_nan(got, lse, ref, what):
    o, l, tol = ref
    got, lse = got.cpu().double(), lse.cpu().double()
    bad, lbad = torch.isnan(o), torch.isnan(l)
    assert bad.any(), what
    assert torch.equal(torch.isnan(got), bad), (what, (torch.isnan(got) != bad).nonzero()[:8].tolist())
    assert torch.equal(torch.isnan(lse), lbad), what
    assert ((got - o).abs() <= tol)[~bad].all(), what
    fine = ~lbad & ~torch.isinf(l)
    assert torch.equal(torch.isinf(lse), torch.isinf(l)), what
    assert ((lse - l).abs()[fine] <= 1e-4 * (1 + l[fine].abs())).all(), what


NANS = {
    "causal": dict(page=16, HQ=4, HKV=2, D=64, q=[40, 70], ctx=[30, 0], W=5,
                   at=[(0, 31, 0, 5), (0, 69, 1, 63), (1, 0, 0, 1), (1, 50, 1, 8)]),
    "causal_128": dict(page=64, HQ=2, HKV=2, D=128, q=[150], ctx=[70], W=4,
                       at=[(0, 75, 0, 127), (0, 130, 1, 64), (0, 200, 0, 0), (0, 219, 1, 33)]),
    "window": dict(page=32, HQ=4, HKV=1, D=128, q=[90, 33], ctx=[200, 40], W=10, window=50, sinks=20,
                   at=[(0, 18, 0, 3), (0, 100, 0, 4), (0, 160, 0, 77), (0, 230, 0, 100), (0, 289, 0, 9),
                       (1, 10, 0, 11)]),
    "pages_of_48": dict(page=48, HQ=2, HKV=1, D=64, q=[130], ctx=[20], W=4, at=[(0, 30, 0, 3), (0, 100, 0, 40)]),
}


@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("bound", [0, WIDE])
@pytest.mark.parametrize("name", list(NANS))
def test_prefill_keeps_a_nan_to_the_rows_that_see_it(dev, form, name, bound, what):
    """A stored NaN reaches the rows that see its key, in V its own dim only; a
    query's NaN its own row."""
    form(bound)
    c = dict(NANS[name], kv=E4M3)
    g = torch.Generator().manual_seed(181)

    def spoil(table, kc, vc, ks, vs):
        for r, j, h, d in c["at"]:
            if what != "q":
                (kc if what == "k" else vc).view(torch.int8)[table[r][j // c["page"]], j % c["page"], h, d] = -1

    q = None
    if what == "q":
        q = torch.randn(sum(c["q"]), c["HQ"], c["D"], generator=g).to(BF)
        q[7, 1, 3], q[-1, 0] = math.nan, math.nan
    got, lse, ref = _prefill(dev, c, g, bound, spoil, q)
    _check_nan(got, lse, ref, (name, bound, what))


@pytest.mark.parametrize("D", [64, 128])
def test_decode_keeps_a_nan_to_the_rows_that_see_it(dev, D):
    from srswa import cache8
    c = dict(page=16, HQ=6, HKV=2, D=D, W=160, kv=E4M3)
    g = torch.Generator().manual_seed(191)
    lens, dql = [2503, 61, 9], 5
    table, kc, vc, ks, vs = _state(c, g, lens)
    for r, j, h, d in ((0, 2500, 0, 3), (0, 2502, 1, 40), (1, 58, 0, 63), (2, 6, 1, 0), (2, 0, 0, 17)):
        vc.view(torch.int8)[table[r][j // 16], j % 16, h, d] = 127
    q = torch.randn(3 * dql, 6, D, generator=g).to(BF)
    for win in (None, 7):
        ref = O.attend(q, kc, vc, ks, vs, table, [0, 5, 10, 15], lens, 0.125, window=win, sinks=2)
        got = cache8.cache8_decode(*(t.to(dev) for t in (q, kc, vc, ks, vs)),
                                   torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(lens).to(dev),
                                   scale=0.125, decode_query_len=dql, window=win, sinks=2, return_lse=True)
        _check_nan(*got, ref, win)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_smallest_and_largest_v_scales(dev, form, dtype):
    """A cache of zeros (scale 2^-100) and, in bf16, the largest finite values."""
    form(WIDE)
    from srswa import cache8
    g = torch.Generator().manual_seed(201)
    table, n = _table(g, [600, 600], 16, 38)
    kc, ks = _cache(g, n, 16, 1, 64, E4M3)
    vc, vs = _cache(g, n, 16, 1, 64, E4M3)
    for p in table[0]:
        vc.view(torch.int8)[p], vs[p] = 0, 2.0 ** -100
    for p in table[1]:
        vs[p] = 2.0 ** 119 if dtype == BF else 2.0 ** 4
    q = torch.randn(2, 2, 64, generator=g).to(dtype)
    ref = O.attend(q, kc, vc, ks, vs, table, [0, 1, 2], [600, 600], 0.125)
    args = [t.to(dev) for t in (q, kc, vc, ks, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev)]
    lens = torch.tensor([600, 600]).to(dev)
    _check(*cache8.cache8_decode(*args, lens, scale=0.125, return_lse=True), ref, "decode")
    _check(*cache8.cache8_prefill(*args, torch.arange(3).to(dev), lens, WIDE, scale=0.125, return_lse=True), ref,
           "tiles")


def test_decode_and_append_of_many_requests(dev):
    """More requests than a wave has lanes, long and short, shared out by units."""
    from srswa import cache8
    g = torch.Generator().manual_seed(211)
    lens = torch.randint(0, 40, (130,), generator=g).tolist()
    lens[3], lens[100], lens[129] = 5000, 3000, 4500
    table, n = _table(g, [x + 30 for x in lens], 32, 160)
    kc, ks = _cache(g, n, 32, 3, 64, torch.int8)
    vc, vs = _cache(g, n, 32, 3, 64, torch.int8)
    runs = torch.randint(0, 4, (130,), generator=g).tolist()
    runs[66], runs[129] = 29, 30
    k, v = (torch.randn(sum(runs), 3, 64, generator=g).to(BF) for _ in range(2))
    ref = [O.append(x, y, s, table, lens, runs) for x, y, s in ((k, kc, ks), (v, vc, vs))]
    d = [t.to(dev) for t in (k, v, kc, vc, ks, vs)]
    bt = torch.tensor(table, dtype=torch.int32).to(dev)
    cache8.cache8_append(*d, bt, torch.tensor(lens).to(dev),
                         cu_seqlens=torch.tensor([0] + runs).cumsum(0).to(dev), max_new_len=30)
    for got, want in zip(d[2:], (ref[0][0], ref[1][0], ref[0][1], ref[1][1])):
        assert torch.equal(got.cpu(), want)
    lens = [a + b for a, b in zip(lens, runs)]
    q = torch.randn(130, 3, 64, generator=g).to(BF)
    want = O.attend(q, ref[0][0], ref[1][0], ref[0][1], ref[1][1], table, list(range(131)), lens, 0.125)
    _check(*cache8.cache8_decode(q.to(dev), *d[2:], bt, torch.tensor(lens).to(dev), scale=0.125, return_lse=True), want,
           "130 requests")


def test_offsets_past_32_bits(dev, form):
    """Pages more than 2^32 bytes into a cache: append, decode, prefill and a page copy there."""
    from srswa import cache8, cache_pages
    g = torch.Generator().manual_seed(231)
    page, H, D, N = 64, 4, 128, 140_000
    far = torch.zeros(2, N, page, H, D, dtype=torch.int8, device=dev)
    sc = torch.ones(2, N, H, device=dev)
    lens, ids = [150, 70], [N - 1, 7, N - 3, N - 9, 131_073]
    kc, ks = _cache(g, 6, page, H, D, torch.int8)
    vc, vs = _cache(g, 6, page, H, D, torch.int8)
    table = [[0, 1, 2], [3, 4, -1]]
    far_table = torch.tensor([[ids[x] if x >= 0 else -1 for x in row] for row in table], dtype=torch.int32).to(dev)
    for i, x in enumerate(ids):
        far[0, x], far[1, x], sc[0, x], sc[1, x] = kc[i].to(dev), vc[i].to(dev), ks[i].to(dev), vs[i].to(dev)
    k, v = (torch.randn(2, H, D, generator=g).to(BF) for _ in range(2))
    kc, ks = O.append(k, kc, ks, table, lens, [1, 1])
    vc, vs = O.append(v, vc, vs, table, lens, [1, 1])
    state = (far[0], far[1], sc[0], sc[1])
    sl = torch.tensor(lens, dtype=torch.int32).to(dev)
    cache8.cache8_append(k.to(dev), v.to(dev), *state, far_table, sl)
    lens, sl = [n + 1 for n in lens], sl + 1
    q = torch.randn(2 * 40, H, D, generator=g).to(BF)
    ref = O.attend(q, kc, vc, ks, vs, table, [0, 40, 80], lens, 0.1)
    for bound in (40, WIDE):
        form(bound)
        got = cache8.cache8_prefill(q.to(dev), *state, far_table, torch.tensor([0, 40, 80]).to(dev), sl, bound, scale=0.1,
                                    return_lse=True)
        _check(*got, ref, bound)
    pool = torch.zeros(N, dtype=torch.int32, device=dev)
    pool[far_table[far_table >= 0].long()] = 1
    pool[:N - 2] += 1                                     # held by others: the free page is the last but one
    pool[N - 2] = 0
    st, missing = cache_pages.pages_reorder(cache_pages.PageTable(far_table, sl, pool), torch.zeros_like(sl), state,
                                            page_size=page)
    assert int(missing) == 0 and st.block_table[1].tolist() == [N - 1, 7, N - 2]
    o, lse = cache8.cache8_decode(q[38:40].to(dev), *state, st.block_table, st.seq_lens, scale=0.1, return_lse=True)
    one = O.attend(q[38:40], kc, vc, ks, vs, [table[0], table[0]], [0, 1, 2], [lens[0]] * 2, 0.1)
    _check(o, lse, one, "forked")


def test_a_page_s_rows_far_apart(dev, form):
    """A cache stored by place in the page first: token strides past 2^25 bytes."""
    from srswa import cache8
    g = torch.Generator().manual_seed(241)
    page, H, D, N = 64, 4, 128, 65_700
    base = torch.zeros(page, N, H, D, dtype=torch.int8, device=dev)
    far = base.permute(1, 0, 2, 3)
    assert far.stride(1) > 1 << 25
    lens, table, ids = [150, 64], [[0, 1, 2], [3, -1, -1]], [N - 1, 7, N - 3, 40_000]
    kc, ks = _cache(g, 4, page, H, D, torch.int8)
    _, vs = _cache(g, 4, page, H, D, torch.int8)
    sk, sv = torch.ones(N, H, device=dev), torch.ones(N, H, device=dev)
    for i, x in enumerate(ids):
        far[x], sk[x], sv[x] = kc[i].to(dev), ks[i].to(dev), vs[i].to(dev)
    bt = torch.tensor([[ids[x] if x >= 0 else -1 for x in row] for row in table], dtype=torch.int32).to(dev)
    q = torch.randn(80, H, D, generator=g).to(BF)
    ref = O.attend(q, kc, kc, ks, vs, table, [0, 40, 80], lens, 0.1)
    for bound in (40, WIDE):
        form(bound)
        got = cache8.cache8_prefill(q.to(dev), far, far, sk, sv, bt, torch.tensor([0, 40, 80]).to(dev),
                                    torch.tensor(lens).to(dev), bound, scale=0.1, return_lse=True)
        _check(*got, ref, bound)


def test_many_selected_blocks_of_few_long_requests(dev):
    """A table of selected blocks longer than the sequence has, shared out by units."""
    from srswa.unlimited_dash_ops import dash_sparse_attn_decode
    g = torch.Generator().manual_seed(221)
    c = dict(page=16, HKV=2, D=128, W=320, kv=E4M3)
    lens = [5000, 2000]
    table, kc, vc, ks, vs = _state(c, g, lens)
    ids = torch.stack([torch.randperm(330, generator=g)[:300] for _ in range(4)]).reshape(2, 2, 300).to(torch.int32)
    q = torch.randn(2, 4, 128, generator=g).to(HF)
    ref = O.attend(q, kc, vc, ks, vs, table, [0, 1, 2], lens, 0.1, window=32, topk=ids)
    out = torch.empty_like(q, device=dev)
    dash_sparse_attn_decode(q.to(dev), kc.to(dev), vc.to(dev), ids.to(dev), None,
                            torch.tensor(table, dtype=torch.int32).to(dev), torch.tensor(lens).to(dev), 2, 0.1, out, 1,
                            local_blocks=2, sparse_block_size=16, k_scale=ks.to(dev), v_scale=vs.to(dev))
    _check(out, None, ref, "selected")


# ------------------------------------------------------------ used together
def _serve(dev, g, kv):
    """A pool, its caches and helpers for the runs below."""
    from srswa import cache8, cache_pages
    page, H, D, N, R, W = 16, 2, 64, 40, 4, 8
    i32 = dict(dtype=torch.int32, device=dev)
    st = cache_pages.PageTable(torch.full((R, W), -1, **i32), torch.zeros(R, **i32), torch.zeros(N, **i32))
    kc, vc = (torch.zeros(N, page, H, D, device=dev).to(kv) for _ in range(2))
    ks, vs = torch.full((N, H), math.nan, device=dev), torch.full((N, H), math.nan, device=dev)
    return cache8, cache_pages, st, (kc, vc, ks, vs), page, H, D


@pytest.mark.parametrize("kv", [torch.int8, E4M3])
def test_prompt_fork_append_compact_decode(dev, kv):
    """Prompts are stored, one is forked and one freed, tokens are appended, the
    pool is compacted: what decode sees stays what the tokens say."""
    g = torch.Generator().manual_seed(31)
    cache8, pages, st, caches, page, H, D = _serve(dev, g, kv)
    seqs = [torch.randn(2, n, H, D, generator=g).to(BF) for n in (37, 16, 50, 5)]

    def store(st, old, new):
        st2, missing = pages.pages_reserve(st, torch.tensor([s.shape[1] for s in new]).to(dev), page_size=page)
        assert int(missing) == 0
        runs = [b.shape[1] - a for a, b in zip(old, new)]
        x = torch.cat([s[:, o:] for s, o in zip(new, old)], 1).to(dev)
        cache8.cache8_append(x[0], x[1], *caches, st2.block_table, torch.tensor(old).to(dev),
                             cu_seqlens=torch.tensor([0] + runs).cumsum(0).to(dev), max_new_len=max(runs))
        return st2

    def look(st, seqs, what):
        q = torch.randn(4, 4, D, generator=g).to(BF)
        o, lse = cache8.cache8_decode(q.to(dev), *caches, st.block_table, st.seq_lens, scale=0.125, return_lse=True)
        kc, vc, ks, vs = (t.cpu() for t in caches)
        table, lens = st.block_table.tolist(), st.seq_lens.tolist()
        assert lens == [s.shape[1] for s in seqs]
        _check(o, lse, O.attend(q, kc, vc, ks, vs, table, [0, 1, 2, 3, 4], lens, 0.125), what)
        for r, s in enumerate(seqs):                      # the stored values are the tokens'
            for x, c, sc in ((s[0], kc, ks), (s[1], vc, vs)):
                if not s.shape[1]:
                    continue
                pg = torch.tensor([table[r][j // page] for j in range(s.shape[1])])
                at = torch.arange(s.shape[1]) % page
                val = c[pg, at].float() * sc[pg][..., None]
                amax = x.float().abs().max()
                assert ((val - x.float()).abs() <= x.float().abs() * 2.0 ** -4 * 1.1 + amax / 60).all(), what

    st = store(st, [0] * 4, seqs)
    look(st, seqs, "stored")
    st, missing = pages.pages_reorder(st, torch.tensor([0, 0, 2, -1]).to(dev), caches, page_size=page)
    assert int(missing) == 0
    seqs = [seqs[0], seqs[0], seqs[2], seqs[3][:, :0]]
    look(st, seqs, "forked")
    old = [s.shape[1] for s in seqs]
    seqs = [torch.cat([s, torch.randn(2, n, H, D, generator=g).to(BF)], 1) for s, n in zip(seqs, (3, 20, 1, 9))]
    st = store(st, old, seqs)
    look(st, seqs, "appended")
    st, n = pages.pages_compact(st, caches)
    assert int(n) == int((st.ref > 0).sum()) and int(st.block_table.max()) == int(n) - 1
    look(st, seqs, "compacted")


def test_captured_step_replays(dev):
    """append and decode of one step captured together, replayed on new inputs
    between eager calls, equal to the eager step each time."""
    from srswa import cache8
    g = torch.Generator().manual_seed(41)
    page, H, D, R = 16, 2, 64, 3
    lens = [700, 33, 1]
    table, n = _table(g, [x + 8 for x in lens], page, 46)
    kc, ks = _cache(g, n, page, H, D, E4M3)
    vc, vs = _cache(g, n, page, H, D, E4M3)
    bt = torch.tensor(table, dtype=torch.int32).to(dev)
    live = [t.to(dev) for t in (kc, vc, ks, vs)]
    eager = [t.clone() for t in live]
    k = torch.zeros(R, H, D, dtype=BF, device=dev)
    v, q = torch.zeros_like(k), torch.zeros(R, 4, D, dtype=BF, device=dev)
    start = torch.tensor(lens, dtype=torch.int32).to(dev)

    def step(c):
        cache8.cache8_append(k, v, *c, bt, start)
        return cache8.cache8_decode(q, *c, bt, start + 1, scale=0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in live])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(live)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        start.copy_(torch.tensor(lens, dtype=torch.int32) + i)
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip(live, eager):
            assert torch.equal(a.view(torch.int8), b.view(torch.int8)), i
        torch.randn(1 << 16, device=dev).sum().item()


def test_another_stream_and_two_calls_at_once(dev):
    from srswa import cache8
    g = torch.Generator().manual_seed(51)
    c = dict(page=64, HQ=4, HKV=2, D=128, W=40, kv=torch.int8)
    table, kc, vc, ks, vs = _state(c, g, [2500, 900])
    q = torch.randn(2, 4, 128, generator=g).to(BF).to(dev)
    args = [t.to(dev) for t in (kc, vc, ks, vs)] + [torch.tensor(table, dtype=torch.int32).to(dev),
                                                   torch.tensor([2500, 900]).to(dev)]
    want = cache8.cache8_decode(q, *args, scale=0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cache8.cache8_decode(q, *args, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
