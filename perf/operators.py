"""The 8-bit paged cache as measurable cases: writing it, attending to it, moving its pages.

Four operators.  ``append`` quantises new keys and values into pages with one
scale per page and kv head; ``decode`` attends one or a few new tokens per
request to such a cache (every key, a sliding window with first tokens that
stay visible, or the router's selected blocks); ``prefill`` does so for many
tokens per request; ``pages`` deals out, reorders (shares, copies, frees) and
compacts the pages of a pool.

``listed()`` names the cases, ``draw(rng)`` gives another of the same ranges.
Lengths depend on the case alone, their order and all values on the seed.
Where ``own`` is false, ``run`` is plain torch in fp32; where it is true, the
package's entry points.
"""

import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
CACHE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
MIN_EXP = -100          # the smallest scale is 2 ** MIN_EXP (a page of zeros)
F64 = torch.float64


def _package():
    path = os.path.join(os.getcwd(), "unlimited-ocr_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from srswa import cache8, cache_pages
    from srswa.unlimited_dash_ops import attend_triton
    return cache8, cache_pages, attend_triton


# --------------------------------------------------------------------- cases
def listed():
    return [
        # a serving step's new tokens, one per request, most into pages already begun
        dict(name="append_step_b64_int8", kind="append", R=64, nlo=1, nhi=1, slo=300, shi=40000, H=10, D=128, BS=64,
             dtype="bf16", kv="int8"),
        # a prefill batch written behind cached prefixes: ragged runs, odd starts, many whole pages
        dict(name="append_chunk_r5_e4m3", kind="append", R=5, nlo=13, nhi=8000, slo=0, shi=30011, H=10, D=128, BS=64,
             dtype="bf16", kv="e4m3"),
        # one interactive request, short cache, one new token: latency
        dict(name="decode_b1_e4m3", kind="decode", R=1, lo=777, hi=777, HQ=10, HKV=10, D=128, BS=64, dql=1, window=0,
             sinks=0, lse=False, dtype="bf16", kv="e4m3"),
        # a batch of very uneven requests, all keys visible, with the softmax statistics
        dict(name="decode_b48_e4m3", kind="decode", R=48, lo=700, hi=40000, HQ=10, HKV=10, D=128, BS=64, dql=1,
             window=0, sinks=0, lse=True, dtype="bf16", kv="e4m3"),
        # two tokens per request, grouped heads, a sliding window behind first tokens that stay visible
        dict(name="decode_window_b64_int8", kind="decode", R=64, lo=4096, hi=131072, HQ=16, HKV=4, D=128, BS=32,
             dql=2, window=512, sinks=100, lse=False, dtype="f16", kv="int8"),
        # the router's selected blocks and a window (the DASH serving step), ids shared by the heads
        dict(name="selected_b48_e4m3", kind="selected", R=48, lo=700, hi=40000, HQ=10, HKV=10, D=128, BS=64, dql=1,
             K=8, LB=8, bias=True, dtype="bf16", kv="e4m3"),
        # a serving prefill batch of uneven requests behind long contexts: window and first tokens
        dict(name="prefill_window_r6_e4m3", kind="prefill", R=6, qlo=70, qhi=1900, ctx=30011, HQ=10, HKV=10, D=128,
             BS=64, window=512, sinks=273, dtype="bf16", kv="e4m3"),
        # one chunk of a long document, every earlier key visible
        dict(name="prefill_2k_of_32k_int8", kind="prefill", R=1, qlo=2048, qhi=2048, ctx=30720, HQ=10, HKV=10, D=128,
             BS=64, window=0, sinks=0, dtype="bf16", kv="int8"),
        # short grouped prompts without a prefix, narrow heads
        dict(name="prefill_r7_gqa_f16", kind="prefill", R=7, qlo=1, qhi=700, ctx=0, HQ=16, HKV=4, D=64, BS=16,
             window=0, sinks=0, dtype="f16", kv="e4m3"),
        # a serving step deals pages to the requests that begin one
        dict(name="pages_reserve_b256", kind="reserve", R=256, W=512, N=131072, lo=300, hi=30000, add=70, BS=64),
        # beam search keeps the better halves: rows reordered, full pages shared, begun pages copied, 12 layers
        dict(name="pages_reorder_b64_12l", kind="reorder", R=64, W=128, N=2048, lo=200, hi=6000, layers=12, H=10, D=128,
             BS=64, kv="int8"),
        # a pool with holes is compacted, 12 layers
        dict(name="pages_compact_12l", kind="compact", R=40, W=256, N=2048, fill=0.5, layers=12, H=10, D=128, BS=64,
             kv="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "selected", "prefill", "prefill", "reserve",
                       "reorder", "compact"])
    HQ, HKV = rng.choice([(10, 10), (10, 10), (8, 8), (16, 4), (16, 8), (8, 1)])
    base = dict(kind=kind, D=rng.choice([128, 128, 64]), BS=rng.choice([64, 64, 32, 16, 128]))
    typed = dict(dtype=rng.choice(["bf16", "bf16", "f16"]), kv=rng.choice(["e4m3", "int8"]))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 30, 2000), rng.choice([0, 1, 4, rng.randint(2, 300)]))])
    if kind == "append":
        nhi = rng.choice([1, rng.randint(1, 5), _log(rng, 10, 8000)])
        return dict(base, R=_log(rng, 1, 64) if nhi < 100 else rng.randint(1, 5), nlo=rng.choice([0, 1]), nhi=nhi,
                    slo=0, shi=_log(rng, 100, 40000), H=HKV, **typed)
    if kind == "decode":
        return dict(base, R=_log(rng, 1, 48), lo=rng.choice([1, 300]), hi=_log(rng, 500, 40000), HQ=HQ, HKV=HKV,
                    dql=rng.choice([1, 1, 2, 3]), window=window, sinks=sinks, lse=rng.random() < 0.3, **typed)
    if kind == "selected":
        return dict(base, R=_log(rng, 1, 64), lo=300, hi=_log(rng, 1000, 40000), HQ=HQ, HKV=HKV,
                    dql=rng.choice([1, 1, 2]), K=rng.choice([8, 4, 12, 7]), LB=rng.choice([8, 4, 2]),
                    bias=rng.random() < 0.7, **typed)
    if kind == "prefill":
        R = rng.randint(1, 6)
        return dict(base, R=R, qlo=rng.randint(0, 90), qhi=_log(rng, 20, 1200), HQ=HQ, HKV=HKV,
                    ctx=rng.choice([0, _log(rng, 100, 30000 // R)]), window=window, sinks=sinks, **typed)
    if kind == "reserve":
        return dict(kind=kind, R=_log(rng, 1, 256), W=512, N=_log(rng, 3000, 131072), lo=100,
                    hi=_log(rng, 1000, 16000), add=_log(rng, 1, 300), BS=rng.choice([32, 64]))
    most = 2048 * 64 // max(64, base["BS"])
    if kind == "reorder":
        R = _log(rng, 2, 64)
        return dict(base, R=R, W=_log(rng, 40, 128), N=most, lo=60, hi=rng.randint(300, 1000) if base["BS"] < 64
                    else rng.randint(300, 2500), layers=rng.randint(1, 12), H=HKV, kv="int8")
    return dict(base, R=_log(rng, 2, 40), W=256, N=_log(rng, 100, most), fill=rng.uniform(0.1, 0.9),
                layers=rng.randint(1, 12), H=HKV, kv="int8")


# ------------------------------------------------------------------- helpers
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _lengths(n, lo, hi):
    """n lengths spread evenly over the logarithm of [lo, hi], odd ones among them."""
    lo1 = max(1, lo)
    return [max(lo, min(hi, int(lo1 * (max(hi, 1) / lo1) ** ((b + 0.5) / n)) + (b * 37) % 61)) for b in range(n)]


def _shuffled(g, v):
    return [v[i] for i in torch.randperm(len(v), generator=g, device="cuda").tolist()]


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(g, nblk, extra=3):
    """Page table [R, max nblk] of randomly dealt pages (-1 behind a request's last), and the pool's size."""
    n = sum(nblk) + extra
    perm = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    bt = torch.full((len(nblk), max(1, max(nblk))), -1, dtype=torch.int32, device="cuda")
    o = 0
    for r, m in enumerate(nblk):
        bt[r, :m] = perm[o:o + m]
        o += m
    return bt, n


def _pow2(e):
    """2 ** e in fp32, exactly (e an int32 tensor within the normal range)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _need(a, kv):
    """The smallest power of two s >= 2 ** MIN_EXP with a <= QMAX s (a >= 0, fp32)."""
    m, x = torch.frexp(a)                                 # a = m 2^x, m in [0.5, 1)
    mq, xq = math.frexp(QMAX[kv])
    e = x - xq + (m > mq).to(x.dtype)
    return _pow2(torch.where(a > 0, e.clamp(min=MIN_EXP), torch.full_like(e, MIN_EXP)))


def _round8(y, kv):
    """y (fp32, in units of the scale) as the cache's bytes."""
    if kv == "e4m3":
        return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.int8)
    return torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127.0, 127.0).to(torch.int8)


def _values(b, kv):
    """The bytes (int8 storage) as fp32, in units of the scale."""
    return b.view(torch.float8_e4m3fn).float() if kv == "e4m3" else b.float()


def _fill(g, npages, BS, H, D, kv):
    """A cache of npages quantised pages [npages, BS, H, D] with its scales [npages, H]; the
    magnitude differs from page to page and head to head."""
    out = torch.empty(npages, BS, H, D, dtype=torch.int8, device="cuda")
    sc = torch.empty(npages, H, device="cuda")
    step = max(1, (1 << 27) // (BS * H * D))
    for i in range(0, npages, step):
        n = min(step, npages - i)
        x = _randn(g, n, BS, H, D) * torch.exp(0.5 * _randn(g, n, 1, H, 1))
        s = _need(x.abs().amax((1, 3)), kv)
        out[i:i + n] = _round8(x / s[:, None, :, None], kv)
        sc[i:i + n] = s
    return out.view(CACHE[kv]), sc


def _spoil(bt, npages, *pairs):
    """The pages that no request holds: scales of NaN, bytes of NaN where the format has one."""
    free = torch.ones(npages, dtype=torch.bool, device="cuda")
    free[bt[bt >= 0].long()] = False
    for cache, scale in pairs:
        cache.view(torch.int8)[free] = 127
        scale[free] = float("nan")


def _runs(c):
    n = _lengths(c["R"], c["nlo"], c["nhi"])
    if c["nlo"] == 0 and c["R"] > 2:
        n[c["R"] // 2] = 0
    return n, [s + (7 * r) % 64 for r, s in enumerate(_lengths(c["R"], c["slo"], c["shi"]))]


def _qlens(c):
    lo, hi = min(c["qlo"], c["qhi"]), c["qhi"]
    ql = [max(lo, min(hi, int(lo + (hi - lo) * r / max(1, c["R"] - 1)) + (r * 13) % 7)) for r in range(c["R"])]
    return ql if sum(ql) else [1] * c["R"]


def _ctxs(c):
    return [max(0, int(c["ctx"] * (r + 1) / c["R"]) - (r * 29) % 53) for r in range(c["R"])]


def _decode_lens(c):
    return [max(n, c["dql"]) for n in _lengths(c["R"], c["lo"], c["hi"])]


def _visible(c, lo, hi):
    """Keys visible to the query positions lo .. hi - 1 together, and visible (position, key) pairs."""
    if hi <= lo:
        return 0, 0
    w, s = c.get("window", 0), c.get("sinks", 0)
    if w <= 0:
        return hi, sum(p + 1 for p in (lo, hi - 1)) * (hi - lo) // 2
    keys = hi - max(0, lo - w + 1) + min(s, max(0, lo - w + 1))
    pairs = sum(min(p + 1, w) + min(s, max(0, p + 1 - w)) for p in range(lo, hi))
    return keys, pairs


def _pool_rows(c):
    """Lengths of the rows of a reorder / reserve case that fit its table and pool."""
    lens, free, out = _lengths(c["R"], c["lo"], c["hi"]), c["N"] - 2 * c["R"], []
    for n in lens:
        n = max(1, min(n, c["W"] * c["BS"] - 1, (free - (c["R"] - len(out))) * c["BS"]))
        free -= -(-n // c["BS"])
        out.append(n)
    return out


def _parents(c):
    """Groups of four beams (the last may be smaller); every group keeps its first two, twice."""
    return [r // 4 * 4 + (r % 4) // 2 for r in range(c["R"])]


def _copies(c, lens):
    """Begun pages that a reorder has to copy (the first child of a parent keeps its page)."""
    return [r for r, p in enumerate(_parents(c)) if p in _parents(c)[:r] and lens[p] % c["BS"]]


# ------------------------------------------------------------------- prepare
def prepare(case, seed):
    c, g = case, _gen(seed)
    return dict({"append": _prep_append, "decode": _prep_decode, "selected": _prep_selected, "prefill": _prep_prefill,
                 "reserve": _prep_reserve, "reorder": _prep_reorder, "compact": _prep_compact}[c["kind"]](c, g), c=c)


def _prep_append(c, g):
    n, start = _runs(c)
    order = torch.randperm(c["R"], generator=g, device="cuda").tolist()
    n, start = [n[i] for i in order], [start[i] for i in order]
    bt, npages = _table(g, [-(-(a + b) // c["BS"]) for a, b in zip(n, start)])
    kc, ks = _fill(g, npages, c["BS"], c["H"], c["D"], c["kv"])
    vc, vs = _fill(g, npages, c["BS"], c["H"], c["D"], c["kv"])
    total = sum(n)
    mag = torch.exp(0.5 * _randn(g, total, c["H"], 1))
    return dict(k=(_randn(g, total, c["H"], c["D"]) * mag).to(DT[c["dtype"]]),
                v=(_randn(g, total, c["H"], c["D"]) * mag).to(DT[c["dtype"]]), kc=kc, vc=vc, ks=ks, vs=vs, bt=bt,
                cu=torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32), start=_i32(start), most=max(n))


def _cached(c, g, lens):
    bt, npages = _table(g, [-(-n // c["BS"]) for n in lens])
    kc, ks = _fill(g, npages, c["BS"], c["HKV"], c["D"], c["kv"])
    vc, vs = _fill(g, npages, c["BS"], c["HKV"], c["D"], c["kv"])
    _spoil(bt, npages, (kc, ks), (vc, vs))
    return dict(kc=kc, vc=vc, ks=ks, vs=vs, bt=bt, sl=_i32(lens))


def _prep_decode(c, g):
    lens = _shuffled(g, _decode_lens(c))
    return dict(_cached(c, g, lens), q=_randn(g, c["R"] * c["dql"], c["HQ"], c["D"], dtype=DT[c["dtype"]]))


def _prep_selected(c, g):
    lens = _shuffled(g, _decode_lens(c))
    s = _cached(c, g, lens)
    rows, K = c["R"] * c["dql"], c["K"]
    pos = (s["sl"][:, None] - c["dql"] + torch.arange(c["dql"], device="cuda")[None]).view(-1, 1)
    nb = ((pos - c["LB"] * c["BS"] + 1) // c["BS"]).clamp(min=0)           # whole blocks before the window
    r = torch.rand(rows, max(K, int(nb.max())), device="cuda", generator=g)
    r = torch.where(torch.arange(r.shape[1], device="cuda")[None] < nb, r, torch.full((), -1.0, device="cuda"))
    v, i = r.topk(K, dim=1)
    i = torch.where(v >= 0, i, torch.full_like(i, 1 << 30)).sort(dim=1).values
    ids = torch.where(i < (1 << 30), i, torch.full_like(i, -1)).to(torch.int32)
    bias = torch.where(ids >= 0, _randn(g, rows, K), torch.zeros((), device="cuda"))
    q = _randn(g, rows, c["HQ"], c["D"], dtype=DT[c["dtype"]])
    return dict(s, q=q, ids=ids[None].expand(c["HKV"], rows, K),
                bias=bias[None].expand(c["HKV"], rows, K) if c["bias"] else None, out=torch.empty_like(q))


def _prep_prefill(c, g):
    ql, ctx = _qlens(c), _ctxs(c)
    order = torch.randperm(c["R"], generator=g, device="cuda").tolist()
    ql, ctx = [ql[i] for i in order], [ctx[i] for i in order]
    return dict(_cached(c, g, [a + b for a, b in zip(ql, ctx)]), most=max(ql),
                cu=torch.tensor([0] + ql, device="cuda").cumsum(0).to(torch.int32),
                q=_randn(g, sum(ql), c["HQ"], c["D"], dtype=DT[c["dtype"]]))


def _prep_reserve(c, g):
    lens = _shuffled(g, _pool_rows(c))
    held, _ = _table(g, [-(-n // c["BS"]) for n in lens], extra=c["N"] - sum(-(-n // c["BS"]) for n in lens))
    bt = torch.full((c["R"], c["W"]), -1, dtype=torch.int32, device="cuda")
    bt[:, :held.shape[1]] = held
    ref = torch.zeros(c["N"], dtype=torch.int32, device="cuda")
    ref[bt[bt >= 0].long()] = 1
    add = [min(1 + (r * 31) % c["add"], c["W"] * c["BS"] - n) for r, n in enumerate(lens)]
    return dict(bt=bt, sl=_i32(lens), ref=ref, new=_i32([a + b for a, b in zip(lens, add)]))


def _layers(c, g):
    """[layers, K and V, pages, tokens, heads, dims] bytes and [layers, K and V, pages, heads] scales of a whole model."""
    kv = torch.randint(-127, 128, (c["layers"], 2, c["N"], c["BS"], c["H"], c["D"]), dtype=torch.int8, device="cuda",
                       generator=g)
    return dict(kv=kv, sc=torch.exp(_randn(g, c["layers"], 2, c["N"], c["H"])))


def _prep_reorder(c, g):
    lens = _pool_rows(c)
    groups = _shuffled(g, list(range(-(-c["R"] // 4))))                  # the last, smaller group stays last
    whole = [x for x in groups if 4 * x + 4 <= c["R"]]
    perm = [4 * x + j for x in whole for j in range(4)] + list(range(4 * len(whole), c["R"]))
    lens = [lens[i] for i in perm]
    held, _ = _table(g, [-(-n // c["BS"]) for n in lens], extra=c["N"] - sum(-(-n // c["BS"]) for n in lens))
    bt = torch.full((c["R"], c["W"]), -1, dtype=torch.int32, device="cuda")
    bt[:, :held.shape[1]] = held
    ref = torch.zeros(c["N"], dtype=torch.int32, device="cuda")
    ref[bt[bt >= 0].long()] = 1
    return dict(_layers(c, g), bt=bt, sl=_i32(lens), ref=ref, par=_i32(_parents(c)))


def _prep_compact(c, g):
    live = max(1, min(int(c["N"] * c["fill"]), c["R"] * c["W"]))
    pages = torch.randperm(c["N"], generator=g, device="cuda")[:live].to(torch.int32)
    bt = torch.full((c["R"] * c["W"],), -1, dtype=torch.int32, device="cuda")
    per = -(-live // c["R"])
    at = torch.arange(live, device="cuda")
    bt[at // per * c["W"] + at % per] = pages
    bt = bt.view(c["R"], c["W"])
    if c["R"] > 1:
        bt[1, 0] = bt[0, 0]                                              # a shared first page
    ref = torch.zeros(c["N"], dtype=torch.int32, device="cuda")
    held = bt[bt >= 0].long()
    ref.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    sl = ((bt >= 0).sum(1) * c["BS"] - 3).clamp(min=0).to(torch.int32)
    return dict(_layers(c, g), bt=bt, sl=sl, ref=ref)


# ----------------------------------------------------------------------- run
def run(state):
    return {"append": _run_append, "decode": _run_decode, "selected": _run_selected, "prefill": _run_prefill,
            "reserve": _run_reserve, "reorder": _run_reorder, "compact": _run_compact}[state["c"]["kind"]](state["c"],
                                                                                                          state)


def _plain_store(x, cache, scale, kv, pg, tok, new, live):
    """One of K / V: pages pg [P] take tokens x[tok] where new [P, BS], after the tokens live [P, BS]."""
    raw = cache.view(torch.int8)[pg]                                     # [P, BS, H, D]
    xn = x[tok].float()
    a = torch.where(new[..., None, None] & torch.isfinite(xn), xn.abs(), torch.zeros((), device=xn.device)).amax((1, 3))
    old, need = scale[pg], _need(a, kv)
    kept = live.any(1)[:, None]
    s = torch.where(kept, torch.maximum(old, need), need)
    grown = _round8(_values(raw, kv) * (old / s)[:, None, :, None], kv)
    b = torch.where(live[..., None, None], grown, raw)
    cache.view(torch.int8)[pg] = torch.where(new[..., None, None], _round8(xn / s[:, None, :, None], kv), b)
    scale[pg] = s


def _run_append(c, s):
    if own:
        cache8, _, _ = _package()
        cache8.cache8_append(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["start"],
                             cu_seqlens=s["cu"], max_new_len=s["most"])
        return dict(kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])
    BS, dev = c["BS"], s["bt"].device
    start, n = s["start"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    b = (start // BS)[:, None] + torch.arange((max(1, s["most"]) - 1) // BS + 2, device=dev)[None]     # [R, T] blocks
    pos = b[..., None] * BS + torch.arange(BS, device=dev)
    new = (pos >= start[:, None, None]) & (pos < (start + n)[:, None, None])
    pages = s["bt"].gather(1, b.clamp(max=s["bt"].shape[1] - 1)).long()
    r, t = (new.any(-1) & (b < s["bt"].shape[1]) & (pages >= 0)).nonzero(as_tuple=True)
    tok = (s["cu"][:-1].long()[r, None] + pos[r, t] - start[r, None]).clamp(0, s["k"].shape[0] - 1)
    live = pos[r, t] < start[r, None]
    _plain_store(s["k"], s["kc"], s["ks"], c["kv"], pages[r, t], tok, new[r, t], live)
    _plain_store(s["v"], s["vc"], s["vs"], c["kv"], pages[r, t], tok, new[r, t], live)
    return dict(kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


def _take(cache, scale, kv, bt, pos, BS):
    """Dequantised rows [R, HKV, n, D] fp32 of the keys pos [R, n] (zeros where the page is missing)."""
    pg = bt.gather(1, (pos // BS).clamp(0, bt.shape[1] - 1)).long()
    x = _values(cache.view(torch.int8)[pg.clamp(min=0), (pos % BS).clamp(min=0)], kv) * scale[pg.clamp(min=0)][..., None]
    return torch.where((pg >= 0)[..., None, None], x, torch.zeros((), device=x.device)).transpose(1, 2)


def _softmax_av(z, ok, v):
    """Masked softmax of z [..., n, L] times v [..., L, D], and the log of its sum; rows without a key give 0, -inf."""
    z = torch.where(ok, z, torch.full((), -math.inf, device=z.device))
    m = z.amax(-1, keepdim=True)
    m0 = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = torch.exp(z - m0)
    t = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(t > 0, t, torch.ones_like(t))
    return o, (m0 + torch.log(t)).squeeze(-1)


def _run_decode(c, s):
    R, dql, HQ, HKV, D, BS = c["R"], c["dql"], c["HQ"], c["HKV"], c["D"], c["BS"]
    if own:
        cache8, _, _ = _package()
        got = cache8.cache8_decode(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["sl"], scale=D ** -0.5,
                                   decode_query_len=dql, window=c["window"] or None, sinks=c["sinks"],
                                   return_lse=c["lse"])
        return dict(o=got[0], lse=got[1]) if c["lse"] else dict(o=got)
    dev = s["q"].device
    sl = s["sl"].long()
    qp = sl[:, None] - dql + torch.arange(dql, device=dev)[None]         # [R, dql]
    pos = torch.arange(s["bt"].shape[1] * BS, device=dev)[None].expand(R, -1)
    if c["window"]:
        lo = (sl - dql - c["window"] + 1).clamp(min=0)                   # first key of the first row's window
        first = torch.arange(c["sinks"], device=dev)[None].expand(R, -1)
        first = torch.where(first < lo[:, None], first, torch.full_like(first, -1))
        pos = torch.cat([first, lo[:, None] + torch.arange(c["window"] + dql - 1, device=dev)[None]], 1)
    ok = (pos[:, None] >= 0) & (pos[:, None] <= qp[..., None])           # [R, dql, n]
    if c["window"]:
        ok = ok & ((pos[:, None] > qp[..., None] - c["window"]) | (pos[:, None] < c["sinks"]))
    ok = ok & (s["bt"].gather(1, (pos // BS).clamp(0, s["bt"].shape[1] - 1)) >= 0)[:, None]
    k = _take(s["kc"], s["ks"], c["kv"], s["bt"], pos, BS)
    v = _take(s["vc"], s["vs"], c["kv"], s["bt"], pos, BS)
    v = torch.where(ok.any(1)[:, None, :, None], v, torch.zeros((), device=dev))
    q = s["q"].float().view(R, dql, HKV, HQ // HKV, D).permute(0, 2, 1, 3, 4).reshape(R, HKV, -1, D)
    z = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5                   # [R, HKV, dql * G, n]
    o, lse = _softmax_av(z, ok[:, None, :, None].expand(R, HKV, dql, HQ // HKV, -1).reshape(z.shape), v)
    o = o.view(R, HKV, dql, HQ // HKV, D).permute(0, 2, 1, 3, 4).reshape(R * dql, HQ, D).to(s["q"].dtype)
    lse = lse.view(R, HKV, dql, HQ // HKV).permute(0, 2, 1, 3).reshape(R * dql, HQ)
    return dict(o=o, lse=lse) if c["lse"] else dict(o=o)


def _run_selected(c, s):
    R, dql, HQ, HKV, D, BS, K = c["R"], c["dql"], c["HQ"], c["HKV"], c["D"], c["BS"], c["K"]
    if own:
        _, _, attend = _package()
        attend.dash_sparse_attn_decode(s["q"], s["kc"], s["vc"], s["ids"], s["bias"], s["bt"], s["sl"], HKV, D ** -0.5,
                                       s["out"], dql, local_blocks=c["LB"], sparse_block_size=BS, k_scale=s["ks"],
                                       v_scale=s["vs"])
        return s["out"]
    dev, LW = s["q"].device, c["LB"] * BS
    qp = (s["sl"].long()[:, None] - dql + torch.arange(dql, device=dev)[None]).view(-1, 1)         # [rows, 1]
    bt = s["bt"].repeat_interleave(dql, 0)
    ids = s["ids"][0].long()                                             # one selection for every head here
    remote = (ids[..., None] * BS + torch.arange(BS, device=dev)).view(-1, K * BS)
    pos = torch.cat([remote, qp - LW + 1 + torch.arange(LW, device=dev)[None]], 1)
    ok = torch.cat([(ids >= 0).repeat_interleave(BS, 1) & (remote < qp - LW + 1), pos[:, K * BS:] >= 0], 1)
    add = torch.zeros(pos.shape, device=dev)
    if s["bias"] is not None:
        add[:, :K * BS] = s["bias"][0].repeat_interleave(BS, 1)
    k = _take(s["kc"], s["ks"], c["kv"], bt, pos.clamp(min=0), BS)
    v = _take(s["vc"], s["vs"], c["kv"], bt, pos.clamp(min=0), BS)
    v = torch.where(ok[:, None, :, None], v, torch.zeros((), device=dev))
    q = s["q"].float().view(R * dql, HKV, HQ // HKV, D)
    z = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5 + add[:, None, None]
    return _softmax_av(z, ok[:, None, None], v)[0].reshape(R * dql, HQ, D).to(s["q"].dtype)


def _run_prefill(c, s):
    R, HQ, HKV, D, BS = c["R"], c["HQ"], c["HKV"], c["D"], c["BS"]
    if own:
        cache8, _, _ = _package()
        return cache8.cache8_prefill(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["cu"], s["sl"], s["most"],
                                     scale=D ** -0.5, window=c["window"] or None, sinks=c["sinks"])
    dev, most = s["q"].device, s["most"]
    cu, sl = s["cu"].long(), s["sl"].long()
    ql = cu[1:] - cu[:-1]
    t = torch.arange(most, device=dev)[None]
    row = torch.where(t < ql[:, None], cu[:-1, None] + t, torch.zeros_like(t))
    qp = torch.where(t < ql[:, None], (sl - ql)[:, None] + t, torch.full_like(t, -1))
    pos = torch.arange(s["bt"].shape[1] * BS, device=dev)[None]
    ok = pos[:, None] <= qp[..., None]                                   # [R, most, L]
    if c["window"]:
        ok = ok & ((pos[:, None] > qp[..., None] - c["window"]) | (pos[:, None] < c["sinks"]))
    k = _take(s["kc"], s["ks"], c["kv"], s["bt"], pos.expand(R, -1), BS)
    v = _take(s["vc"], s["vs"], c["kv"], s["bt"], pos.expand(R, -1), BS)
    v = torch.where(ok.any(1)[:, None, :, None], v, torch.zeros((), device=dev))
    q = s["q"][row].float().view(R, most, HKV, HQ // HKV, D).permute(0, 2, 3, 1, 4)
    z = torch.matmul(q.reshape(R, HKV, -1, D), k.transpose(2, 3)).view(R, HKV, HQ // HKV, most, -1) * D ** -0.5
    o, _ = _softmax_av(z, ok[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(R, most, HQ, D)
    return o[t.expand(R, -1) < ql[:, None]].to(s["q"].dtype)


def _run_reserve(c, s):
    if own:
        _, pages, _ = _package()
        st, short = pages.pages_reserve(pages.PageTable(s["bt"], s["sl"], s["ref"]), s["new"], page_size=c["BS"])
        return dict(bt=st.block_table, sl=st.seq_lens, ref=st.ref, short=short)
    W, dev = c["W"], s["bt"].device
    need = (torch.arange(W, device=dev)[None] < ((s["new"] + c["BS"] - 1) // c["BS"])[:, None]) & (s["bt"] < 0)
    free = (s["ref"] == 0).nonzero().squeeze(1).to(torch.int32)
    rank = need.view(-1).cumsum(0).view(need.shape) - 1
    got = need & (rank < free.numel())
    bt = torch.where(got, torch.cat([free, free.new_zeros(1)])[rank.clamp(0, free.numel())], s["bt"])
    ref = s["ref"].clone()
    ref[bt[got].long()] = 1
    return dict(bt=bt, sl=s["new"].clone(), ref=ref, short=(need & ~got).sum().to(torch.int32).view(1))


def _held(bt, n):
    """How often each of n pages stands in bt."""
    ids = bt[bt >= 0].long()
    return torch.zeros(n, dtype=torch.int32, device=bt.device).index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))


def _run_reorder(c, s):
    if own:
        _, pages, _ = _package()
        caches = [x for i in range(c["layers"]) for x in (s["kv"][i, 0], s["kv"][i, 1], s["sc"][i, 0], s["sc"][i, 1])]
        st, short = pages.pages_reorder(pages.PageTable(s["bt"], s["sl"], s["ref"]), s["par"], caches,
                                        page_size=c["BS"])
        return dict(bt=st.block_table, sl=st.seq_lens, ref=st.ref, short=short, kv=s["kv"], sc=s["sc"])
    R, W, BS, N, dev = c["R"], c["W"], c["BS"], c["N"], s["bt"].device
    par = s["par"].long()
    alive = par >= 0
    rows = s["bt"][par.clamp(min=0)]
    sl = torch.where(alive, s["sl"][par.clamp(min=0)], torch.zeros_like(s["sl"]))
    at = torch.arange(R, device=dev)
    first = alive & ~((par[:, None] == par[None]) & (at[None] < at[:, None])).any(1)
    full = (sl // BS).long()
    bt = torch.where((alive[:, None] & (torch.arange(W, device=dev)[None] < full[:, None])) | first[:, None], rows,
                     torch.full_like(rows, -1))
    src = rows.gather(1, full.clamp(max=W - 1)[:, None]).squeeze(1)
    want = alive & ~first & (sl % BS > 0) & (src >= 0)
    ref = s["ref"] - _held(s["bt"], N) + _held(bt, N)
    free = (ref == 0).nonzero().squeeze(1).to(torch.int32)
    rank = want.cumsum(0) - 1
    got = want & (rank < free.numel())
    r = got.nonzero().squeeze(1)
    dst = free[rank[r]]
    bt[r, full[r]] = dst
    ref[dst.long()] = 1
    s["kv"][:, :, dst.long()] = s["kv"][:, :, src[r].long()]
    s["sc"][:, :, dst.long()] = s["sc"][:, :, src[r].long()]
    return dict(bt=bt, sl=sl, ref=ref, short=(want & ~got).sum().to(torch.int32).view(1), kv=s["kv"], sc=s["sc"])


def _run_compact(c, s):
    if own:
        _, pages, _ = _package()
        caches = [x for i in range(c["layers"]) for x in (s["kv"][i, 0], s["kv"][i, 1], s["sc"][i, 0], s["sc"][i, 1])]
        st, live = pages.pages_compact(pages.PageTable(s["bt"], s["sl"], s["ref"]), caches)
        return dict(bt=st.block_table, sl=st.seq_lens, ref=st.ref, live=live, kv=s["kv"], sc=s["sc"])
    held = s["ref"] > 0
    n = held.sum()
    at = torch.arange(c["N"], device=held.device)
    dst = ((at < n) & ~held).nonzero().squeeze(1)
    src = ((at >= n) & held).nonzero().squeeze(1)
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    ref = s["ref"].clone()
    ref[dst] = ref[src]
    ref[src] = 0
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    s["sc"][:, :, dst] = s["sc"][:, :, src]
    bt = torch.where(s["bt"] >= 0, to[s["bt"].clamp(min=0).long()], s["bt"])
    return dict(bt=bt, sl=s["sl"].clone(), ref=ref, live=n.to(torch.int32).view(1), kv=s["kv"], sc=s["sc"])


# ---------------------------------------------------------------------- work
def work(case):
    c, kind = case, case["kind"]
    if kind == "append":
        n, start = _runs(c)
        row = c["H"] * c["D"]
        touched = sum(-(-(s + m) // c["BS"]) - s // c["BS"] for m, s in zip(n, start) if m)
        return dict(bytes=sum(n) * row * 2 * (2 + 1) + touched * c["H"] * 16 + 4 * touched, flops=sum(n) * row * 4)
    if kind in ("decode", "selected", "prefill"):
        g = c["HQ"] * c["D"]
        keys = pairs = rows = 0
        if kind == "prefill":
            spans = [(x, x + q) for q, x in zip(_qlens(c), _ctxs(c))]
        else:
            spans = [(n - c["dql"], n) for n in _decode_lens(c)]
        for lo, hi in spans:
            rows += hi - lo
            if kind == "selected":
                for p in range(lo, hi):
                    nb = min(c["K"], max(0, (p - c["LB"] * c["BS"] + 1) // c["BS"]))
                    m = nb * c["BS"] + min(p + 1, c["LB"] * c["BS"])
                    keys, pairs = keys + m, pairs + m
            else:
                a, b = _visible(c, lo, hi)
                keys, pairs = keys + a, pairs + b
        return dict(bytes=keys * c["HKV"] * (2 * c["D"] + 8 / c["BS"]) + rows * g * 4, flops=4 * g * pairs)
    if kind == "reserve":
        return dict(bytes=2 * 4 * (c["R"] * c["W"] + c["N"] + c["R"]), flops=0)
    page = c["layers"] * 2 * (c["BS"] * c["H"] * c["D"] + 4 * c["H"])
    if kind == "reorder":
        moved = len(_copies(c, _pool_rows(c)))
    else:
        live = max(1, min(int(c["N"] * c["fill"]), c["R"] * c["W"]))
        moved = live * (c["N"] - live) / c["N"]                          # expected: live pages past the live count
    return dict(bytes=2 * page * moved + 2 * 4 * (c["R"] * c["W"] + c["N"] + c["R"]), flops=0)


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, page by page and request by request."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "append":
        return _exact_append(c, s)
    if c["kind"] in ("decode", "prefill", "selected"):
        return _exact_attend(c, s)
    return None                                                          # whole numbers and copies


def _exact_append(c, s):
    out = {}
    cu, start, bt = s["cu"].tolist(), s["start"].tolist(), s["bt"].tolist()
    for x, cache, scale, a, b in ((s["k"], s["kc"], s["ks"], "kc", "ks"), (s["v"], s["vc"], s["vs"], "vc", "vs")):
        qmax = QMAX[c["kv"]]
        val = cache.to(torch.float32).to(F64)
        sc = scale.to(F64)
        for r in range(c["R"]):
            pos, end = start[r], start[r] + cu[r + 1] - cu[r]
            while pos < end:
                page, o = bt[r][pos // c["BS"]], pos % c["BS"]
                n = min(c["BS"] - o, end - pos)
                y = x[cu[r] + pos - start[r]:][:n].to(F64)               # [n, H, D]
                need = torch.exp2(torch.ceil(torch.log2((y.abs().amax((0, 2)) / qmax).clamp(min=2.0 ** MIN_EXP))))
                s1 = torch.maximum(need, sc[page]) if o else need
                to8 = (lambda z: z.to(torch.float32).to(torch.float8_e4m3fn).to(torch.float32).to(F64)) \
                    if c["kv"] == "e4m3" else torch.round
                val[page, :o] = to8(val[page, :o] * (sc[page] / s1)[None, :, None])
                val[page, o:o + n] = to8(y / s1[None, :, None])
                sc[page] = s1
                pos += n
        out[a], out[b] = val, sc
    return out


def _exact_attend(c, s):
    HQ, HKV, D, BS = c["HQ"], c["HKV"], c["D"], c["BS"]
    G, scale = HQ // HKV, D ** -0.5
    lens, bt = s["sl"].tolist(), s["bt"].long()
    cu = s["cu"].tolist() if c["kind"] == "prefill" else [r * c["dql"] for r in range(c["R"] + 1)]
    o = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=F64, device="cuda")
    for r, L in enumerate(lens):
        n = cu[r + 1] - cu[r]
        if not n:
            continue
        pg = bt[r, :-(-L // BS)]
        p = torch.arange(L - n, L, device="cuda")
        j = torch.arange(L, device="cuda")
        see = j[None] <= p[:, None]
        bias = torch.zeros(n, L, dtype=F64, device="cuda")
        if c["kind"] == "selected":
            lw = c["LB"] * BS
            near = j[None] > (p - lw)[:, None]
            pick = torch.zeros(n, L, dtype=torch.bool, device="cuda")
            for i in range(n):
                for k, b in enumerate(s["ids"][0, cu[r] + i].tolist()):
                    if b >= 0:
                        pick[i, b * BS:(b + 1) * BS] = True
                        if s["bias"] is not None:
                            bias[i, b * BS:(b + 1) * BS] = s["bias"][0, cu[r] + i, k].to(F64)
            bias = bias.masked_fill(near, 0.0)
            see = see & (near | pick)
        elif c["window"]:
            see = see & ((j[None] > (p - c["window"])[:, None]) | (j[None] < c["sinks"]))
        for h in range(HKV):
            kh, vh = ((x.view(torch.int8)[pg, :, h].view(x.dtype).to(torch.float32).to(F64)
                       * y[pg, h].to(F64)[:, None, None]).reshape(-1, D)[:L] for x, y in ((s["kc"], s["ks"]),
                                                                                          (s["vc"], s["vs"])))
            for q in range(h * G, h * G + G):
                z = s["q"][cu[r]:cu[r + 1], q].to(F64) @ kh.T * scale + bias
                z = z.masked_fill(~see, -math.inf)
                o[cu[r]:cu[r + 1], q] = torch.softmax(z, -1) @ vh
                lse[cu[r]:cu[r + 1], q] = torch.logsumexp(z, -1)
    if c["kind"] == "decode":
        return dict(o=o, lse=lse) if c["lse"] else dict(o=o)
    return o
