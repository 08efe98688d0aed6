"""Oracle of the scaled 8-bit paged cache and of the page pool: plain loops in 64
bits on the CPU, from the definitions (no counterpart in the reference).

A cache value stands for byte * scale[page, kv head].  ``append`` gives the state
after new tokens, ``attend`` the outputs, their log-sum-exp and the bound that a
kernel's roundings stay within, ``reserve`` / ``reorder`` / ``compact`` a pool's
next state."""

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
MIN_EXP = -100
F64 = torch.float64


def scale_for(a, dtype):
    """The smallest 2^e >= 2^-100 with a <= QMAX 2^e."""
    e = MIN_EXP
    while a > QMAX[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_bytes(y, dtype):
    """Values in units of the scale -> stored values (saturating, nearest even;
    NaN stays NaN in e4m3 and is 0 in int8)."""
    if dtype == torch.int8:
        return torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448.0, 448.0).float().to(dtype)


def append(x, cache, scale, table, start, runs):
    """x [total, H, D] appended to cache [pages, page, H, D] with scale [pages, H];
    table a list of page lists, start / runs per request.  New (cache, scale)."""
    cache, scale = cache.clone(), scale.clone()
    raw = cache.view(torch.int8)
    page, dt, npages = cache.shape[1], cache.dtype, cache.shape[0]
    row = 0
    for r, n in enumerate(runs):
        for b in range(start[r] // page, -(-(start[r] + n) // page) if n else 0):
            lo, hi = max(start[r], b * page), min(start[r] + n, (b + 1) * page)
            if lo >= hi or b >= len(table[r]) or not 0 <= table[r][b] < npages:
                continue
            pg, o = table[r][b], lo - b * page
            for h in range(cache.shape[2]):
                y = x[row + lo - start[r]:row + hi - start[r], h].to(F64)
                fin = y[torch.isfinite(y)]
                s = scale_for(fin.abs().max().item() if fin.numel() else 0.0, dt)
                old = scale[pg, h].item()
                if o:
                    s = max(s, old)
                    if s != old:
                        b8 = to_bytes(cache[pg, :o, h].float().to(F64) * (old / s), dt)
                        raw[pg, :o, h] = b8.view(torch.int8)
                raw[pg, o:o + hi - lo, h] = to_bytes(y / s, dt).view(torch.int8)
                scale[pg, h] = s
        row += n
    return cache, scale


def attend(q, kc, vc, ks, vs, table, cu, lens, scale, window=None, sinks=0, topk=None, bias=None):
    """q [rows, HQ, D], request r's rows cu[r] .. cu[r + 1) at the end of its
    lens[r] keys.  Returns (o, lse, tol): o, tol [rows, HQ, D], lse [rows, HQ].

    tol bounds a kernel that multiplies in q's type (K) and fp16 (P, V) and sums
    in fp32: with A = sum p |v| / sum p, every weight may be off by half an fp16
    step (2^-11), by twice the logit's error dz and by that of its V scale's
    logarithm (2^-16 for scales down to 2^-100), and the sums by n 2^-23; the
    output is rounded once more (half a step of its type)."""
    rows, HQ, D = q.shape
    HKV, page, npages = kc.shape[2], kc.shape[1], kc.shape[0]
    G = HQ // HKV
    o = torch.zeros(rows, HQ, D, dtype=F64)
    tol = torch.zeros(rows, HQ, D, dtype=F64)
    lse = torch.full((rows, HQ), -math.inf, dtype=F64)
    half = torch.finfo(q.dtype).eps / 2
    for r in range(len(lens)):
        for i in range(cu[r], cu[r + 1]):
            p = lens[r] - (cu[r + 1] - i)
            for h in range(HKV):
                at, add = [], []
                slot = {}
                if topk is not None:
                    for s, b in enumerate(topk[h, i].tolist()):
                        if b >= 0 and b not in slot:
                            slot[b] = 0.0 if bias is None else bias[h, i, s].item()
                for j in range(min(p + 1, len(table[r]) * page)):
                    if not 0 <= table[r][j // page] < npages:
                        continue
                    if topk is not None:
                        if j > p - window:
                            add.append(0.0)
                        elif j // page in slot:
                            add.append(slot[j // page])
                        else:
                            continue
                    elif window is not None and not (j > p - window or j < sinks):
                        continue
                    else:
                        add.append(0.0)
                    at.append(j)
                if not at:
                    continue
                jj = torch.tensor(at)
                pg = torch.tensor([table[r][j // page] for j in at])
                k = kc[pg, jj % page, h].float().to(F64) * ks[pg, h].to(F64)[:, None]
                v = vc[pg, jj % page, h].float().to(F64) * vs[pg, h].to(F64)[:, None]
                for g in range(h * G, (h + 1) * G):
                    x = q[i, g].to(F64)
                    z = (k * x).sum(1) * scale + torch.tensor(add, dtype=F64)
                    dz = ((k * x).abs().sum(1) * abs(scale)).max().item() * (D + 4) * 2.0 ** -24 \
                        + z.abs().max().item() * 2.0 ** -22
                    lse[i, g] = torch.logsumexp(z, 0)
                    w = torch.exp(z - lse[i, g])
                    o[i, g] = w @ v
                    a = w @ v.abs()
                    e = a * (2.0 ** -11 + 2.0 ** -16 + 2 * dz + (len(at) + 16) * 2.0 ** -23)
                    tol[i, g] = e + half * (o[i, g].abs() + e) + torch.finfo(q.dtype).tiny
    return o, lse, tol


# ------------------------------------------------------------------ page pool
def reserve(table, ref, new_lens, page):
    """(table, ref, missing) after every row has pages for its new length."""
    table, ref, missing = [list(t) for t in table], list(ref), 0
    free = [i for i, n in enumerate(ref) if n == 0]
    for r, n in enumerate(new_lens):
        for b in range(min(len(table[r]), -(-max(n, 0) // page))):
            if table[r][b] < 0:
                if free:
                    table[r][b] = free.pop(0)
                    ref[table[r][b]] = 1
                else:
                    missing += 1
    return table, ref, missing


def reorder(table, lens, ref, parents, page):
    """(table, lens, ref, missing, copies): copies a list of (source, destination)."""
    R, W, N = len(table), len(table[0]), len(ref)
    new, nlen, want, seen = [], [], [], set()
    for r, p in enumerate(parents):
        if not 0 <= p < R:
            new.append([-1] * W)
            nlen.append(0)
            continue
        nlen.append(lens[p])
        full = max(lens[p], 0) // page
        if p not in seen:
            seen.add(p)
            new.append(list(table[p]))
        else:
            new.append([x if b < full else -1 for b, x in enumerate(table[p])])
            if max(lens[p], 0) % page and full < W and 0 <= table[p][full] < N:
                want.append((r, full, table[p][full]))
    ref = list(ref)
    for rows, d in ((table, -1), (new, 1)):
        for row in rows:
            for x in row:
                if 0 <= x < N:
                    ref[x] += d
    free, missing, copies = [i for i, n in enumerate(ref) if n == 0], 0, []
    for r, b, src in want:
        if free:
            new[r][b] = free.pop(0)
            ref[new[r][b]] = 1
            copies.append((src, new[r][b]))
        else:
            missing += 1
    return new, nlen, ref, missing, copies


def compact(table, ref):
    """(table, ref, n, moves): moves a list of (source, destination)."""
    n = sum(x > 0 for x in ref)
    holes = [i for i in range(n) if ref[i] <= 0]
    movers = [i for i in range(n, len(ref)) if ref[i] > 0]
    to = dict(zip(movers, holes))
    new = list(ref)
    for s, d in to.items():
        new[d], new[s] = ref[s], 0
    return [[to.get(x, x) for x in row] for row in table], new, n, list(to.items())
