"""Plain forms of the page operators and of chunk selection, for the tests: Python lists and 64 bits."""

import math

import torch


def fork(block, tables, lens, refs, parents, children):
    """``(tables, lens, refs, copies)`` as lists; copies: (source, fresh, slots) or (-1, -1, 0)."""
    tables, lens, refs = [list(r) for r in tables], list(lens), list(refs)
    old = (([list(r) for r in tables]), list(lens))
    free = [p for p, r in enumerate(refs) if r == 0]
    copies, named = [], set()
    for a, b in zip(parents, children):
        copy = (-1, -1, 0)
        ok = 0 <= a < len(lens) and 0 <= b < len(lens) and old[1][b] == 0 and b not in named
        if 0 <= b < len(lens) and a != -1:
            named.add(b)
        if ok:
            full, rest = divmod(old[1][a], block)
            if rest and not 0 <= old[0][a][full] < len(refs):
                ok = False
            elif rest and not free:
                ok = False
        if ok:
            row = [-1] * len(tables[b])
            for j in range(full):
                row[j] = old[0][a][j]
                refs[row[j]] += 1
            if rest:
                row[full] = free.pop(0)
                refs[row[full]] += 1
                copy = (old[0][a][full], row[full], rest)
            tables[b], lens[b] = row, old[1][a]
        copies.append(copy)
    return tables, lens, refs, copies


def release(block, tables, lens, refs, rows):
    tables, lens, refs = [list(r) for r in tables], list(lens), list(refs)
    for r in sorted(set(rows) - {-1}):
        for j in range(-(-lens[r] // block)):
            refs[tables[r][j]] = max(0, refs[tables[r][j]] - 1)
        tables[r], lens[r] = [-1] * len(tables[r]), 0
    return tables, lens, refs


def compact(tables, refs):
    """``(tables, refs, live, moves)``, moves a list of (source, destination)."""
    refs = list(refs)
    live = sum(r > 0 for r in refs)
    holes = [p for p in range(live) if refs[p] <= 0]
    moves = list(zip([p for p in range(live, len(refs)) if refs[p] > 0], holes))
    to = dict(moves)
    for s, d in moves:
        refs[d], refs[s] = refs[s], 0
    return [[to.get(p, p) for p in row] for row in tables], refs, live, moves


def key_bounds(keys, bounds, tables, starts, lens):
    """``bounds`` with the chunks of each request's tokens [start, len) made anew."""
    bounds = bounds.clone()
    block, chunk = keys.shape[1], keys.shape[1] // bounds.shape[2]
    for b, (lo, hi) in enumerate(zip(starts, lens)):
        if lo >= hi:
            continue
        for c in range(lo // chunk, -(-hi // chunk)):
            page, slot = int(tables[b][c * chunk // block]), c * chunk % block
            rows = keys[page, slot:slot + min(chunk, hi - c * chunk)]
            bounds[page, :, slot // chunk, 0] = rows.amin(0)
            bounds[page, :, slot // chunk, 1] = rows.amax(0)
    return bounds


def select_chunks(q, bounds, tables, lens, block, top):
    """int32 ``[batch, kv_heads, top]``, ascending, -1 behind the last: the maximum of q . k over
    the box between the bounds, summed over a kv head's q heads, in 64 bits."""
    batch, nq, _ = q.shape
    nkv, per = bounds.shape[1], bounds.shape[2]
    group, chunk = nq // nkv, block // per
    out = torch.full((batch, nkv, top), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        chunks = -(-n // chunk)
        pages = tables[b].long().clamp_min(0)
        for h in range(nkv):
            if chunks <= top:
                mine = list(range(chunks))
            else:
                box = bounds[pages, h].flatten(0, 1)[:chunks].double()  # [chunks, 2, dim]
                x = q[b, h * group:(h + 1) * group].double()
                s = torch.zeros(chunks, dtype=torch.float64)
                for i in range(group):
                    s += (x[i].clamp_min(0) * box[:, 1] + x[i].clamp_max(0) * box[:, 0]).sum(-1)
                s = [1.7976931348623157e308 if math.isnan(v) or v == math.inf else v for v in s.tolist()]
                s[0] = s[-1] = math.inf
                mine = sorted(sorted(range(chunks), key=lambda c, s=s: (-s[c], c))[:top])
            out[b, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
    return out


def attention(q, k, v, scale):
    """64-bit attention of q [heads, D] over k, v [T, D]: ``(out, softmax-weighted mean of |v|)``."""
    if k.shape[0] == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, z
    p = torch.softmax(q.double() @ k.double().T * scale, -1)
    return p @ v.double(), p @ v.double().abs()


def sparse_attention(q, kc, vc, tables, lens, selected, chunk, scale):
    batch, nq, dim = q.shape
    block, nkv = kc.shape[1], kc.shape[2]
    group = nq // nkv
    out = torch.zeros(batch, nq, dim, dtype=torch.float64)
    mean = torch.zeros_like(out)
    for b, n in enumerate(lens):
        for h in range(nkv):
            at = [t for c in selected[b, h].tolist() if c >= 0 for t in range(c * chunk, min(n, (c + 1) * chunk))]
            at = torch.tensor(at, dtype=torch.long)
            page = tables[b].long()[at // block] if len(at) else at
            rows = slice(h * group, (h + 1) * group)
            out[b, rows], mean[b, rows] = attention(q[b, rows], kc[page, at % block, h], vc[page, at % block, h], scale)
    return out, mean


def attention_bound(dtype, expect, mean_abs):
    """How far the tensor-core kernels may be off. With u half a step of the dtype relative to the
    value (bf16 2^-8, fp16 2^-11): each probability is rounded to the dtype before it meets its
    value (u of the weighted mean of |v|) and the result once more (u of the result, and of the
    first error). In fp32: a score is a sum of D <= 128 products, at most (D + 2) 2^-24 of
    sum |q k| scale (below 9 for the tests' normal inputs) off, below 2^-13.7; it enters numerator
    and denominator; exponentials and sums add below 2^-20: 2^-12 of the weighted mean of |v|
    covers them, and an fp16 probability below its normal range (2^-25 off, times at most 2^12
    tokens of those that share the denominator's 1) as well."""
    u = torch.finfo(dtype).eps / 2
    return u * expect.abs() + (u * (1 + u) + 2.0 ** -12) * mean_abs + 1e-30
