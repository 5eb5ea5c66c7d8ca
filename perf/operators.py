"""The paged-cache operators on the work they meet in serving: cases, inputs, plain forms.

Three families around one paged KV cache ([blocks, block_size, kv_heads, head_dim], 256-token
blocks in the models this package serves):

* pages: copying pages, forking a sequence (full pages shared, the partly filled one copied) and
  releasing the sequences a beam step drops, and compacting the live pages to the front;
* prefix: decode attention of a batch whose groups share their first tokens' pages, the shared part
  computed once for a group;
* sparse: decode attention over the chunks of a context that a cheap upper bound of the scores
  selects, and the per-chunk key bounds that it reads.

``run`` computes the plain form in elementary torch operations where ``own`` is false and calls
``nano_vllm_multimodal_b200.ops`` where it is true; ``exact`` is a 64-bit form written apart.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 1.7976931348623157e308  # infinite and NaN chunk scores count as the largest finite one


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one layer's two planes, a handful of pages: a copy-on-write step, where latency is all
        dict(name="copy_few", op="copy", dtype="bf16", planes=2, blocks=96, block=16, nkv=8, dim=128, pairs=8),
        # parallel sampling: 8 prompts forked into 48 sequences over all planes of a 28-layer cache, 16 dropped
        dict(name="fork_beam", op="fork", dtype="bf16", planes=56, blocks=150, block=256, nkv=8, dim=128, parents=8,
             children=48, dropped=16, context=2048),
        # a cache at half load compacted before its top half is handed back
        dict(name="compact_half", op="compact", dtype="bf16", planes=56, blocks=144, block=256, nkv=8, dim=128,
             live=0.5, rows=24),
        # four samples of one short prompt: the smallest call
        dict(name="prefix_few", op="prefix", dtype="bf16", groups=1, batch=4, nq=16, nkv=8, dim=128, block=256,
             prefix=512, suffix=64),
        # a serving batch behind one system prompt
        dict(name="prefix_batch", op="prefix", dtype="bf16", groups=1, batch=64, nq=16, nkv=8, dim=128, block=256,
             prefix=8192, suffix=1024),
        # several tenants' prompts of their own lengths, half-width heads, small pages, odd sizes
        dict(name="prefix_tenants", op="prefix", dtype="fp16", groups=7, batch=93, nq=14, nkv=2, dim=64, block=32,
             prefix=4090, suffix=333),
        # a long document asked many questions at once: compute-bound
        dict(name="prefix_document", op="prefix", dtype="bf16", groups=1, batch=256, nq=16, nkv=2, dim=128, block=256,
             prefix=32768, suffix=512),
        # one request over a short context: the smallest call
        dict(name="sparse_one", op="sparse", dtype="bf16", batch=1, nq=16, nkv=8, dim=128, block=256, chunk=32,
             context=4000, top=32),
        # half-width heads, small pages, odd sizes
        dict(name="sparse_odd", op="sparse", dtype="fp16", batch=19, nq=14, nkv=2, dim=64, block=64, chunk=16,
             context=20011, top=77),
        # a long-context decode batch
        dict(name="sparse_long", op="sparse", dtype="bf16", batch=48, nq=16, nkv=8, dim=128, block=256, chunk=32,
             context=32768, top=64),
        # each decode step's newest key folded into its chunk's bounds
        dict(name="bounds_step", op="bounds", dtype="bf16", batch=256, nkv=8, dim=128, block=256, chunk=32,
             context=1000, new=1),
        # prefill's keys
        dict(name="bounds_prefill", op="bounds", dtype="bf16", batch=16, nkv=8, dim=128, block=256, chunk=32,
             context=16384, new=16384),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["copy", "fork", "compact", "prefix", "prefix", "sparse", "sparse", "bounds"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    nq, nkv, dim = rng.choice([(16, 8, 128), (16, 2, 128), (32, 8, 128), (8, 8, 128), (14, 2, 64), (16, 1, 64)])
    block = rng.choice([16, 32, 64, 128, 256, 256])
    if op in ("copy", "fork", "compact"):
        planes = rng.choice([2, 8, 24, 56])
        page = planes * block * nkv * dim * 2
        most = max(12, min(4096, int(2.0e9 / page)))  # pages of a cache of at most 2 GB
        blocks = _log_int(rng, 12, most)
        base = dict(op=op, dtype=dtype, planes=planes, blocks=blocks, block=block, nkv=nkv, dim=dim)
        if op == "copy":
            return dict(base, pairs=_log_int(rng, 1, blocks // 2))
        if op == "compact":
            return dict(base, live=round(rng.uniform(0.1, 0.9), 3), rows=_log_int(rng, 1, 64))
        children = _log_int(rng, 1, blocks // 3)
        parents = rng.randint(1, min(8, children))
        width = max(1, (blocks - children) // parents)
        return dict(base, parents=parents, children=children, dropped=rng.randint(0, children // 2),
                    context=rng.randint(1, width * block - 1))
    if op == "prefix":
        prefix, suffix = _log_int(rng, 1, 40000), _log_int(rng, 1, 1500)
        batch = _log_int(rng, 1, max(1, min(300, int(1.6e7 / ((prefix + suffix + block) * nkv)))))
        return dict(op=op, dtype=dtype, groups=rng.randint(1, min(batch, 6)), batch=batch, nq=nq, nkv=nkv, dim=dim,
                    block=block, prefix=prefix, suffix=suffix)
    chunk = rng.choice([c for c in (16, 32, 64) if c <= block])
    if op == "sparse":
        context = _log_int(rng, 1, 60000)
        batch = _log_int(rng, 1, max(1, min(128, int(1.2e7 / ((context + block) * nkv)))))
        return dict(op=op, dtype=dtype, batch=batch, nq=nq, nkv=nkv, dim=dim, block=block, chunk=chunk,
                    context=context, top=_log_int(rng, 2, 160))
    context = _log_int(rng, 1, 16384)
    batch = _log_int(rng, 1, max(1, min(256, int(2.0e6 / ((context + block) * nkv)))))
    return dict(op=op, dtype=dtype, batch=batch, nkv=nkv, dim=dim, block=block, chunk=chunk, context=context,
                new=rng.choice([1, _log_int(rng, 1, context)]))


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _ints(g, lo, hi, shape):
    """Uniform whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def _prepare_pages(case, g):
    s = {"case": case}
    blocks, block = case["blocks"], case["block"]
    s["cache"] = _normal(g, (case["planes"], blocks, block, case["nkv"], case["dim"]), DTYPES[case["dtype"]])
    order = _perm(g, blocks)
    if case["op"] == "copy":
        s["src"], s["dst"] = order[: case["pairs"]].contiguous(), order[case["pairs"]: 2 * case["pairs"]].contiguous()
        return s
    s["refs"] = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    if case["op"] == "compact":
        n = max(1, min(blocks, round(case["live"] * blocks)))
        width = -(-n // case["rows"])
        tables = torch.full((case["rows"] * width,), -1, dtype=torch.int32, device="cuda")
        tables[:n] = order[:n]
        s["tables"] = tables.view(case["rows"], width).contiguous()
        s["refs"][order[:n].long()] = 1
        return s
    # the parents' rows hold their pages, the children's are empty
    parents, children = case["parents"], case["children"]
    width = -(-case["context"] // block)
    rows = parents + children
    tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    held = _ints(g, max(1, case["context"] // 2), case["context"], (parents,))
    lens[:parents] = held
    pages = order[: parents * width].view(parents, width)
    used = torch.arange(width, device="cuda") * block < held[:, None]
    tables[:parents] = torch.where(used, pages, -1)
    s["refs"][pages[used].long()] = 1
    s["tables"], s["lens"] = tables, lens
    s["parents"] = (torch.arange(children, device="cuda") % parents).to(torch.int32)
    s["children"] = (parents + _perm(g, children)).to(torch.int32)
    s["dropped"] = s["children"][: case["dropped"]].contiguous()
    return s


def _cache(case, g, blocks):
    """Keys that drift from page to page, and values."""
    shape = (blocks, case["block"], case["nkv"], case["dim"])
    keys = _normal(g, shape, DTYPES[case["dtype"]])
    keys += 0.5 * _normal(g, (blocks, 1) + shape[2:], DTYPES[case["dtype"]])
    return keys


def _prepare_prefix(case, g):
    batch, groups, block = case["batch"], case["groups"], case["block"]
    cuts = torch.sort(torch.randperm(batch - 1, generator=g, device="cuda")[: groups - 1] + 1).values if groups > 1 else \
        torch.empty(0, dtype=torch.int64, device="cuda")
    offsets = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), batch)]).to(torch.int32)
    # one group: the prefix of the case; several: lengths of their own up to it
    prefix = _ints(g, max(1, case["prefix"] // 2), case["prefix"], (groups,))
    prefix[groups - 1] = case["prefix"]
    whole, tail = case["prefix"] // block, -(-(case["suffix"] + block - 1) // block)
    pages = groups * whole + batch * tail
    keys = _cache(case, g, pages)
    values = _normal(g, keys.shape, keys.dtype)
    order = _perm(g, pages)
    group_of = torch.searchsorted(offsets[1:].contiguous(), torch.arange(batch, device="cuda", dtype=torch.int32), right=True)
    shared = order[: groups * whole].view(groups, whole)[group_of]
    mine = order[groups * whole:].view(batch, tail)
    # whole pages are shared; from the page in which the prefix ends on, each request has pages of its own
    used = (prefix // block)[group_of][:, None]
    col = torch.arange(whole + tail, device="cuda")[None, :]
    own_page = mine.gather(1, (col - used).clamp(0, tail - 1))
    tables = torch.where(col < used, torch.cat([shared, mine], 1), own_page)
    tables = torch.where(col < used + tail, tables, -1).to(torch.int32)
    # a fork has copied the prefix's last tokens into them
    first = tables.gather(1, used)[:, 0].long()
    leader = first[offsets[:-1].long()][group_of]
    part = torch.arange(block, device="cuda") < (prefix % block)[group_of][:, None]
    part = part[..., None, None]
    keys[first] = torch.where(part, keys[leader], keys[first])
    values[first] = torch.where(part, values[leader], values[first])
    lens = prefix[group_of] + _ints(g, 1, case["suffix"], (batch,))
    return {"case": case, "q": _normal(g, (batch, case["nq"], case["dim"]), keys.dtype), "keys": keys, "values": values,
            "tables": tables.contiguous(), "lens": lens.to(torch.int32), "offsets": offsets, "prefix": prefix,
            "scale": case["dim"] ** -0.5, "max_prefix": case["prefix"], "max_context": case["prefix"] + case["suffix"]}


def _prepare_chunks(case, g):
    batch, block, chunk = case["batch"], case["block"], case["chunk"]
    width = -(-case["context"] // block)
    keys = _cache(case, g, batch * width)
    tables = _perm(g, batch * width).view(batch, width).contiguous()
    lens = _ints(g, max(1, case["context"] - case["context"] // 4), case["context"], (batch,))
    s = {"case": case, "keys": keys, "tables": tables, "lens": lens}
    by_chunk = keys.view(batch * width, block // chunk, chunk, case["nkv"], case["dim"])
    if case["op"] == "bounds":
        s["start"] = (lens - case["new"]).clamp_min(0)
        s["bounds"] = torch.zeros(batch * width, case["nkv"], block // chunk, 2, case["dim"], dtype=keys.dtype, device="cuda")
        s["new"] = case["new"]
        return s
    # the bounds that a program has kept as it went
    bounds = torch.stack([by_chunk.amin(2), by_chunk.amax(2)], 2)  # [pages, chunks, 2, heads, dim]
    s["bounds"] = bounds.permute(0, 3, 1, 2, 4).contiguous()
    s["values"] = _normal(g, keys.shape, keys.dtype)
    s["q"] = _normal(g, (batch, case["nq"], case["dim"]), keys.dtype)
    s["scale"], s["top"] = case["dim"] ** -0.5, case["top"]
    s["max_context"] = case["context"]
    return s


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] in ("copy", "fork", "compact"):
        return _prepare_pages(case, g)
    if case["op"] == "prefix":
        return _prepare_prefix(case, g)
    return _prepare_chunks(case, g)


# ---------------------------------------------------------------- plain forms

def _copy_plain(s):
    cache = s["cache"]
    cache[:, s["dst"].long()] = cache[:, s["src"].long()]
    return {"cache": cache}


def _free_plain(tables, lens, refs, rows, block):
    rows = rows.long()
    held = torch.arange(tables.shape[1], device=tables.device) * block < lens[rows][:, None]
    at = torch.where(held, tables[rows], refs.numel()).reshape(-1).long()
    less = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=refs.device).scatter_add(0, at, torch.ones_like(at, dtype=torch.int32))
    tables, lens = tables.clone(), lens.clone()
    tables[rows] = -1
    lens[rows] = 0
    return tables, lens, refs - less[:-1]


def _fork_plain(s):
    cache, tables, lens, refs = s["cache"], s["tables"], s["lens"], s["refs"]
    block, pages = cache.shape[2], cache.shape[1]
    parents, children = s["parents"].long(), s["children"].long()
    held, rows = lens[parents], tables[parents]
    full, rest = held // block, held % block
    part = rest > 0
    col = torch.arange(tables.shape[1], device=tables.device)
    shared = col < full[:, None]
    order = torch.argsort((refs > 0).to(torch.int32), stable=True)  # free pages first, ascending
    fresh = order[(torch.cumsum(part.to(torch.int64), 0) - 1).clamp_min(0)]
    child = torch.where(shared, rows, torch.where(part[:, None] & (col == full[:, None]), fresh[:, None].to(torch.int32), -1))
    out_tables, out_lens = tables.clone(), lens.clone()
    out_tables[children] = child
    out_lens[children] = held
    at = torch.where(child >= 0, child, pages).reshape(-1).long()
    more = torch.zeros(pages + 1, dtype=torch.int32, device=refs.device).scatter_add(0, at, torch.ones_like(at, dtype=torch.int32))
    out_refs = refs + more[:-1]
    # the filled slots of each partly filled page; a whole page's copy is the page onto itself
    last = rows.gather(1, full.clamp_max(tables.shape[1] - 1).long()[:, None])[:, 0].long()
    own_page = rows[:, 0].long()
    src, dst = torch.where(part, last, own_page), torch.where(part, fresh, own_page)
    slots = torch.arange(block, device=cache.device)[None, None, :, None, None] < torch.where(part, rest, block)[None, :, None, None, None]
    cache[:, dst] = torch.where(slots, cache[:, src], cache[:, dst])
    out = _free_plain(out_tables, out_lens, out_refs, s["dropped"], block)
    return {"cache": cache, "forked_tables": out_tables, "forked_lens": out_lens, "forked_refs": out_refs,
            "tables": out[0], "lens": out[1], "refs": out[2]}


def _compact_plain(s):
    cache, tables, refs = s["cache"], s["tables"], s["refs"]
    pages, most = refs.numel(), refs.numel() // 2
    live = refs > 0
    n = live.sum()
    page = torch.arange(pages, device=refs.device)
    hole, far = ~live & (page < n), live & (page >= n)
    dst = torch.argsort((~hole).to(torch.int32), stable=True)[:most]
    src = torch.argsort(torch.where(far, 0, torch.where(hole, 2, 1)), stable=True)[:most]
    move = torch.arange(most, device=refs.device) < far.sum()
    to = torch.where(move, dst, src)  # without a move: the page onto itself
    cache[:, to] = cache[:, src]
    remap = page.clone()
    remap[src] = to
    out_refs = refs.clone()
    out_refs[src] = torch.where(move, 0, refs[src])
    out_refs[to] = refs[src]
    out_tables = torch.where(tables >= 0, remap[tables.clamp_min(0).long()].to(torch.int32), tables)
    return {"cache": cache, "tables": out_tables, "refs": out_refs, "live": n.to(torch.int32).reshape(1)}


def _softmax(x):
    """Over the last axis; a row of nothing but -inf gives zeros."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _attend(q, k, v, keep, scale):
    """q [B, heads, D] over k, v [B, kv heads, T, D] where keep [B, 1 or kv heads, T]."""
    batch, nq, dim = q.shape
    nkv = k.shape[1]
    x = q.float().view(batch, nkv, nq // nkv, dim) @ k.float().transpose(-1, -2) * scale
    p = _softmax(torch.where(keep[:, :, None, :], x, -math.inf))
    return (p @ v.float()).reshape(batch, nq, dim).to(q.dtype)


def _prefix_plain(s):
    tables, keys = s["tables"].clamp_min(0).long(), s["keys"]
    k = keys[tables].flatten(1, 2).transpose(1, 2)
    v = s["values"][tables].flatten(1, 2).transpose(1, 2)
    keep = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None]
    return {"out": _attend(s["q"], k, v, keep[:, None], s["scale"])}


def _select_plain(s):
    q, bounds, lens, tables = s["q"], s["bounds"], s["lens"], s["tables"].long()
    pages, nkv, per, _, dim = bounds.shape
    batch, chunk = q.shape[0], s["keys"].shape[1] // per
    by_head = q.double().view(batch, nkv, -1, dim)
    up, down = by_head.clamp_min(0).sum(2), by_head.clamp_max(0).sum(2)
    b = bounds[tables].transpose(1, 2).flatten(2, 3)  # [batch, heads, chunks, 2, dim]
    score = (b[..., 1, :].double() * up[:, :, None] + b[..., 0, :].double() * down[:, :, None]).sum(-1)
    score = torch.where(torch.isnan(score), LARGEST, score).clamp_max(LARGEST)
    n = (lens + chunk - 1) // chunk
    at = torch.arange(score.shape[-1], device=q.device)
    forced = (at == 0) | (at == n[:, None] - 1)
    inside = at < n[:, None]
    score = torch.where(forced[:, None], math.inf, score)
    first = torch.argsort(torch.where(inside[:, None], -score, math.inf), dim=-1, stable=True)[..., : s["top"]]
    if first.shape[-1] < s["top"]:
        first = torch.nn.functional.pad(first, (0, s["top"] - first.shape[-1]), value=score.shape[-1])
    chosen = torch.where(first < n[:, None, None], first, 1 << 30).sort(-1).values
    return torch.where(chosen < 1 << 30, chosen, -1).to(torch.int32)


def _sparse_plain(s):
    keys, chunk = s["keys"], s["keys"].shape[1] // s["bounds"].shape[2]
    chosen = _select_plain(s)
    batch, nkv, top = chosen.shape
    token = (chosen.clamp_min(0)[..., None] * chunk + torch.arange(chunk, device=chosen.device)).flatten(2)
    keep = (chosen >= 0).repeat_interleave(chunk, -1) & (token < s["lens"][:, None, None])
    token = torch.where(keep, token, 0).long()
    page = s["tables"].long().gather(1, (token // keys.shape[1]).flatten(1)).view_as(token)
    head = torch.arange(nkv, device=chosen.device)[None, :, None]
    slot = token % keys.shape[1]
    out = _attend(s["q"], keys[page, slot, head], s["values"][page, slot, head], keep, s["scale"])
    return {"out": out, "selected": chosen}


def _bounds_plain(s):
    keys, bounds, tables, lens = s["keys"], s["bounds"], s["tables"].long(), s["lens"].long()
    pages, nkv, per, _, dim = bounds.shape
    block = keys.shape[1]
    chunk = block // per
    first = s["start"].long() // chunk
    at = first[:, None] + torch.arange((s["new"] - 1) // chunk + 2, device=keys.device)
    at = torch.where(at * chunk < lens[:, None], at, first[:, None])  # behind the last: the first once more
    token = at[..., None] * chunk + torch.arange(chunk, device=keys.device)
    page = tables.gather(1, at * chunk // block)
    rows = keys[page[..., None], token % block]  # [batch, chunks, chunk, heads, dim]
    inside = (token < lens[:, None, None])[..., None, None]
    low = torch.where(inside, rows, math.inf).amin(2)
    high = torch.where(inside, rows, -math.inf).amax(2)
    bounds[page, :, at % per] = torch.stack([low, high], 3)
    return {"bounds": bounds}


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    from nano_vllm_multimodal_b200 import ops
    op = s["case"]["op"]
    if op == "copy":
        ops.paged_copy_blocks(s["cache"], s["src"], s["dst"])
        return {"cache": s["cache"]}
    if op == "fork":
        tables, lens, refs, _ = ops.paged_fork(s["cache"], s["tables"], s["lens"], s["refs"], s["parents"], s["children"])
        out = ops.paged_free(tables, lens, refs, s["dropped"], s["cache"].shape[2])
        return {"cache": s["cache"], "forked_tables": tables, "forked_lens": lens, "forked_refs": refs,
                "tables": out[0], "lens": out[1], "refs": out[2]}
    if op == "compact":
        tables, refs, live, _ = ops.paged_compact(s["cache"], s["tables"], s["refs"])
        return {"cache": s["cache"], "tables": tables, "refs": refs, "live": live}
    if op == "prefix":
        return {"out": ops.shared_prefix_decode_attention(
            s["q"], s["keys"], s["values"], s["lens"], s["tables"], s["offsets"], s["prefix"], s["scale"],
            max_prefix_len=s["max_prefix"], max_context_len=s["max_context"])}
    if op == "sparse":
        out, selected = ops.sparse_decode_attention(s["q"], s["keys"], s["values"], s["bounds"], s["lens"], s["tables"],
                                                    s["scale"], s["top"], max_context_len=s["max_context"])
        return {"out": out, "selected": selected}
    return {"bounds": ops.paged_key_bounds_(s["bounds"], s["keys"], s["tables"], s["start"], s["lens"], s["new"])}


def run(state):
    if own:
        return _own(state)
    return {"copy": _copy_plain, "fork": _fork_plain, "compact": _compact_plain, "prefix": _prefix_plain,
            "sparse": _sparse_plain, "bounds": _bounds_plain}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    row = case["nkv"] * case["dim"] * size
    if op in ("copy", "fork", "compact"):
        page = case["planes"] * case["block"] * row
        if op == "copy":
            return {"bytes": 2.0 * case["pairs"] * page + 8 * case["pairs"], "flops": 0.0}
        if op == "fork":  # a forked page is half full in the mean
            rows, width = case["parents"] + case["children"], -(-case["context"] // case["block"])
            return {"bytes": case["children"] * page * 1.0 + 4.0 * (5 * rows * width + 5 * case["blocks"]), "flops": 0.0}
        live = max(1, min(case["blocks"], round(case["live"] * case["blocks"])))
        moved = live * (1 - live / case["blocks"])  # live pages that lie behind the first `live` places, in the mean
        return {"bytes": 2.0 * moved * page + 8.0 * (case["blocks"] + live), "flops": 0.0}
    if op == "prefix":
        batch, groups = case["batch"], case["groups"]
        prefix = case["prefix"] * (1 + 0.75 * (groups - 1)) / groups  # of a group, in the mean
        own_tokens = batch * (case["suffix"] + 1) / 2
        rows = batch * case["nq"] * case["dim"]
        return {"bytes": 2 * row * (groups * prefix + own_tokens) + 2.0 * rows * size + 4.0 * batch * (prefix + case["suffix"]) / case["block"],
                "flops": 4.0 * rows * (prefix + (case["suffix"] + 1) / 2)}
    tokens = case["batch"] * case["context"] * 0.875
    if op == "sparse":
        read = min(tokens, case["batch"] * case["top"] * case["chunk"])
        chunks = tokens / case["chunk"]
        rows = case["batch"] * case["nq"] * case["dim"]
        return {"bytes": 2 * row * (chunks + read) + 2.0 * rows * size + 4.0 * case["batch"] * case["nkv"] * case["top"],
                "flops": 4.0 * rows / case["batch"] * read + 4.0 * chunks * case["nkv"] * case["dim"]}
    # the newest tokens' chunks: the first of them begins before the new tokens
    read = case["batch"] * min(case["context"] * 0.875, case["new"] + (case["chunk"] - 1) / 2)
    chunks = case["batch"] * math.ceil(read / case["batch"] / case["chunk"])
    return {"bytes": row * (read + 2.0 * chunks), "flops": 2.0 * read * case["nkv"] * case["dim"]}


# ---------------------------------------------------------------- 64-bit forms

def exact(case, seed):
    def pages_by_hand(s):
        cache, op = s["cache"], s["case"]["op"]
        if op == "copy":
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                cache[:, b] = cache[:, a]
            return {"cache": cache}
        refs = s["refs"].tolist()
        tables = s["tables"].tolist()
        as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        if op == "compact":
            live = sum(r > 0 for r in refs)
            holes = [p for p in range(live) if refs[p] == 0]
            moved = {}
            for p in range(live, len(refs)):
                if refs[p] > 0:
                    to = holes[len(moved)]
                    moved[p] = to
                    cache[:, to] = cache[:, p]
                    refs[to], refs[p] = refs[p], 0
            tables = [[moved.get(p, p) for p in row] for row in tables]
            return {"cache": cache, "tables": as_ints(tables), "refs": as_ints(refs), "live": as_ints([live])}
        block, lens = cache.shape[2], s["lens"].tolist()
        free = [p for p, r in enumerate(refs) if r == 0]
        for a, b in zip(s["parents"].tolist(), s["children"].tolist()):
            full, rest = divmod(lens[a], block)
            row = [-1] * len(tables[a])
            for j in range(full):
                row[j] = tables[a][j]
                refs[row[j]] += 1
            if rest:
                row[full] = free.pop(0)
                refs[row[full]] = 1
                cache[:, row[full], :rest] = cache[:, tables[a][full], :rest]
            tables[b], lens[b] = row, lens[a]
        forked = {"forked_tables": as_ints(tables), "forked_lens": as_ints(lens), "forked_refs": as_ints(refs)}
        for b in s["dropped"].tolist():
            for j in range(-(-lens[b] // block)):
                refs[tables[b][j]] -= 1
            tables[b], lens[b] = [-1] * len(tables[b]), 0
        return dict(forked, cache=cache, tables=as_ints(tables), lens=as_ints(lens), refs=as_ints(refs))

    def attention_64(q, k, v, scale):
        """One request, in 64 bits: q [heads, D], k and v [T, D] of each kv head."""
        per = q.shape[0] // len(k)
        rows = []
        for h in range(q.shape[0]):
            x = torch.mv(k[h // per].double(), q[h].double()) * scale
            rows.append(torch.mv(v[h // per].double().t(), torch.softmax(x, 0)))
        return torch.stack(rows)

    s = prepare(case, seed)
    op, block = case["op"], case["block"]
    if op in ("copy", "fork", "compact"):
        return pages_by_hand(s)
    lens, keys = s["lens"].tolist(), s["keys"]
    if op == "bounds":
        bounds, chunk = s["bounds"], case["chunk"]
        for b, (lo, hi) in enumerate(zip(s["start"].tolist(), lens)):
            pages = s["tables"][b].tolist()
            for c in range(lo // chunk, -(-hi // chunk)):
                page, slot = pages[c * chunk // block], c * chunk % block
                rows = keys[page, slot: slot + min(chunk, hi - c * chunk)]
                bounds[page, :, slot // chunk, 0] = rows.amin(0)
                bounds[page, :, slot // chunk, 1] = rows.amax(0)
        return {"bounds": bounds}
    if case["batch"] * case["nq"] > 4200:
        return None
    outs, picked = [], []
    for b, n in enumerate(lens):
        pages = s["tables"][b, : -(-n // block)].long()
        k = keys[pages].flatten(0, 1)[:n].transpose(0, 1)
        v = s["values"][pages].flatten(0, 1)[:n].transpose(0, 1)
        if op == "prefix":
            outs.append(attention_64(s["q"][b], list(k), list(v), s["scale"]))
            continue
        chunk, per = case["chunk"], case["nq"] // case["nkv"]
        chunks = -(-n // chunk)
        low_high = s["bounds"][pages].transpose(0, 1).flatten(1, 2)[:, :chunks].double()
        some_k, some_v = [], []
        for h in range(case["nkv"]):
            q = s["q"][b, h * per: (h + 1) * per].double()
            # the largest q . x over all x between the bounds, summed over the heads
            score = torch.maximum(q[:, None] * low_high[h, None, :, 0], q[:, None] * low_high[h, None, :, 1]).sum((0, 2))
            score[0] = score[-1] = math.inf
            ranked = sorted(range(chunks), key=lambda c, x=score.tolist(): (-x[c], c))
            mine = sorted(ranked[: case["top"]])
            picked.append(mine + [-1] * (case["top"] - len(mine)))
            at = [t for c in mine for t in range(c * chunk, min(n, (c + 1) * chunk))]
            at = torch.tensor(at, device="cuda")
            some_k.append(k[h][at])
            some_v.append(v[h][at])
        outs.append(attention_64(s["q"][b], some_k, some_v, s["scale"]))
    out = {"out": torch.stack(outs)}
    if op == "sparse":
        out["selected"] = torch.tensor(picked, dtype=torch.int32, device="cuda").view(case["batch"], case["nkv"], case["top"])
    return out
