"""Shared-prefix decode attention (``nib_shared_prefix_decode_attention``) against the 64-bit
oracle of the dense decode attention over each request's own table (``oracle.paged_decode_attention``):
sharing changes what is read, not the result. Bounds: ``tests/_cache_forms.attention_bound``."""

import pytest
import torch

import oracle as O
from nano_vllm_multimodal_b200 import ops
from nano_vllm_multimodal_b200.layers.attention import shared_prefix_attention
from tests import _cache_forms as F

pytestmark = pytest.mark.gpu


def _case(seed, nq, nkv, dim, block, groups, alone=(), dtype=torch.bfloat16, poison=True):
    """``groups``: (prefix, [tokens behind it of each request]); ``alone``: lengths of requests
    behind the last group. Whole prefix pages are shared, a partly filled one is copied into each
    request's own page, every slot behind a context holds NaN."""
    g = torch.Generator().manual_seed(seed)
    reqs = [(p, p + s) for p, own in groups for s in own] + [(0, n) for n in alone]
    width = max(1, max(-(-n // block) for _, n in reqs))
    pages = sum(max(1, -(-n // block)) for _, n in reqs) + len(groups) * width + 3
    order = torch.randperm(pages, generator=g).tolist()
    kc = torch.randn(pages, block, nkv, dim, generator=g).to(dtype)
    vc = torch.randn(pages, block, nkv, dim, generator=g).to(dtype)
    tables = torch.full((len(reqs), width), -1, dtype=torch.int32)
    lens, offsets, prefix, at = [], [0], [], 0
    for p, own in groups:
        shared = [order.pop() for _ in range(-(-p // block))]
        for s in own:
            n = p + s
            for j in range(-(-n // block)):
                if j < p // block:
                    tables[at, j] = shared[j]
                else:
                    tables[at, j] = order.pop()
                    if j == p // block and p % block:
                        kc[tables[at, j], :p % block] = kc[shared[j], :p % block]
                        vc[tables[at, j], :p % block] = vc[shared[j], :p % block]
            lens.append(n)
            at += 1
        offsets.append(at)
        prefix.append(p)
    for n in alone:
        for j in range(-(-n // block)):
            tables[at, j] = order.pop()
        lens.append(n)
        at += 1
    if poison:
        for b, n in enumerate(lens):
            if n % block:
                kc[tables[b, n // block], n % block:] = float("nan")
                vc[tables[b, n // block], n % block:] = float("nan")
        for page in order:
            kc[page], vc[page] = float("nan"), float("inf")
    q = torch.randn(len(reqs), nq, dim, generator=g).to(dtype)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return dict(q=q, kc=kc, vc=vc, lens=i32(lens), tables=tables, offsets=i32(offsets), prefix=i32(prefix),
                scale=dim ** -0.5)


def _call(c, **hints):
    return ops.shared_prefix_decode_attention(c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), c["lens"].cuda(),
                                              c["tables"].cuda(), c["offsets"].cuda(), c["prefix"].cuda(), c["scale"], **hints)


def _check(c, out, what=""):
    args = (c["q"], c["kc"], c["vc"], c["lens"], c["tables"], c["scale"])
    e, mean = O.paged_decode_attention(*args).double(), O.paged_decode_attention_abs(*args).double()
    off = (out.cpu().double() - e).abs()
    bound = F.attention_bound(c["q"].dtype, e, mean)
    assert out.dtype == c["q"].dtype and out.shape == c["q"].shape
    assert bool((off <= bound).all()), f"{what}: {int((~(off <= bound)).sum())} off, at most {float((off / bound).max()):.2f} of the bound"


HEADS = [(16, 8, 128), (16, 2, 128), (8, 8, 64), (14, 2, 64), (16, 1, 128)]


@pytest.mark.parametrize("nq,nkv,dim", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block,groups,alone", [
    (16, [(1, [0])], []),                                            # a prefix of one token and nothing behind it
    (16, [(48, [1, 2, 300])], []),
    (256, [(700, [1, 90, 256, 0, 513])], [1, 300]),                  # ends inside a page; two requests without a group
    (32, [(64, [5] * 40), (0, [7, 40]), (97, [1]), (333, [0] * 9)], [64]),  # an empty prefix, a group of one
    (64, [(129, list(range(0, 70)))], []),                           # many rows: several row tiles, a ragged last one
])
def test_matches_the_dense_oracle(nq, nkv, dim, dtype, block, groups, alone):
    c = _case(nq * 7 + nkv + block, nq, nkv, dim, block, groups, alone, dtype)
    out = _call(c)
    _check(c, out, f"{nq}/{nkv} D{dim} block {block}")
    longest = int(c["lens"].max())
    hinted = _call(c, max_prefix_len=max(1, int(c["prefix"].max())), max_context_len=longest)
    _check(c, hinted, "with bounds")
    assert torch.equal(out, _call(c)), "the same bits twice"
    for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
        _check(c, _call(c, variant=variant), f"variant {variant}")


def test_long_prefix_and_many_splits():
    c = _case(5, 16, 8, 128, 256, [(20000, [3, 700]), (9001, [1])], [], poison=False)
    for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
        _check(c, _call(c, max_prefix_len=20000, max_context_len=20700, variant=variant))


@pytest.mark.parametrize("nq,nkv,requests", [(16, 8, 64), (16, 2, 40)])
def test_repeated_calls_give_the_same_bits(nq, nkv, requests):
    """Tiles land in any order when the cache comes from memory: one CTA's long run of tiles, for 128
    rows (two streams of the same rows) and for more, repeated behind other traffic. Hints below the
    prefix's length leave each CTA more tiles."""
    c = _case(requests, nq, nkv, 128, 64, [(12000, [i % 7 for i in range(requests)])], [], poison=False)
    cu = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}
    other = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for hint in (12000, 3000, 500):
        first = None
        for i in range(15):
            if i % 3:
                other.fill_(i)
            out = ops.shared_prefix_decode_attention(*(cu[k] for k in ("q", "kc", "vc", "lens", "tables", "offsets", "prefix")),
                                                     c["scale"], max_prefix_len=hint, variant=ops.PREFIX_ROWS256)
            first = out if first is None else first
            assert torch.equal(out, first), (hint, i)
        _check(c, first, f"hint {hint}")


@pytest.mark.parametrize("requests", [130, 300])
def test_many_requests(requests):
    c = _case(requests, 16, 2, 128, 64, [(1500, [i % 50 for i in range(requests)])], [])
    for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
        _check(c, _call(c, max_prefix_len=1500, max_context_len=1550, variant=variant))


def test_short_and_empty_requests_in_a_group():
    """Requests that are shorter than their group's prefix, a padded batch's empty ones among
    them, are computed by themselves; the first long enough one names the prefix's pages."""
    c = _case(8, 16, 8, 128, 16, [(100, [4, 9, 30, 0])], [20])
    c["lens"][0], c["lens"][2] = 0, 37
    c["tables"][0] = -1
    out = _call(c)
    _check(c, out)
    assert not out[0].any()
    c["lens"][1], c["lens"][3] = 99, 1  # nobody holds the whole prefix
    c["kc"], c["vc"] = c["kc"].nan_to_num(1.0), c["vc"].nan_to_num(1.0)
    _check(c, _call(c))


def test_hints_below_the_lengths_and_no_groups():
    c = _case(9, 16, 8, 128, 32, [(300, [40, 1, 7])], [90])
    _check(c, _call(c, max_prefix_len=10, max_context_len=20), "hints only choose the split")
    c["offsets"], c["prefix"] = torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    _check(c, _call(c), "no groups")


def test_values_of_one_sign_and_extreme_scores():
    """Scores far apart: the prefix wins for some heads, the tokens behind it for others."""
    c = _case(10, 8, 8, 64, 16, [(200, [50, 3, 90])], [], poison=False)
    c["vc"] = c["vc"].abs()
    c["q"] = c["q"] * 30
    c["q"][1] = 0  # equal scores
    args = (c["q"], c["kc"], c["vc"], c["lens"], c["tables"], c["scale"])
    e, mean = O.paged_decode_attention(*args).double(), O.paged_decode_attention_abs(*args).double()
    # scores are 30 times the normal ones: their error, 2^-13.7 at 1, is below 30 * 2^-13 each way
    bound = F.attention_bound(c["q"].dtype, e, mean) + 2 * 30 * 2.0 ** -13 * mean
    for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
        assert bool(((_call(c, variant=variant).cpu().double() - e).abs() <= bound).all())


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_negative_and_zero_scales(variant, scale):
    c = _case(13, 16, 2, 128, 16, [(200, [5, 40, 3])], [], poison=True)
    _check(dict(c, scale=scale), _call(dict(c, scale=scale), variant=variant))


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
def test_rising_maxima_and_bad_prefix_pages(variant):
    """Keys that grow along the prefix raise every row's maximum tile after tile; a prefix page that
    does not exist is left out, whatever lies in the memory that its tokens would have come to."""
    c = _case(14, 16, 1, 128, 32, [(1000, [5, 40, 3, 9, 1, 0, 2, 77, 8, 8])], [], poison=False)
    c["kc"][c["tables"][0, :31].long()] *= torch.linspace(0.2, 6, 31).to(torch.bfloat16).view(-1, 1, 1, 1)
    args = (c["q"], c["kc"], c["vc"], c["lens"], c["tables"], c["scale"])
    e, mean = O.paged_decode_attention(*args).double(), O.paged_decode_attention_abs(*args).double()
    # scores are up to 6 times the normal ones: their error, 2^-13.7 at 1, is below 6 * 2^-13 each way
    bound = F.attention_bound(c["q"].dtype, e, mean) + 2 * 6 * 2.0 ** -13 * mean
    assert bool(((_call(c, variant=variant).cpu().double() - e).abs() <= bound).all())
    c = _case(15, 16, 8, 128, 16, [(300, [5, 40, 3])], [], poison=True)
    keep = torch.ones(304, dtype=torch.bool)
    keep[16 * 7:16 * 8] = False
    keep[16 * 15:16 * 16] = False
    c["tables"][0, 7], c["tables"][0, 15] = -1, 10 ** 6  # the first request's table names the prefix
    out = _call(c, variant=variant)
    for b in range(3):
        n = int(c["lens"][b])
        good = c["tables"][1 if b == 0 else b].clone()  # the shared pages, by a table that has them all
        row = torch.where((good >= 0) & (torch.arange(len(good)) < 18), good, c["tables"][b])
        at = torch.tensor([t for t in range(n) if t >= 300 or keep[t]])
        page = row.long()[at // 16]
        for h in range(8):
            e, mean = F.attention(c["q"][b, 2 * h:2 * h + 2], c["kc"][page, at % 16, h], c["vc"][page, at % 16, h], c["scale"])
            off = (out[b, 2 * h:2 * h + 2].cpu().double() - e).abs()
            assert bool((off <= F.attention_bound(c["q"].dtype, e, mean)).all()), (b, h)


def test_strided_inputs():
    """q from a fused qkv row, both caches slices of one allocation, tables from a wider array."""
    c = _case(12, 16, 8, 128, 16, [(90, [10, 33, 1])], [5])
    qkv = torch.randn(4, 32 * 128).to(torch.bfloat16).cuda()
    qkv[:, :2048] = c["q"].cuda().reshape(4, -1)
    both = torch.stack([c["kc"], c["vc"]], 1).cuda()  # [pages, 2, block, heads, dim]
    wide = torch.full((4, c["tables"].shape[1] + 5), 7, dtype=torch.int32).cuda()
    wide[:, :-5] = c["tables"].cuda()
    out = ops.shared_prefix_decode_attention(qkv[:, :2048].view(4, 16, 128), both[:, 0], both[:, 1], c["lens"].cuda(),
                                             wide[:, :-5], c["offsets"].cuda(), c["prefix"].cuda(), c["scale"])
    _check(c, out)
    out = shared_prefix_attention(qkv[:, :2048].view(4, 16, 128), both[:, 0], both[:, 1], c["lens"].cuda().long(),
                                  wide[:, :-5].long(), c["offsets"].cuda().long(), c["prefix"].cuda().long(), c["scale"])
    _check(c, out)


def test_captured_replayed_and_on_two_streams():
    """Graphs replayed with other lengths and groups in place equal eager calls; two streams at once
    do not meet in a workspace."""
    cases = [_case(20 + s, 16, 8, 128, 64, gr, [9], poison=False) for s, gr in
             enumerate([[(500, [1, 2, 3, 4, 5, 6]), (64, [0, 7])], [(130, [9, 200]), (257, [64, 1, 0, 5, 33, 2])]])]
    wide = max(c["tables"].shape[1] for c in cases)
    pages = max(c["kc"].shape[0] for c in cases)
    for c in cases:
        c["tables"] = torch.nn.functional.pad(c["tables"], (0, wide - c["tables"].shape[1]), value=-1)
        for k in ("kc", "vc"):
            c[k] = torch.nn.functional.pad(c[k], (0, 0) * 3 + (0, pages - c[k].shape[0]))
    keys = ("q", "kc", "vc", "lens", "tables", "offsets", "prefix")
    buf = {k: cases[0][k].cuda() for k in keys}
    call = lambda b: ops.shared_prefix_decode_attention(*(b[k] for k in keys), cases[0]["scale"])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(buf)
    for c in (cases[1], cases[0]):
        for k in keys:
            buf[k].copy_(c[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(buf))
        _check(c, out)
    del graph
    bufs = [{k: c[k].cuda() for k in keys} for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = []
        for s, b in zip(streams, bufs):
            with torch.cuda.stream(s):
                outs.append(call(b))
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        _check(c, o)


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
def test_nan_reaches_the_rows_that_meet_it_and_no_others(variant):
    """A NaN query, a NaN key among the shared tokens (one kv head) and one behind them: NaN in
    exactly the rows whose attention meets one."""
    c = _case(16, 16, 8, 128, 16, [(300, [5, 40, 3])], [20], poison=True)
    c["q"][1, 7] = float("nan")
    c["kc"][c["tables"][0, 3], 2, 5, 9] = float("nan")   # shared: heads 10 and 11 of requests 0, 1, 2
    c["kc"][c["tables"][3, 0], 1, 0, 0] = float("nan")   # heads 0 and 1 of request 3
    expect = torch.zeros(4, 16, dtype=torch.bool)
    expect[1, 7] = expect[3, :2] = True
    expect[:3, 10:12] = True
    out = _call(c, variant=variant).cpu()
    assert torch.equal(torch.isnan(out).all(-1), expect) and torch.equal(torch.isnan(out).any(-1), expect)


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
def test_large_calls_on_two_streams(variant):
    cases = [_case(70 + s, 16, 2, 128, 64, [(3000, [i % 9 for i in range(n)])], [], poison=False) for s, n in enumerate((60, 35))]
    gpu = [{k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()} for c in cases]
    call = lambda d: ops.shared_prefix_decode_attention(  # noqa: E731
        *(d[k] for k in ("q", "kc", "vc", "lens", "tables", "offsets", "prefix", "scale")), variant=variant)
    alone = [call(d) for d in gpu]
    streams = [torch.cuda.Stream() for _ in gpu]
    torch.cuda.synchronize()
    for _ in range(10):
        outs = []
        for s, d in zip(streams, gpu):
            with torch.cuda.stream(s):
                outs.append(call(d))
    torch.cuda.synchronize()
    for c, a, o in zip(cases, alone, outs):
        assert torch.equal(a, o)
        _check(c, o)


def test_reports(monkeypatch):
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    c = _case(30, 16, 8, 128, 16, [(40, [3, 4])], [5], poison=False)
    _check(c, _call(c))
    bad = dict(c, tables=c["tables"].clone())
    bad["tables"][0, 1] = 10 ** 6  # a prefix page
    with pytest.raises(ValueError, match="block"):
        _call(bad)
    bad = dict(c, tables=c["tables"].clone())
    bad["tables"][1, 2] = -7  # a page behind the prefix
    with pytest.raises(ValueError, match="block"):
        _call(bad)
    for name, value in (("offsets", [0, 9]), ("offsets", [-1, 2]), ("prefix", [-4]), ("lens", [10 ** 6, 44, 5])):
        with pytest.raises(ValueError, match="out of range"):
            _call(dict(c, **{name: torch.tensor(value, dtype=torch.int32)}))


def test_refusals():
    c = _case(31, 16, 8, 128, 16, [(40, [3, 4])], [5], poison=False)
    cu = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}

    def call(**over):
        d = dict(cu, **over)
        return ops.shared_prefix_decode_attention(*(d[k] for k in ("q", "kc", "vc", "lens", "tables", "offsets", "prefix", "scale")))

    for over, text in [
        (dict(q=cu["q"].half()), "share a dtype"), (dict(q=cu["q"][..., :64]), "head_dim"),
        (dict(lens=cu["lens"].long()), "context_lens"), (dict(tables=cu["tables"][:2]), "block_tables"),
        (dict(offsets=cu["offsets"].long()), "group_offsets"), (dict(prefix=cu["prefix"][:0]), "group_offsets"),
        (dict(prefix=c["prefix"]), "must be on"), (dict(q=cu["q"][:, :12]), "bad head counts"),
        (dict(kc=cu["kc"][:, :15], vc=cu["vc"][:, :15]), "multiple of 16"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**over)
    f32 = {k: cu[k].float() for k in ("q", "kc", "vc")}
    with pytest.raises(RuntimeError, match="bf16 or f16"):
        call(**f32)
    assert call(q=cu["q"][:0], lens=cu["lens"][:0], tables=cu["tables"][:0], offsets=cu["offsets"] * 0).shape == (0, 16, 128)
