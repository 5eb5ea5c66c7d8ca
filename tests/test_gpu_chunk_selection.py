"""Chunk selection where hundreds of chunks compete for the last places: ties, scores that differ by less
than their 32-bit error, scores that are not finite, chunks without a block; below and above the 256 chunks
that are compared each with each and the 8,192 whose keys stay in shared memory. Selections equal the
64-bit form's."""

import math

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import _cache_forms as F

pytestmark = pytest.mark.gpu

COUNTS = [300, 8193, 9000]
NQ, NKV, DIM, CHUNK = 4, 2, 64, 16


def _case(seed, n, dtype=torch.bfloat16, nq=NQ, nkv=NKV, dim=DIM):
    """One request of n chunks, a block each; random keys behind random bounds."""
    g = torch.Generator().manual_seed(seed)
    kc = torch.randn(n, CHUNK, nkv, dim, generator=g).to(dtype)
    bounds = torch.stack([kc.amin(1), kc.amax(1)], 2).unsqueeze(2).contiguous()  # [blocks, heads, 1, 2, dim]
    q = torch.randn(1, nq, dim, generator=g).to(dtype)
    return dict(q=q, kc=kc, vc=kc, bounds=bounds, tables=torch.randperm(n, generator=g).to(torch.int32)[None], n=n)


def _by_chunk(c, chunks, value):
    """The bounds of these chunks become `value` ([heads, 2, dim])."""
    c["bounds"][c["tables"][0, chunks].long(), :, 0] = value


def _check(c, top, expect=None, what=""):
    lens = torch.tensor([c["n"] * CHUNK - 3], dtype=torch.int32)
    if expect is None:
        expect = F.select_chunks(c["q"], c["bounds"], c["tables"], lens.tolist(), CHUNK, top)
    args = [t.cuda() for t in (c["q"], c["kc"], c["vc"], c["bounds"], lens, c["tables"])]
    _, got = ops.sparse_decode_attention(*args, c["q"].shape[-1] ** -0.5, top)
    assert torch.equal(got.cpu(), expect), (what, int((got.cpu() != expect).sum()), got.cpu()[0, 0].tolist()[:12], expect[0, 0].tolist()[:12])
    assert torch.equal(got, ops.sparse_decode_attention(*args, c["q"].shape[-1] ** -0.5, top)[1]), "the same twice"


@pytest.mark.parametrize("n", COUNTS)
@pytest.mark.parametrize("top", [3, 200, 290])
def test_every_score_equal(n, top):
    """A zero query, a table whose chunks have the same bounds, a NaN query: the lowest indices and the last."""
    lowest = torch.tensor(list(range(top - 1)) + [n - 1], dtype=torch.int32)
    c = _case(n, n)
    c["q"].zero_()
    _check(c, top, lowest.expand(1, NKV, top), "zero query")
    c = _case(n + 1, n)
    _by_chunk(c, torch.arange(n), c["bounds"][5, :, 0].clone())
    _check(c, top, lowest.expand(1, NKV, top), "equal bounds")
    c = _case(n + 2, n)
    c["q"][0, 1, 3] = float("nan")  # head 1: the first kv head
    expect = F.select_chunks(c["q"], c["bounds"], c["tables"], [n * CHUNK - 3], CHUNK, top)
    assert torch.equal(expect[0, 0], lowest)
    _check(c, top, expect, "NaN query")


@pytest.mark.parametrize("n", COUNTS)
@pytest.mark.parametrize("value", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_bound_that_is_not_finite(n, value, dtype):
    """It makes every chunk compete in 64 bits: the others are ranked as without it."""
    c = _case(n, n, dtype)
    c["q"][0, :, 7] = c["q"][0, :, 7].abs() + 0.5  # no 0 x infinity but in the chunk itself
    c["bounds"][c["tables"][0, n // 3].long(), 0, 0, 1, 7] = value
    for top in (4, 150):
        _check(c, top, what=f"{value}")


@pytest.mark.parametrize("equal", [255, 256, 257, 258, 700])
def test_competitors_around_the_number_compared_each_with_each(equal):
    """`equal` chunks tie between better and worse ones; the last place falls on the first, in the middle
    and on the last of them."""
    better, worse = 20, 300
    n = equal + better + worse + 2
    c = _case(equal, n)
    g = torch.Generator().manual_seed(equal)
    order = torch.randperm(n - 2, generator=g) + 1
    # q . bounds dominated by one channel of weight 1 in every head
    c["q"] = c["q"] * 0.01
    c["q"][..., 0] = 1
    flat = torch.zeros(NKV, 2, DIM, dtype=torch.bfloat16)
    flat[..., 0] = 5
    c["bounds"][..., 0] = 1
    _by_chunk(c, order[:equal], flat)
    high = flat.clone()
    high[..., 0] = 9
    _by_chunk(c, order[equal:equal + better], high)
    for places in (1, equal // 2, equal - 1, equal):
        _check(c, 2 + better + places, what=f"{places} of {equal}")


@pytest.mark.parametrize("first,second", [(100, 400), (300, 400), (300, 9000)])
def test_ties_that_only_64_bits_tell_apart(first, second):
    """Two groups of equal scores, the second less by 2^-37 of them, far below what 32 bits show: the last
    place inside the first group, between the two and inside the second."""
    n = first + second + 50
    c = _case(first + second, n)
    c["q"][:] = 1
    c["q"][..., 1] = 2.0 ** -30
    order = torch.randperm(n - 2, generator=torch.Generator().manual_seed(n)) + 1
    flat = torch.ones(NKV, 2, DIM, dtype=torch.bfloat16)
    _by_chunk(c, torch.arange(n), flat * 0.25)
    _by_chunk(c, order[:first], flat)
    less = flat.clone()
    less[..., 1] = 0.5
    _by_chunk(c, order[first:first + second], less)
    for inside in (first // 2, first - 1, first, first + 1, first + second // 3, first + second):
        _check(c, 2 + inside, what=f"{inside} of {first} + {second}")


@pytest.mark.parametrize("n,missing", [(300, 250), (300, 20), (300, 298), (9000, 8700)])
def test_chunks_without_a_block_come_last(n, missing):
    """In their order, when places are left: the last place on a chunk with a block, on the last of these,
    and among those without."""
    c = _case(n + missing, n)
    bad = (torch.randperm(n - 2, generator=torch.Generator().manual_seed(missing)) + 1)[:missing].sort().values
    lens = [n * CHUNK - 3]
    scores = F.select_chunks(c["q"], c["bounds"], c["tables"], lens, CHUNK, n)  # the tables are whole here
    assert scores.shape[-1] == n
    box = c["bounds"][c["tables"][0].long()][:, :, 0].double()
    gone = set(bad.tolist())
    tables = c["tables"].clone()
    c["tables"][0, bad] = torch.where(torch.arange(missing) % 2 == 0, -1, 10 ** 6).to(torch.int32)
    valid = n - missing
    for top in sorted({2, max(2, valid // 2), valid - 1, valid, valid + 1, valid + missing // 2, n - 1} - {0, 1}):
        expect = torch.full((1, NKV, top), -1, dtype=torch.int32)
        for h in range(NKV):
            x = c["q"][0, h * (NQ // NKV):(h + 1) * (NQ // NKV)].double()
            s = sum((x[i].clamp_min(0) * box[:, h, 1] + x[i].clamp_max(0) * box[:, h, 0]).sum(-1) for i in range(NQ // NKV)).tolist()
            s = [-math.inf if i in gone else v for i, v in enumerate(s)]
            s[0] = s[-1] = math.inf
            expect[0, h] = torch.tensor(sorted(sorted(range(n), key=lambda i, s=s: (-s[i], i))[:top]), dtype=torch.int32)
        _check(c, top, expect, f"top {top}")
    assert bool((tables >= 0).all())


def test_many_rows_whose_scores_tie():
    """Rows of every kind in one call: random, zero and NaN queries, equal bounds."""
    n, batch = 700, 24
    c = _case(3, n, nq=16, nkv=8, dim=128)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(batch, 16, 128, generator=g).to(torch.bfloat16)
    q[::4] = 0
    q[1::4, 5] = float("nan")
    tables = torch.stack([torch.randperm(n, generator=g) for _ in range(batch)]).to(torch.int32)
    tables[2::4] = tables[2, 0]
    lens = [n * CHUNK - i * 5 for i in range(batch)]
    expect = F.select_chunks(q, c["bounds"], tables, lens, CHUNK, 64)
    got = ops.sparse_decode_attention(q.cuda(), c["kc"].cuda(), c["vc"].cuda(), c["bounds"].cuda(),
                                      torch.tensor(lens, dtype=torch.int32).cuda(), tables.cuda(), 128 ** -0.5, 64)[1]
    assert torch.equal(got.cpu(), expect)
