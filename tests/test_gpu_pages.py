"""Page operators (``nib_paged_copy_blocks`` / ``fork`` / ``free`` / ``compact``) against plain list
forms: whole numbers and moved bytes are equal, every other byte of the cache stays as it was."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from nano_vllm_multimodal_b200.layers.paged_kv.cuda_backend import CUDAPagedKVBackend
from tests import _cache_forms as F

pytestmark = pytest.mark.gpu


def _cache(seed, shape, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    n = 1
    for s in shape:
        n *= s
    size = torch.empty(0, dtype=dtype).element_size()
    # random bytes: NaNs and infinities among the values are copied like any other
    return torch.randint(0, 256, (n * size,), generator=g, dtype=torch.uint8).view(dtype).view(shape)


def _same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


SHAPES = [
    ((2, 3, 24, 16, 8, 128), torch.bfloat16),   # K and V of three layers
    ((24, 256, 2, 64), torch.float16),          # one layer's keys
    ((5, 24, 48, 1, 8), torch.float32),         # small rows, five planes
    ((3, 24, 7, 1, 3), torch.bfloat16),         # 42-byte blocks: two-byte copies
    ((2, 24, 1, 1, 2), torch.float32),          # one-token blocks of eight bytes
    ((1, 24, 500, 2, 120), torch.bfloat16),     # a block of several pieces with a ragged last one
]


@pytest.mark.parametrize("shape,dtype", SHAPES)
@pytest.mark.parametrize("n", [0, 1, 11])
def test_copy_blocks(shape, dtype, n):
    c = _cache(sum(shape) + n, shape, dtype)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n:2 * n]
    e = c.clone()
    blocks = e.view(-1, *shape[-4:])
    for s, d in zip(src, dst):
        blocks[:, d] = blocks[:, s]
    g = c.cuda()
    assert ops.paged_copy_blocks(g, _ints(src), _ints(dst)) is None
    assert _same(g, e)


def test_copy_blocks_of_views_and_other_dims():
    """A layer's slice of the runner's allocation (planes with a stride of their own), bounds kept
    beside the cache (block_dim -5), a source read twice, padding pairs."""
    c = _cache(3, (2, 4, 20, 16, 2, 64))
    g = c.cuda()
    ops.paged_copy_blocks(g[:, 2], _ints([3, 3, -1, 5]), _ints([7, 9, 4, -1]))
    c[:, 2, 7] = c[:, 2, 3]
    c[:, 2, 9] = c[:, 2, 3]
    assert _same(g, c)
    b = _cache(4, (3, 20, 2, 4, 2, 64))
    h = b.cuda()
    ops.paged_copy_blocks(h, _ints([0, 19]), _ints([10, 11]), block_dim=-5)
    b[:, 10], b[:, 11] = b[:, 0], b[:, 19]
    assert _same(h, b)


def test_copy_blocks_leaves_ambiguous_pairs_out(monkeypatch):
    """A destination that another pair reads or writes would depend on the copies' order: such
    pairs are left out (the others run), and validation mode reports them."""
    c = _cache(5, (2, 16, 8, 2, 64))
    src, dst = [0, 1, 2, 3, 4, 12, 13], [5, 5, 6, 2, 7, 99, 13]  # 5 twice; 2 is a source; 99 no block; 13 onto itself
    e = c.clone()
    e[:, 6], e[:, 7] = c[:, 2], c[:, 4]
    g = c.cuda()
    ops.paged_copy_blocks(g, _ints(src), _ints(dst))
    assert _same(g, e)
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    with pytest.raises(ValueError, match="out of range"):
        ops.paged_copy_blocks(c.cuda(), _ints([0, 1]), _ints([5, 5]))
    with pytest.raises(ValueError, match="invalid physical block"):
        ops.paged_copy_blocks(c.cuda(), _ints([0]), _ints([16]))
    ops.paged_copy_blocks(c.cuda(), _ints([0, -1]), _ints([5, 5]))  # padding is no conflict


def _pool(seed, rows, width, blocks, block, empty, spare=0):
    """Rows of distinct blocks with lengths that end anywhere, `empty` of them empty at the end."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(blocks, generator=g).tolist()
    tables = [[-1] * width for _ in range(rows)]
    lens, refs = [0] * rows, [0] * blocks
    for r in range(rows - empty):
        lens[r] = int(torch.randint(0, width * block + 1, (1,), generator=g))
        if r < 3:
            lens[r] = [width * block, 1, block][r]  # all of the row, one token, exactly one block
        for j in range(-(-lens[r] // block)):
            if len(order) <= spare:
                lens[r] = j * block
                break
            tables[r][j] = order.pop()
            refs[tables[r][j]] = 1
    return tables, lens, refs


@pytest.mark.parametrize("shape,dtype,width", [
    ((2, 2, 60, 16, 2, 64), torch.bfloat16, 6), ((1, 60, 5, 1, 3), torch.float16, 9), ((4, 60, 64, 1, 128), torch.float32, 1)])
def test_fork_then_free(shape, dtype, width):
    block, blocks = shape[-3], shape[-4]
    tables, lens, refs = _pool(shape[0] + width, 30, width, blocks, block, 16, spare=20)
    parents = [0, 1, 1, 2, 5, 0, 3, 14, 1, 4]  # 14: an empty parent
    children = [29, 14 + 2, 18, 19, 20, 25, 24, 23, 22, 21]
    c = _cache(9, shape, dtype)
    e_tables, e_lens, e_refs, e_copies = F.fork(block, tables, lens, refs, parents, children)
    e = c.clone()
    planes = e.view(-1, *shape[-4:])
    for s, d, n in e_copies:
        if n:
            planes[:, d, :n] = planes[:, s, :n]
    g = c.cuda()
    inputs = [_ints(tables), _ints(lens), _ints(refs)]
    kept = [t.clone() for t in inputs]
    got = ops.paged_fork(g, *inputs, _ints(parents), _ints(children))
    assert got[0].tolist() == e_tables and got[1].tolist() == e_lens and got[2].tolist() == e_refs
    assert list(zip(*got[3].tolist())) == e_copies
    assert _same(g, e)
    assert all(torch.equal(a, b) for a, b in zip(inputs, kept)), "the inputs stay as they were"
    # the children and one parent go again; a row twice, padding, an empty row
    rows = [29, 0, 18, 18, -1, 14, 22]
    f_tables, f_lens, f_refs = F.release(block, e_tables, e_lens, e_refs, rows)
    out = ops.paged_free(*got[:3], _ints(rows), block)
    assert out[0].tolist() == f_tables and out[1].tolist() == f_lens and out[2].tolist() == f_refs


def test_fork_refuses_single_forks(monkeypatch):
    """A child that holds tokens, is named twice or does not exist, and a fork without a free
    block, leave their rows as they were; the other forks take place."""
    block, blocks, width = 4, 8, 3
    tables = [[0, 1, -1], [2, 3, 4], [-1] * 3, [-1] * 3, [-1] * 3, [-1] * 3]
    lens, refs = [6, 9, 0, 0, 0, 0], [1, 1, 1, 1, 1, 0, 1, 1]  # one free block
    cases = [
        ([0, 0], [1, 2]),          # row 1 is not empty
        ([0, 1], [2, 2]),          # row 2 twice: the first
        ([0, 1, 0], [3, 4, 5]),    # one block for three
        ([7, 0, -1], [2, 9, 3]),   # no such row, no such child, padding
    ]
    c = _cache(1, (2, blocks, block, 1, 8))
    for parents, children in cases:
        e = F.fork(block, tables, lens, refs, parents, children)
        g = c.cuda()
        got = ops.paged_fork(g, _ints(tables), _ints(lens), _ints(refs), _ints(parents), _ints(children))
        assert [got[0].tolist(), got[1].tolist(), got[2].tolist()] == [e[0], e[1], e[2]], (parents, children)
        assert list(zip(*got[3].tolist())) == e[3]
        x = c.clone()
        for s, d, n in e[3]:
            if n:
                x[:, d, :n] = x[:, s, :n]
        assert _same(g, x)
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    args = (_ints(tables), _ints(lens), _ints(refs))
    with pytest.raises(ValueError, match="no free page"):
        ops.paged_fork(c.cuda(), *args, _ints([0, 1]), _ints([3, 4]))
    with pytest.raises(ValueError, match="out of range"):
        ops.paged_fork(c.cuda(), *args, _ints([0, 1]), _ints([2, 2]))
    with pytest.raises(ValueError, match="invalid physical block"):
        ops.paged_fork(c.cuda(), _ints([[0, 99, -1]] + tables[1:]), *args[1:], _ints([0]), _ints([2]))
    with pytest.raises(ValueError, match="out of range"):
        ops.paged_free(*args, _ints([6]), block)
    with pytest.raises(ValueError, match="out of range"):  # block 0's count is 0 already
        ops.paged_free(*args[:2], _ints([0] + refs[1:]), _ints([0]), block)


def test_free_never_counts_below_zero():
    tables, lens = [[0, 1], [0, 1], [0, -1]], [8, 8, 2]
    out = ops.paged_free(_ints(tables), _ints(lens), _ints([2, 1, 3]), _ints([0, 1, 2]), 4)
    assert out[2].tolist() == [0, 0, 3] and out[1].tolist() == [0, 0, 0] and out[0].tolist() == [[-1, -1]] * 3


@pytest.mark.parametrize("shape,dtype", [((2, 2, 50, 16, 2, 64), torch.bfloat16), ((1, 51, 5, 1, 3), torch.float16),
                                         ((3, 3000, 1, 1, 4), torch.float32), ((1, 1, 4, 1, 8), torch.bfloat16)])
@pytest.mark.parametrize("load", [0.0, 0.05, 0.5, 0.97, 1.0])
def test_compact(shape, dtype, load):
    blocks = shape[-4]
    g = torch.Generator().manual_seed(blocks)
    refs = [int(x) * (1 + i % 3) for i, x in enumerate(torch.rand(blocks, generator=g) < load)]
    live = [p for p, r in enumerate(refs) if r]
    width = 7
    tables = [live[i:i + width] for i in range(0, len(live), width)] + [live[:width]] if live else [[]]  # a shared row
    tables = [r + [-1] * (width - len(r)) for r in tables]
    c = _cache(blocks, shape, dtype)
    e_tables, e_refs, e_live, moves = F.compact(tables, refs)
    e = c.clone()
    planes = e.view(-1, *shape[-4:])
    for s, d in moves:
        planes[:, d] = planes[:, s]
    d_cache = c.cuda()
    got = ops.paged_compact(d_cache, _ints(tables), _ints(refs))
    assert got[0].tolist() == e_tables and got[1].tolist() == e_refs and got[2].tolist() == [e_live]
    assert [m for m in zip(*got[3].tolist()) if m != (-1, -1)] == moves and got[3].shape == (2, blocks // 2)
    assert _same(d_cache, e)


def test_together_captured_and_replayed():
    """Fork, release, compact as one captured graph on a stream of its own, replayed on new tables."""
    block, blocks, rows, width = 16, 40, 12, 4
    tables, lens, refs = _pool(77, rows, width, blocks, block, 6, spare=12)
    c = _cache(11, (2, blocks, block, 2, 64))
    parents, children, gone = [0, 1, 2, 1], [11, 10, 9, 8], [0, 10]

    def expected(tables, lens, refs, cache):
        e = cache.clone()
        t, ln, r, copies = F.fork(block, tables, lens, refs, parents, children)
        for s, d, n in copies:
            if n:
                e[:, d, :n] = e[:, s, :n]
        t, ln, r = F.release(block, t, ln, r, gone)
        t, r, live, moves = F.compact(t, r)
        for s, d in moves:
            e[:, d] = e[:, s]
        return t, ln, r, live, e

    g, t0, l0, r0 = c.cuda(), _ints(tables), _ints(lens), _ints(refs)
    p, ch, go = _ints(parents), _ints(children), _ints(gone)

    def call():
        t, ln, r, _ = ops.paged_fork(g, t0, l0, r0, p, ch)
        t, ln, r = ops.paged_free(t, ln, r, go, block)
        t, r, live, _ = ops.paged_compact(g, t, r)
        return t, ln, r, live

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    e = expected(tables, lens, refs, c)
    assert [x.tolist() for x in got] == [e[0], e[1], e[2], [e[3]]] and _same(g, e[4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (78, 79):
        tables, lens, refs = _pool(seed, rows, width, blocks, block, 6, spare=12)
        c = _cache(seed, c.shape)
        g.copy_(c), t0.copy_(_ints(tables)), l0.copy_(_ints(lens)), r0.copy_(_ints(refs))
        graph.replay()
        torch.cuda.synchronize()
        e = expected(tables, lens, refs, c)
        assert [x.tolist() for x in out] == [e[0], e[1], e[2], [e[3]]] and _same(g, e[4]), seed
    del graph


def test_two_streams_at_once():
    """Two caches' calls overlap: each has a workspace of its own."""
    block, blocks = 16, 40
    pools = [_pool(s, 12, 4, blocks, block, 6, spare=12) for s in (1, 2)]
    caches = [_cache(s, (2, blocks, block, 8, 128)) for s in (1, 2)]
    on = [torch.cuda.Stream() for _ in pools]
    gpu = [(c.cuda(), *(_ints(x) for x in pool)) for c, pool in zip(caches, pools)]
    p, ch = _ints([0, 1, 2]), _ints([11, 10, 9])
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for s, (c, t, ln, r) in zip(on, gpu):
            with torch.cuda.stream(s):
                got.append(ops.paged_fork(c, t, ln, r, p, ch))
    torch.cuda.synchronize()
    for (tables, lens, refs), out in zip(pools, got):
        e = F.fork(block, tables, lens, refs, [0, 1, 2], [11, 10, 9])
        assert [x.tolist() for x in out[:3]] == list(e[:3])


def test_empty_calls():
    c = _cache(1, (2, 4, 8, 1, 8)).cuda()
    none, keep = _ints([]), c.clone()
    ops.paged_copy_blocks(c, none, none)
    t, ln, r, copies = ops.paged_fork(c, _ints([[-1]]), _ints([0]), _ints([0] * 4), none, none)
    assert t.tolist() == [[-1]] and ln.tolist() == [0] and r.tolist() == [0] * 4 and copies.shape == (3, 0)
    t, ln, r = ops.paged_free(_ints([[1]]), _ints([3]), _ints([0, 1, 0, 0]), none, 8)
    assert t.tolist() == [[1]] and ln.tolist() == [3] and r.tolist() == [0, 1, 0, 0]
    t, r, live, moves = ops.paged_compact(c, torch.empty(0, 3, dtype=torch.int32, device="cuda"), _ints([0] * 4))
    assert t.shape == (0, 3) and live.tolist() == [0] and moves.tolist() == [[-1, -1], [-1, -1]]
    assert _same(c, keep)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB whose last blocks are copied."""
    c = torch.zeros(1, 2200, 256, 32, 128, dtype=torch.bfloat16, device="cuda")  # 4.6 GB
    c[0, 2198] = 3.0
    ops.paged_copy_blocks(c, _ints([2198]), _ints([2199]))
    assert bool((c[0, 2199] == 3.0).all()) and not bool(c[0, 2197].any())
    del c
    torch.cuda.empty_cache()


def test_backend_methods():
    """The ``cuda`` paged-KV backend reaches them next to its store and gather."""
    be = CUDAPagedKVBackend()
    a = be.allocate((2, 2, 12, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    a.tensor.copy_(_cache(2, tuple(a.tensor.shape)))
    c = a.tensor.cpu()
    be.copy_blocks(a.tensor, _ints([1]), _ints([2]))
    c[:, :, 2] = c[:, :, 1]
    assert _same(a.tensor, c)
    tables, lens, refs = [[0, 1], [-1, -1]], [20, 0], [1, 1] + [0] * 10
    t, ln, r, _ = be.fork(a.tensor, _ints(tables), _ints(lens), _ints(refs), _ints([0]), _ints([1]))
    assert t.tolist() == [[0, 1], [0, 2]] and r.tolist()[:3] == [2, 1, 1]
    t, ln, r = be.free(t, ln, r, _ints([0]), 16)
    assert r.tolist()[:3] == [1, 0, 1]
    t, r, live, _ = be.compact(a.tensor, t, r)
    assert t.tolist() == [[-1, -1], [0, 1]] and live.tolist() == [2]
    with pytest.raises(ValueError, match="CUDA tensors"):
        be.copy_blocks(c, _ints([1]), _ints([2]))
