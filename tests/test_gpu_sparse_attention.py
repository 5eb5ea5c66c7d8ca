"""Key bounds and sparse decode attention (``nib_paged_key_bounds``, ``nib_sparse_decode_attention``)
against 64-bit forms: bounds and selections are equal, outputs within
``tests/_cache_forms.attention_bound`` of attention over the selected chunks."""

import pytest
import torch

import oracle as O
from nano_vllm_multimodal_b200 import ops
from nano_vllm_multimodal_b200.layers.attention import sparse_paged_attention
from tests import _cache_forms as F

pytestmark = pytest.mark.gpu


def _case(seed, nq, nkv, dim, block, chunk, lens, dtype=torch.bfloat16, width=None, poison=True):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in lens]
    width = width or max(1, max(need))
    pages = sum(need) + 3
    kc = torch.randn(pages, block, nkv, dim, generator=g)
    kc += 0.5 * torch.randn(pages, 1, nkv, dim, generator=g)
    kc = kc.to(dtype)
    vc = torch.randn(pages, block, nkv, dim, generator=g).to(dtype)
    order = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, k in enumerate(need):
        for j in range(k):
            tables[b, j] = order.pop()
        if poison and lens[b] % block:
            kc[tables[b, k - 1], lens[b] % block:] = float("nan")
            vc[tables[b, k - 1], lens[b] % block:] = float("inf")
    bounds = torch.full((pages, nkv, block // chunk, 2, dim), float("nan"), dtype=dtype)
    bounds = F.key_bounds(kc, bounds, tables, [0] * len(lens), lens)
    q = torch.randn(len(lens), nq, dim, generator=g).to(dtype)
    return dict(q=q, kc=kc, vc=vc, bounds=bounds, lens=torch.tensor(lens, dtype=torch.int32), tables=tables,
                scale=dim ** -0.5, chunk=chunk, block=block)


KEYS = ("q", "kc", "vc", "bounds", "lens", "tables")


def _call(c, top, **hints):
    return ops.sparse_decode_attention(*(c[k].cuda() for k in KEYS), c["scale"], top, **hints)


def _check(c, top, out, selected, what=""):
    lens = c["lens"].tolist()
    e_sel = F.select_chunks(c["q"], c["bounds"], c["tables"], lens, c["block"], top)
    assert torch.equal(selected.cpu(), e_sel), f"{what}: {int((selected.cpu() != e_sel).sum())} of {e_sel.numel()} entries differ"
    e, mean = F.sparse_attention(c["q"], c["kc"], c["vc"], c["tables"], lens, e_sel, c["chunk"], c["scale"])
    off = (out.cpu().double() - e).abs()
    bound = F.attention_bound(c["q"].dtype, e, mean)
    assert out.dtype == c["q"].dtype and out.shape == c["q"].shape
    assert bool((off <= bound).all()), f"{what}: {int((~(off <= bound)).sum())} off"


@pytest.mark.parametrize("nq,nkv,dim", [(16, 8, 128), (16, 2, 128), (8, 8, 64), (14, 2, 64), (16, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block,chunk,top,lens", [
    (16, 16, 2, [1, 16, 17, 33, 400, 0]),
    (256, 32, 9, [1000, 256, 257, 1, 288, 289, 2048]),     # as many chunks as are kept, one more
    (64, 64, 5, [64 * 5, 64 * 5 + 1, 3000]),
    (48, 16, 30, [47, 1500, 479, 481]),                    # blocks that are no power of two
])
def test_matches_the_64_bit_form(nq, nkv, dim, dtype, block, chunk, top, lens):
    c = _case(nq + nkv + dim + block, nq, nkv, dim, block, chunk, lens, dtype)
    out, selected = _call(c, top)
    _check(c, top, out, selected, f"{nq}/{nkv} D{dim} block {block} chunk {chunk}")
    again = _call(c, top, max_context_len=max(lens))
    _check(c, top, *again, "with a bound")
    assert all(torch.equal(a, b) for a, b in zip((out, selected), _call(c, top))), "the same bits twice"


def test_long_contexts():
    c = _case(3, 16, 8, 128, 256, 32, [20000, 9001], poison=False)
    _check(c, 64, *_call(c, 64, max_context_len=20000))
    c = _case(4, 4, 1, 64, 256, 16, [150000], poison=False)  # more chunks than one pass over them holds
    _check(c, 100, *_call(c, 100))


def test_all_chunks_equal_dense_attention():
    c = _case(5, 16, 8, 128, 64, 16, [700, 64, 3], poison=False)
    out, selected = _call(c, 44)
    dense = O.paged_decode_attention(c["q"], c["kc"], c["vc"], c["lens"], c["tables"], c["scale"]).double()
    mean = O.paged_decode_attention_abs(c["q"], c["kc"], c["vc"], c["lens"], c["tables"], c["scale"]).double()
    assert bool(((out.cpu().double() - dense).abs() <= F.attention_bound(c["q"].dtype, dense, mean)).all())
    assert selected[0, 0].tolist() == list(range(44)) and selected[2, 3].tolist() == [0] + [-1] * 43


def test_ties_go_to_the_lowest_index():
    """Equal bounds, zero queries, and pages that a table names twice."""
    c = _case(6, 8, 2, 64, 16, 16, [16 * 40, 16 * 40, 16 * 40], poison=False)
    c["q"][0] = 0
    c["bounds"][c["tables"][1].long()] = c["bounds"][int(c["tables"][1, 0])].clone()
    c["tables"][2, 10:20] = c["tables"][2, 20:30]
    out, selected = _call(c, 7)
    _check(c, 7, out, selected)
    assert selected[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 39] and selected[1, 1].tolist() == [0, 1, 2, 3, 4, 5, 39]


def test_scores_with_nan_and_infinity():
    """A chunk whose bounds hold NaN or infinity ranks as the largest finite score, minus infinity
    below everything; the first and the last chunk stay whatever the others hold."""
    c = _case(7, 4, 2, 64, 16, 16, [16 * 20], poison=False)
    pages = c["tables"][0].long()
    c["q"] = c["q"].abs() + 0.1
    c["bounds"][pages[5], :, :, :, 3] = float("nan")
    c["bounds"][pages[9], :, :, 1, 0] = float("inf")
    c["bounds"][pages[11], :, :, 1, 0] = float("-inf")
    for top in (3, 4, 5, 19):
        out, selected = _call(c, top)
        _check(c, top, out, selected, f"top {top}")
    assert selected[0, 0].tolist() == [i for i in range(20) if i != 11]
    assert _call(c, 4)[1][0, 1].tolist() == [0, 5, 9, 19]
    c["q"][0, 0, 0] = float("nan")  # every score of its head: the lowest indices
    assert _call(c, 5)[1][0, 0].tolist() == [0, 1, 2, 3, 19]


def test_keys_behind_the_context_and_unselected_chunks_do_not_matter():
    c = _case(8, 16, 8, 128, 64, 16, [500, 333])
    out, selected = _call(c, 6)
    for b, n in enumerate(c["lens"].tolist()):  # NaN in every chunk that neither head selects
        used = set(selected[b].flatten().tolist())
        for j in range(-(-n // 16)):
            if j not in used:
                page, slot = int(c["tables"][b, j // 4]), j % 4 * 16
                c["kc"][page, slot:slot + 16], c["vc"][page, slot:slot + 16] = float("nan"), float("nan")
    again = _call(c, 6)
    assert torch.equal(again[0], out) and not torch.isnan(out).any()


def test_strided_inputs_and_module_call():
    c = _case(9, 16, 8, 128, 32, 16, [300, 77, 500])
    qkv = torch.randn(3, 32 * 128).to(torch.bfloat16).cuda()
    qkv[:, :2048] = c["q"].cuda().reshape(3, -1)
    both = torch.stack([c["kc"], c["vc"]], 1).cuda()
    layers = torch.stack([c["bounds"], c["bounds"] * 0], 1).cuda()  # [pages, 2 layers, ...]
    wide = torch.full((3, c["tables"].shape[1] + 3), 5, dtype=torch.int32).cuda()
    wide[:, :-3] = c["tables"].cuda()
    args = (qkv[:, :2048].view(3, 16, 128), both[:, 0], both[:, 1], layers[:, 0], c["lens"].cuda(), wide[:, :-3])
    out, selected = ops.sparse_decode_attention(*args, c["scale"], 6)
    _check(c, 6, out, selected)
    assert torch.equal(sparse_paged_attention(*args[:4], c["lens"].cuda().long(), wide[:, :-3].long(), c["scale"], 6), out)


@pytest.mark.parametrize("nkv,dim,block,chunk", [(8, 128, 256, 32), (2, 64, 64, 16), (1, 64, 16, 16), (3, 128, 24, 8),
                                                 (40, 128, 16, 16), (8, 128, 128, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds(nkv, dim, block, chunk, dtype):
    """Bounds of the chunks that hold new tokens, from the valid tokens alone; the others keep their bytes."""
    lens = [300, 1, block, 0, 77, 2 * block + 3]
    starts = [299, 0, 0, 0, 30, 2 * block + 3]  # one new token, all new, nothing new
    c = _case(nkv + dim + block, nkv, nkv, dim, block, max(16, chunk), lens, dtype, poison=True) if chunk >= 16 else \
        _case(nkv + dim + block, nkv, nkv, dim, block, block, lens, dtype, poison=True)
    before = torch.full((c["kc"].shape[0], nkv, block // chunk, 2, dim), 9.0, dtype=dtype)
    e = F.key_bounds(c["kc"], before, c["tables"], starts, lens)
    got = before.cuda()
    most = max(n - s for n, s in zip(lens, starts))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    same = ops.paged_key_bounds_(got, c["kc"].cuda(), c["tables"].cuda(), i32(starts), i32(lens), most)
    assert same is got and torch.equal(got.cpu(), e)


def test_bounds_of_nan_infinite_and_strided_keys():
    c = _case(2, 2, 2, 64, 32, 16, [100, 64], poison=False)
    c["kc"][int(c["tables"][0, 1]), 5, 0, 7] = float("nan")
    c["kc"][int(c["tables"][0, 0]), 0, 1, 3] = float("-inf")
    both = torch.stack([c["kc"], c["vc"]], 1).cuda()
    before = torch.zeros(c["kc"].shape[0], 2, 2, 2, 64, dtype=torch.bfloat16)
    layers = torch.stack([before, before], 1).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_key_bounds_(layers[:, 1], both[:, 0], c["tables"].cuda(), i32([0, 0]), i32([100, 64]), 100)
    e = F.key_bounds(c["kc"], before, c["tables"], [0, 0], [100, 64])
    got = layers[:, 1].cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(e)) and torch.equal(got.nan_to_num(), e.nan_to_num())
    assert not layers[:, 0].any()


def test_decode_steps_together():
    """Steps as a program takes them: store a token, refresh its chunk's bounds, attend; then fork
    the sequence with its bounds and attend for both."""
    g = torch.Generator().manual_seed(40)
    block, chunk, nkv, nq, dim, top = 32, 16, 2, 8, 64, 3
    kc = torch.full((20, block, nkv, dim), float("nan"), dtype=torch.bfloat16)
    vc, bounds = kc.clone(), torch.full((20, nkv, 2, 2, dim), float("nan"), dtype=torch.bfloat16)
    tables = torch.full((2, 4), -1, dtype=torch.int32)
    tables[0] = torch.tensor([4, 9, 2, 17])
    gk, gv, gb, gt = kc.cuda(), vc.cuda(), bounds.cuda(), tables.cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def store(first, n):
        k = torch.randn(n, nkv, dim, generator=g).to(torch.bfloat16)
        v = torch.randn(n, nkv, dim, generator=g).to(torch.bfloat16)
        slots = [int(tables[0, t // block]) * block + t % block for t in range(first, first + n)]
        ops.paged_store(k.cuda(), v.cuda(), gk, gv, i32(slots))
        kc.view(-1, nkv, dim)[slots], vc.view(-1, nkv, dim)[slots] = k, v

    store(0, 90)
    ops.paged_key_bounds_(gb, gk, gt[:1], i32([0]), i32([90]), 90)
    for n in range(91, 100):
        store(n - 1, 1)
        ops.paged_key_bounds_(gb, gk, gt[:1], i32([n - 1]), i32([n]), 1)
        q = torch.randn(1, nq, dim, generator=g).to(torch.bfloat16)
        out, selected = ops.sparse_decode_attention(q.cuda(), gk, gv, gb, i32([n]), gt[:1], dim ** -0.5, top)
        e = F.key_bounds(kc, bounds, tables[:1], [0], [n])
        c = dict(q=q, kc=kc, vc=vc, bounds=e, lens=torch.tensor([n]), tables=tables[:1], scale=dim ** -0.5, chunk=chunk, block=block)
        _check(c, top, out, selected, f"{n} tokens")
    refs = torch.zeros(20, dtype=torch.int32)
    refs[tables[0].long()] = 1
    pair = torch.stack([gk, gv])
    t2, l2, r2, copies = ops.paged_fork(pair, gt, i32([99, 0]), refs.cuda(), i32([0]), i32([1]))
    ops.paged_copy_blocks(gb, copies[0], copies[1], block_dim=-5)
    q = torch.randn(1, nq, dim, generator=g).to(torch.bfloat16).expand(2, nq, dim)
    out, selected = ops.sparse_decode_attention(q.cuda(), pair[0], pair[1], gb, l2, t2, dim ** -0.5, top)
    assert torch.equal(out[0], out[1]) and torch.equal(selected[0], selected[1]) and not torch.isnan(out).any()
    dense = ops.shared_prefix_decode_attention(q.cuda(), pair[0], pair[1], l2, t2, i32([0, 2]), i32([99]), dim ** -0.5)
    one = ops.decode_attention(q.cuda(), pair[0], pair[1], l2, t2, dim ** -0.5)
    u = torch.finfo(torch.bfloat16).eps / 2
    assert torch.equal(dense[0], dense[1])
    # both round probabilities and the result to bf16: 2 u each way of a mean of |v| below 4
    assert bool(((dense.double() - one.double()).abs() <= 16 * u).all())


def test_captured_replayed_and_on_two_streams():
    cases = [_case(50 + s, 16, 8, 128, 64, 16, lens, width=40, poison=False) for s, lens in
             enumerate([[2000, 100, 640], [7, 2560, 1999]])]
    pages = max(c["kc"].shape[0] for c in cases)
    for c in cases:
        for k in ("kc", "vc", "bounds"):
            c[k] = torch.nn.functional.pad(c[k].flatten(1), (0, 0, 0, pages - c[k].shape[0])).view(pages, *c[k].shape[1:])
    buf = {k: cases[0][k].cuda() for k in KEYS}
    call = lambda b: ops.sparse_decode_attention(*(b[k] for k in KEYS), cases[0]["scale"], 9)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(buf)
    for c in (cases[1], cases[0]):
        for k in KEYS:
            buf[k].copy_(c[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call(buf)))
        _check(c, 9, *out)
    del graph
    bufs = [{k: c[k].cuda() for k in KEYS} for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = []
        for s, b in zip(streams, bufs):
            with torch.cuda.stream(s):
                outs.append(call(b))
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        _check(c, 9, *o)


@pytest.mark.parametrize("top", [3, 40])
def test_nan_reaches_the_rows_that_meet_it_and_no_others(top):
    """A NaN query (its kv head's selection is the lowest indices) and a NaN key in a selected chunk."""
    c = _case(66, 16, 8, 128, 64, 16, [500, 333], poison=True)
    c["q"][0, 5] = float("nan")
    c["kc"][c["tables"][1, 0], 3, 7, 1] = float("nan")   # the first chunk is always selected: heads 14, 15
    out = _call(c, top)[0].cpu()
    expect = torch.zeros(2, 16, dtype=torch.bool)
    expect[0, 5] = expect[1, 14] = expect[1, 15] = True
    assert torch.equal(torch.isnan(out).all(-1), expect) and torch.equal(torch.isnan(out).any(-1), expect)


def test_pages_past_32_bit_offsets():
    """The same pages at the end of caches of 2.4e9 elements give the same bits, for the bounds, the
    sparse and the shared-prefix attention."""
    c = _case(67, 16, 8, 128, 256, 32, [1500, 700], poison=False)
    small = c["kc"].shape[0]
    pages = 9200  # x 256 x 8 x 128 elements
    big = {k: torch.zeros(pages, 256, 8, 128, dtype=torch.bfloat16, device="cuda") for k in ("kc", "vc")}
    for k in big:
        big[k][pages - small:] = c[k].cuda()
    moved = torch.where(c["tables"] >= 0, c["tables"] + (pages - small), -1).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    bounds = torch.zeros(pages, 8, 8, 2, 128, dtype=torch.bfloat16, device="cuda")
    ops.paged_key_bounds_(bounds, big["kc"], moved, i32([0, 0]), c["lens"].cuda(), 1500)
    assert torch.equal(bounds[pages - small:][c["tables"][0].long()].cpu(), c["bounds"][c["tables"][0].long()].nan_to_num())
    far = ops.sparse_decode_attention(c["q"].cuda(), big["kc"], big["vc"], bounds, c["lens"].cuda(), moved, c["scale"], 9)
    near = _call(c, 9)
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    group = (c["lens"].cuda(), i32([0, 2]), i32([1]))
    for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
        shared = [ops.shared_prefix_decode_attention(c["q"].cuda()[:1].expand(2, 16, 128), k, v, group[0], t, *group[1:],
                                                     c["scale"], variant=variant)
                  for k, v, t in ((big["kc"], big["vc"], moved), (c["kc"].cuda(), c["vc"].cuda(), c["tables"].cuda()))]
        assert torch.equal(*shared)
    del big, bounds
    torch.cuda.empty_cache()


def test_reports(monkeypatch):
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    c = _case(60, 16, 8, 128, 16, 16, [200, 100], poison=False)
    _check(c, 4, *_call(c, 4))
    bad = dict(c, tables=c["tables"].clone())
    bad["tables"][0, 3] = 10 ** 6
    with pytest.raises(ValueError, match="block"):
        _call(bad, 4)
    with pytest.raises(ValueError, match="out of range"):
        _call(dict(c, lens=torch.tensor([10 ** 6, 100], dtype=torch.int32)), 4)
    with pytest.raises(ValueError, match="out of range"):
        _call(c, 4, max_context_len=150)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (c["bounds"].cuda(), c["kc"].cuda(), c["tables"].cuda())
    with pytest.raises(ValueError, match="out of range"):
        ops.paged_key_bounds_(*args, i32([0, 0]), i32([200, 100]), 16)  # more new tokens than said
    with pytest.raises(ValueError, match="block"):
        ops.paged_key_bounds_(*args[:2], bad["tables"].cuda(), i32([0, 0]), i32([200, 100]), 200)


def test_bad_pages_and_lengths_stay_in_bounds():
    """Without validation: a bad page's tokens take no part, a chunk in one ranks last, a context
    longer than its bound is cut there."""
    c = _case(61, 4, 1, 64, 16, 16, [16 * 10], poison=False)
    c["tables"][0, 4] = 10 ** 6
    out, selected = _call(c, 9)
    assert selected[0, 0].tolist() == [0, 1, 2, 3, 5, 6, 7, 8, 9] and not torch.isnan(out).any()
    c = _case(62, 4, 1, 64, 16, 16, [16 * 10], poison=False)
    cut = dict(c, lens=torch.tensor([70], dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(_call(c, 3, max_context_len=70), _call(cut, 3, max_context_len=70)))


def test_refusals():
    c = _case(63, 16, 8, 128, 32, 16, [40, 3], poison=False)
    cu = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}

    def call(top=4, **over):
        d = dict(cu, **over)
        return ops.sparse_decode_attention(*(d[k] for k in KEYS), c["scale"], top)

    for over, text in [
        (dict(top=1), "at least 2"), (dict(bounds=cu["bounds"][:, :, :, 0]), "bounds must be"),
        (dict(bounds=cu["bounds"][1:]), "bounds must be"), (dict(bounds=cu["bounds"].half()), "share a dtype"),
        (dict(bounds=cu["bounds"].transpose(3, 4).contiguous().transpose(3, 4)), "contiguous"),
        (dict(bounds=torch.zeros(cu["kc"].shape[0], 8, 4, 2, 128, dtype=torch.bfloat16, device="cuda")), "multiple of 16"),
        (dict(lens=cu["lens"].long()), "context_lens"), (dict(bounds=c["bounds"]), "must be on"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**over)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(RuntimeError, match="max_new_tokens"):
        ops.paged_key_bounds_(cu["bounds"], cu["kc"], cu["tables"], i32([0, 0]), cu["lens"], -1)
    with pytest.raises(RuntimeError, match="start_lens"):
        ops.paged_key_bounds_(cu["bounds"], cu["kc"], cu["tables"], i32([0]), cu["lens"], 1)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.paged_key_bounds_(cu["bounds"][..., :32].contiguous(), cu["kc"][..., :32].contiguous(), cu["tables"], i32([0, 0]), cu["lens"], 1)
    out, selected = call(q=cu["q"][:0], lens=cu["lens"][:0], tables=cu["tables"][:0])
    assert out.shape == (0, 16, 128) and selected.shape == (0, 8, 4)
