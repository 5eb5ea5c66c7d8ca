"""Page operators, shared-prefix and sparse decode attention on the host: what the C ABI refuses
before any launch, CPU tensors, and the tests' own plain forms."""

import ctypes

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from nano_vllm_multimodal_b200._lib import load_ops
from tests import _cache_forms as F

i64, vp = ctypes.c_int64, ctypes.c_void_p
SOME = vp(4096)  # an address that is never looked at: every call below is refused


@pytest.fixture(scope="module")
def lib():
    from nano_vllm_multimodal_b200 import _build
    _build.build()
    lib = ctypes.CDLL(str(_build.LIB))
    lib.nib_last_error.restype = ctypes.c_char_p
    for name in ("nib_paged_fork_workspace_bytes", "nib_paged_compact_workspace_bytes",
                 "nib_shared_prefix_workspace_bytes", "nib_sparse_decode_workspace_bytes"):
        getattr(lib, name).restype = i64
    return lib


class DecodeArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("dtype", ctypes.c_int32), ("batch", i64),
                ("num_heads", ctypes.c_int32), ("num_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("variant", ctypes.c_int32), ("q", vp), ("q_batch_stride", i64), ("q_head_stride", i64),
                ("key_cache", vp), ("value_cache", vp), ("cache_block_stride", i64), ("cache_slot_stride", i64),
                ("cache_head_stride", i64), ("num_blocks", i64), ("block_size", i64), ("block_tables", vp),
                ("block_table_stride", i64), ("max_blocks_per_seq", i64), ("context_lens", vp),
                ("scale", ctypes.c_float), ("reserved2", ctypes.c_int32), ("out", vp), ("out_batch_stride", i64),
                ("out_head_stride", i64), ("workspace", vp), ("workspace_bytes", i64), ("max_context_len", i64),
                ("status", vp)]


class SharedPrefixArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("reserved", ctypes.c_int32), ("attn", DecodeArgs),
                ("group_offsets", vp), ("prefix_lens", vp), ("num_groups", i64), ("max_prefix_len", i64)]


class SparseArgs(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("chunk", ctypes.c_int32), ("top_chunks", ctypes.c_int32),
                ("reserved", ctypes.c_int32), ("attn", DecodeArgs), ("bounds", vp), ("bounds_block_stride", i64),
                ("bounds_head_stride", i64), ("selected", vp)]


def _decode(**over):
    a = DecodeArgs(struct_size=ctypes.sizeof(DecodeArgs), dtype=2, batch=3, num_heads=16, num_kv_heads=8, head_dim=128,
                   block_size=256, num_blocks=10, max_blocks_per_seq=4, block_table_stride=4, scale=0.1)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_attention_arguments(lib):
    def prefix(groups=1, size=ctypes.sizeof(SharedPrefixArgs), **over):
        s = SharedPrefixArgs(struct_size=size, attn=_decode(**over), num_groups=groups)
        return lib.nib_shared_prefix_decode_attention(ctypes.byref(s), None), lib.nib_last_error().decode()

    def sparse(chunk=32, top=4, size=ctypes.sizeof(SparseArgs), **over):
        s = SparseArgs(struct_size=size, chunk=chunk, top_chunks=top, attn=_decode(**over))
        return lib.nib_sparse_decode_attention(ctypes.byref(s), None), lib.nib_last_error().decode()

    for call in (prefix, sparse):
        assert call(size=8) == (1, call(size=8)[1]) and "struct size" in call(size=8)[1]
        assert call(struct_size=8)[0] == 1
        assert call()[0] == 1 and "null pointer" in call()[1]
        assert call(dtype=0)[0] == 1 and "bf16 or f16" in call(dtype=0)[1]
        assert call(head_dim=96)[0] == 1 and call(num_heads=12)[0] == 1 and call(batch=-1)[0] == 1
        assert call(batch=0) [0] == 0
    assert "group count" in prefix(groups=-1)[1]
    for chunk in (0, 8, 24, 96, 512):
        assert sparse(chunk=chunk)[0] == 1 and "chunk" in sparse(chunk=chunk)[1]
    assert "two chunks" in sparse(top=1)[1]
    s = SparseArgs(struct_size=1)
    assert lib.nib_sparse_decode_workspace_bytes(ctypes.byref(s)) == -1
    assert lib.nib_shared_prefix_workspace_bytes(ctypes.byref(SharedPrefixArgs())) == -1
    s = SparseArgs(struct_size=ctypes.sizeof(SparseArgs), chunk=32, top_chunks=64, attn=_decode(max_blocks_per_seq=64))
    for batch, groups in ((0, 0), (0, 3), (1, 0)):  # no request, no group: nothing to divide the work by
        empty = SharedPrefixArgs(struct_size=ctypes.sizeof(SharedPrefixArgs), attn=_decode(batch=batch), num_groups=groups)
        assert lib.nib_shared_prefix_workspace_bytes(ctypes.byref(empty)) >= 0
    empty = SparseArgs(struct_size=ctypes.sizeof(SparseArgs), chunk=32, top_chunks=4, attn=_decode(batch=0))
    assert lib.nib_sparse_decode_workspace_bytes(ctypes.byref(empty)) == 0
    keys = 3 * 8 * (64 * 256 // 32) * 8  # 64-bit keys of every chunk
    assert lib.nib_sparse_decode_workspace_bytes(ctypes.byref(s)) >= keys


def test_decode_workspace_of_an_empty_batch(lib):
    lib.nib_decode_attention_workspace_bytes.restype = i64
    assert lib.nib_decode_attention_workspace_bytes(ctypes.byref(_decode(batch=0))) == 0


def test_page_arguments(lib):
    bad = [
        (lib.nib_paged_copy_blocks, (SOME, i64(2), i64(1 << 20), i64(4), i64(64), None, None, i64(1), None, None), "null pointer"),
        (lib.nib_paged_copy_blocks, (SOME, i64(2), i64(64), i64(4), i64(64), SOME, SOME, i64(1), None, None), "overlap"),
        (lib.nib_paged_copy_blocks, (SOME, i64(2), i64(1 << 20), i64(4), i64(64), SOME, SOME, i64(-1), None, None), "negative"),
        (lib.nib_paged_copy_blocks, (SOME, i64(1), i64(0), i64(4), i64(63), SOME, SOME, i64(1), None, None), "even"),
        (lib.nib_paged_copy_blocks, (SOME, i64(1), i64(0), i64(4), i64(64), SOME, SOME, i64(70000), None, None), "65536"),
        (lib.nib_paged_free, (SOME, i64(4), i64(-1), i64(4), i64(16), SOME, SOME, i64(4), SOME, i64(1), SOME, SOME, SOME, None, None), "bad sizes"),
        (lib.nib_paged_free, (SOME, i64(4), i64(2), i64(4), i64(16), SOME, SOME, i64(4), None, i64(1), SOME, SOME, SOME, None, None), "null pointer"),
        (lib.nib_paged_compact, (SOME, i64(1), i64(0), i64(4), i64(64), SOME, i64(4), i64(2), i64(4), SOME, SOME, SOME, SOME, SOME, SOME, i64(0), None, None), "workspace"),
        (lib.nib_paged_compact, (SOME, i64(1), i64(0), i64(4), i64(64), SOME, i64(4), i64(2), i64(4), SOME, SOME, SOME, None, SOME, SOME, i64(99), None, None), "null pointer"),
        (lib.nib_paged_fork, (SOME, i64(1), i64(0), i64(4), i64(64), i64(16), SOME, i64(4), i64(2), i64(4), SOME, SOME, SOME, SOME, i64(1), SOME, SOME, SOME, SOME, SOME, i64(1), None, None), "workspace"),
        (lib.nib_paged_fork, (SOME, i64(1), i64(0), i64(4), i64(64), i64(24), SOME, i64(4), i64(2), i64(4), SOME, SOME, SOME, SOME, i64(1), SOME, SOME, SOME, SOME, SOME, i64(99), None, None), "whole slots"),
    ]
    for fn, args, text in bad:
        assert fn(*args) != 0 and text in lib.nib_last_error().decode(), (fn.__name__, text, lib.nib_last_error())
    assert lib.nib_paged_fork_workspace_bytes(i64(-1), i64(2)) == -1
    assert lib.nib_paged_compact_workspace_bytes(i64(-1)) == -1


def test_cpu_tensors_raise():
    load_ops()
    x = torch.zeros(2, 4, 16, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 2, dtype=torch.int32)
    q, b = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.paged_copy_blocks(x, i, i), lambda: ops.paged_fork(x, t, i, i, i, i),
                 lambda: ops.paged_free(t, i, i, i, 16), lambda: ops.paged_compact(x, t, i),
                 lambda: ops.shared_prefix_decode_attention(q, x[0], x[1], i, t, i, i[:1], 0.1),
                 lambda: ops.sparse_decode_attention(q, x[0], x[1], b, i, t, 0.1, 2),
                 lambda: ops.paged_key_bounds_(b, x[0], t, i, i, 1)):
        with pytest.raises(NotImplementedError):
            call()


def test_plain_forms():
    """The tests' own forms on a case worked out by hand."""
    tables, lens, refs, copies = F.fork(4, [[0, 2], [-1, -1], [-1, -1]], [6, 0, 0], [1, 0, 1, 0, 0], [0, 0], [2, 1])
    assert tables == [[0, 2], [0, 3], [0, 1]] and lens == [6, 6, 6] and refs == [3, 1, 1, 1, 0]
    assert copies == [(2, 1, 2), (2, 3, 2)]
    assert F.release(4, tables, lens, refs, [0, 0, -1]) == ([[-1, -1], [0, 3], [0, 1]], [0, 6, 6], [2, 1, 0, 1, 0])
    assert F.compact([[4, 0, -1], [6, -1, -1]], [1, 0, 0, 0, 2, 0, 1]) == ([[1, 0, -1], [2, -1, -1]], [1, 2, 1, 0, 0, 0, 0], 3, [(4, 1), (6, 2)])
    # one channel: q = (2, -1), boxes [lo, hi] = [0, 1], [-3, 0], [1, 2], [0, 0]: scores 2, 3, 3, 0
    q = torch.tensor([[[2.0], [-1.0]]])
    box = torch.tensor([[0.0, 1.0], [-3.0, 0.0], [1.0, 2.0], [0.0, 0.0]]).view(4, 1, 1, 2, 1)
    tables = torch.arange(4, dtype=torch.int32)[None]
    assert F.select_chunks(q, box, tables, [16 * 4], 16, 3).tolist() == [[[0, 1, 3]]]
    assert F.select_chunks(q, box, tables, [16 * 2 + 1], 16, 5).tolist() == [[[0, 1, 2, -1, -1]]]
