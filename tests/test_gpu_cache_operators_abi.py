"""Shared-prefix and sparse decode attention through the C ABI, into outputs of the caller's own layout:
any strides, an address of two-byte alignment. ``nib_decode_attention`` takes the same with the same struct."""

import ctypes

import pytest
import torch

from nano_vllm_multimodal_b200 import _lib, ops
from tests import test_gpu_shared_prefix as P
from tests import test_gpu_sparse_attention as S
from tests.test_cache_operators_host import DecodeArgs, SharedPrefixArgs, SparseArgs

pytestmark = pytest.mark.gpu

GUARD = 7.0


@pytest.fixture(scope="module")
def lib():
    lib = _lib.cdll()
    lib.nib_last_error.restype = ctypes.c_char_p
    for name in ("nib_shared_prefix_workspace_bytes", "nib_sparse_decode_workspace_bytes", "nib_decode_attention_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_int64
    for name in ("nib_shared_prefix_decode_attention", "nib_sparse_decode_attention", "nib_decode_attention"):
        getattr(lib, name).argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    return lib


def _args(d, out, strides):
    q, kc = d["q"], d["kc"]
    return DecodeArgs(struct_size=ctypes.sizeof(DecodeArgs), dtype=2 if q.dtype == torch.bfloat16 else 1, batch=q.shape[0],
                      num_heads=q.shape[1], num_kv_heads=kc.shape[2], head_dim=q.shape[2], q=q.data_ptr(),
                      q_batch_stride=q.stride(0), q_head_stride=q.stride(1), key_cache=kc.data_ptr(),
                      value_cache=d["vc"].data_ptr(), cache_block_stride=kc.stride(0), cache_slot_stride=kc.stride(1),
                      cache_head_stride=kc.stride(2), num_blocks=kc.shape[0], block_size=kc.shape[1],
                      block_tables=d["tables"].data_ptr(), block_table_stride=d["tables"].stride(0),
                      max_blocks_per_seq=d["tables"].shape[1], context_lens=d["lens"].data_ptr(), scale=d["scale"],
                      out=out, out_batch_stride=strides[0], out_head_stride=strides[1])


def _run(lib, name, s, attn):
    size = {"nib_decode_attention": "nib_decode_attention_workspace_bytes", "nib_shared_prefix_decode_attention":
            "nib_shared_prefix_workspace_bytes", "nib_sparse_decode_attention": "nib_sparse_decode_workspace_bytes"}[name]
    need = getattr(lib, size)(ctypes.byref(s))
    ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    attn.workspace, attn.workspace_bytes = ws.data_ptr(), need
    rc = getattr(lib, name)(ctypes.byref(s), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.nib_last_error().decode()
    torch.cuda.synchronize()


# (elements in front of the output, spare elements behind a head, behind a request)
LAYOUTS = [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (3, 5, 7), (2, 2, 2)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("requests", [3, 170])   # of 16 heads: few rows, and more than 16 an SM
def test_outputs_of_any_layout(lib, layout, requests):
    front, head_gap, batch_gap = layout
    heads, dim = 16, 64
    head_stride = dim + head_gap
    strides = (heads * head_stride + batch_gap, head_stride)
    prefix = P._case(91, heads, 1, dim, 16, [(100, [i % 20 for i in range(requests)])], [], poison=False)
    sparse = S._case(92, heads, 1, dim, 16, 16, [30 + 7 * i % 300 for i in range(requests)], poison=False)
    for name, c in (("nib_shared_prefix_decode_attention", prefix), ("nib_sparse_decode_attention", sparse),
                    ("nib_decode_attention", prefix)):
        d = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}
        buf = torch.full((front + requests * strides[0] + 8,), GUARD, dtype=torch.bfloat16, device="cuda")
        attn = _args(d, buf.data_ptr() + 2 * front, strides)
        if name == "nib_decode_attention":
            _run(lib, name, attn, attn)
        elif name == "nib_sparse_decode_attention":
            selected = torch.empty(requests, 1, 12, dtype=torch.int32, device="cuda")
            s = SparseArgs(struct_size=ctypes.sizeof(SparseArgs), chunk=16, top_chunks=12, attn=attn, bounds=d["bounds"].data_ptr(),
                           bounds_block_stride=d["bounds"].stride(0), bounds_head_stride=d["bounds"].stride(1),
                           selected=selected.data_ptr())
            _run(lib, name, s, s.attn)
        else:
            s = SharedPrefixArgs(struct_size=ctypes.sizeof(SharedPrefixArgs), attn=attn, num_groups=1,
                                 group_offsets=d["offsets"].data_ptr(), prefix_lens=d["prefix"].data_ptr())
            _run(lib, name, s, s.attn)
        out = buf[front:front + requests * strides[0]].as_strided((requests, heads, dim), (strides[0], strides[1], 1), front)
        if name == "nib_sparse_decode_attention":
            S._check(c, 12, out, selected, f"{name} {layout}")
        else:
            P._check(c, out, f"{name} {layout}")
        out.fill_(GUARD)
        assert bool((buf == GUARD).all()), "nothing is written between the heads"


def test_the_library_and_the_binding_agree(lib):
    """A contiguous output through the C ABI holds the binding's bits."""
    c = P._case(93, 16, 2, 128, 16, [(300, [i % 20 for i in range(20)])], [], poison=False)
    d = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}
    out = torch.empty_like(d["q"])
    s = SharedPrefixArgs(struct_size=ctypes.sizeof(SharedPrefixArgs), attn=_args(d, out.data_ptr(), (16 * 128, 128)), num_groups=1,
                         group_offsets=d["offsets"].data_ptr(), prefix_lens=d["prefix"].data_ptr())
    _run(lib, "nib_shared_prefix_decode_attention", s, s.attn)
    assert torch.equal(out, ops.shared_prefix_decode_attention(*(d[k] for k in ("q", "kc", "vc", "lens", "tables", "offsets",
                                                                                "prefix", "scale"))))
