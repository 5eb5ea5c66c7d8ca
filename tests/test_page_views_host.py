"""Which cache views the page operators refuse, on the host. The operators' CUDA bodies are entered with
CPU tensors: a view is looked at before anything touches a device, and a CPU tensor gets no further than that."""

import pytest
import torch

from nano_vllm_multimodal_b200._lib import load_ops

B, BLOCK = 24, 16
INTS = [torch.zeros(3, dtype=torch.int32)] * 2


def _enter(name, cache):
    """What the CUDA body of page operator ``name`` says of ``cache``."""
    load_ops()
    refs, tables, lens = torch.zeros(B, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    args = {"paged_copy_blocks": (cache, *INTS, -4, None), "paged_fork": (cache, tables, lens, refs, *INTS, -4, None),
            "paged_compact": (cache, tables, refs, -4, None)}[name]
    op = getattr(torch.ops.nanoinfer_b200, name).default
    with pytest.raises(Exception) as e:
        op.redispatch(torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA), *args)
    return str(e.value)


OPS = ["paged_copy_blocks", "paged_fork", "paged_compact"]
REFUSAL = "the dims before the blocks must have one stride"


@pytest.mark.parametrize("name", OPS)
@pytest.mark.parametrize("sizes", [
    (2, 3),        # a real outer dim, an expanded one inside it: six planes where the storage has two
    (3,),          # one expanded dim
    (2, 1, 3),     # a dim of one between them
])
def test_expanded_planes_are_refused(name, sizes):
    inner = torch.zeros((2,) + (1,) * (len(sizes) - 1) + (B, BLOCK, 2, 64), dtype=torch.bfloat16)
    cache = inner.expand(*sizes, B, BLOCK, 2, 64) if len(sizes) > 1 else inner[:1].expand(3, B, BLOCK, 2, 64)
    assert REFUSAL in _enter(name, cache)


@pytest.mark.parametrize("name", OPS)
def test_views_without_one_plane_stride_are_refused(name):
    cache = torch.zeros(4, 3, B, BLOCK, 2, 64, dtype=torch.bfloat16)
    assert REFUSAL in _enter(name, cache[:, :2])                       # a gap between the outer dim's planes
    assert REFUSAL in _enter(name, cache.transpose(0, 1))              # the outer dims in another order
    assert REFUSAL in _enter(name, cache[:1].expand(5, 3, B, BLOCK, 2, 64))  # the outer dim expanded
    assert "contiguous" in _enter(name, cache[..., :32])
    assert "one behind the other" in _enter(name, cache[:, :, ::2])


@pytest.mark.parametrize("name", OPS)
def test_views_with_one_plane_stride_pass(name):
    cache = torch.zeros(2, 4, B, BLOCK, 2, 64, dtype=torch.bfloat16)
    for view in (cache, cache[:, 2], cache[1:2], cache[0], cache[:, 1:2], cache[0, 3]):
        said = _enter(name, view)
        assert "stride" not in said and "contiguous" not in said and "one behind" not in said, said
