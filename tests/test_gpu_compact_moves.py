"""What a program keeps beside the cache follows a compaction: ``paged_compact``'s moves through
``paged_copy_blocks``, in one call or, in pools of more than 131,073 blocks, in pieces."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import _cache_forms as F

pytestmark = pytest.mark.gpu

PAIRS = 65536


@pytest.mark.parametrize("blocks", [1000, 131072, 131073, 150001])
@pytest.mark.parametrize("load", [0.5, 0.999])   # a quarter of the blocks move; a hundred or fewer in a long padded list
def test_moves_in_pieces(blocks, load):
    g = torch.Generator().manual_seed(blocks)
    refs = (torch.rand(blocks, generator=g) < load).to(torch.int32)
    cache = torch.randint(0, 2 ** 31 - 1, (2, blocks, 1, 1, 2), generator=g, dtype=torch.int32)
    beside = torch.randint(0, 2 ** 31 - 1, (blocks, 3, 2), generator=g, dtype=torch.int32)
    _, _, live, moves = F.compact([[]], refs.tolist())
    src, dst = (torch.tensor(v, dtype=torch.long) for v in zip(*moves))
    e_cache, e_beside = cache.clone(), beside.clone()
    e_cache[:, dst], e_beside[dst] = cache[:, src], beside[src]
    c, b = cache.cuda(), beside.cuda()
    _, _, got_live, got = ops.paged_compact(c, torch.full((1, 1), -1, dtype=torch.int32, device="cuda"), refs.cuda())
    for s, d in zip(*(m.split(PAIRS) for m in got)):
        ops.paged_copy_blocks(b, s, d, block_dim=0)
    assert got_live.tolist() == [live] and torch.equal(c.cpu(), e_cache) and torch.equal(b.cpu(), e_beside)
    if got.shape[1] > PAIRS:
        with pytest.raises(RuntimeError, match="at most 65536 pairs"):
            ops.paged_copy_blocks(b, got[0], got[1], block_dim=0)
