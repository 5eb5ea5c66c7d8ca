"""Validation mode of the cache operators: every wrong argument that the header names is reported, wherever
in its list it stands, and correct calls report nothing."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import _cache_forms as F
from tests import test_gpu_shared_prefix as P
from tests import test_gpu_sparse_attention as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
@pytest.mark.parametrize("groups", [1, 3, 40, 100])
def test_a_bad_group_is_reported_wherever_it_stands(monkeypatch, variant, groups):
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    c = P._case(groups, 16, 8, 128, 16, [(20, [i % 3] if i % 5 else []) for i in range(groups)], [4], poison=False)
    P._check(c, P._call(c, variant=variant))
    last = int(c["offsets"][-1])
    for g in {0, groups // 2, groups - 1}:
        for name, at, value in (("prefix", g, -1), ("offsets", g + 1, last + 2), ("offsets", g, -1)):
            bad = c[name].clone()
            bad[at] = value
            with pytest.raises(ValueError, match="out of range"):
                P._call(dict(c, **{name: bad}), variant=variant)
        if 0 < g < groups - 1:  # a decreasing offset in the middle
            bad = c["offsets"].clone()
            bad[g + 1] = 0
            if int(bad[g]) > 0:
                with pytest.raises(ValueError, match="out of range"):
                    P._call(dict(c, offsets=bad), variant=variant)


@pytest.mark.parametrize("chunk", [1, 16, 64])
@pytest.mark.parametrize("new", [1, 2, 17, 64, 150])
def test_more_new_tokens_than_said_are_reported(monkeypatch, chunk, new):
    """One token more than the bound is reported even where it lies in a chunk that is refreshed anyway, and
    where the bound says that there are none; the bound itself, and more than there are, report nothing."""
    monkeypatch.setenv("NANOINFER_B200_VALIDATE", "1")
    c = S._case(chunk + new, 2, 2, 64, 64, 64, [150, 40, 0], poison=False)
    kc, tables, lens = c["kc"].cuda(), c["tables"].cuda(), c["lens"].cuda()
    starts = lens - torch.tensor([new, 0, 0], dtype=torch.int32, device="cuda")
    before = torch.full((kc.shape[0], 2, 64 // chunk, 2, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    e = F.key_bounds(c["kc"], before.cpu(), c["tables"], starts.tolist(), lens.tolist())
    for most in (new, new + 1, 10 ** 9):
        assert torch.equal(ops.paged_key_bounds_(before.clone(), kc, tables, starts, lens, most).cpu(), e)
    for most in {0, new - 1}:
        with pytest.raises(ValueError, match="out of range"):
            ops.paged_key_bounds_(before.clone(), kc, tables, starts, lens, most)
    assert torch.equal(ops.paged_key_bounds_(before.clone(), kc, tables, lens, lens, 0), before)
