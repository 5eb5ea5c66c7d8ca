"""Validation mode of the cache operators: every wrong argument that the header names is reported, wherever
in its list it stands, and correct calls report nothing."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import test_gpu_shared_prefix as P

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
