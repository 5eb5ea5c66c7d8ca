"""Infinite keys in shared-prefix and sparse decode attention: a row that meets a score of +inf is NaN, as
its softmax is; a score of -inf has no weight; a row of nothing but such scores is zero."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import _cache_forms as F
from tests import test_gpu_shared_prefix as P
from tests import test_gpu_sparse_attention as S

pytestmark = pytest.mark.gpu

SIGNS = torch.tensor([1.0, -1.0] * 8)
INF = float("inf")


def _expect(c, b, h, tokens):
    """Attention of request b's head h over `tokens`."""
    block, kvh = c["kc"].shape[1], h // (c["q"].shape[1] // c["kc"].shape[2])
    page = c["tables"][b].long()[tokens // block]
    return F.attention(c["q"][b, h:h + 1], c["kc"][page, tokens % block, kvh], c["vc"][page, tokens % block, kvh], c["scale"])


def _near(c, out, b, h, tokens):
    e, mean = _expect(c, b, h, tokens)
    return bool(((out[b, h:h + 1].cpu().double() - e).abs() <= F.attention_bound(out.dtype, e, mean)).all())


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
@pytest.mark.parametrize("prefix,at", [(300, 0), (300, 299), (1000, 640), (300, 305)])  # the last: behind the prefix, request 1 alone
def test_shared_prefix(variant, prefix, at):
    c = P._case(at, 16, 8, 128, 16, [(prefix, [5, 40, 3])], [20], poison=True)
    c["q"][..., 5] = SIGNS
    rows = [1] if at >= prefix else [0, 1, 2]
    for b in rows:  # the same contents wherever the prefix's copies lie
        c["kc"][c["tables"][b, at // 16], at % 16, :, 5] = INF
    out = P._call(c, variant=variant)
    expect = torch.zeros(4, 16, dtype=torch.bool)
    expect[rows] = SIGNS > 0
    assert torch.equal(torch.isnan(out).all(-1).cpu(), expect) and torch.equal(torch.isnan(out).any(-1).cpu(), expect)
    for b in range(4):
        n = int(c["lens"][b])
        tokens = torch.tensor([t for t in range(n) if not (b in rows and t == at)])
        for h in range(16):
            assert expect[b, h] or _near(c, out, b, h, tokens), (b, h)


@pytest.mark.parametrize("variant", [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256])
def test_shared_prefix_of_scores_without_weight(variant):
    """Every key of the prefix at -inf for half of the heads: these attend to what is behind it; a request
    with nothing behind it gives zeros there."""
    c = P._case(3, 16, 8, 128, 16, [(160, [33, 0, 300])], [], poison=True)
    c["q"][..., 5] = SIGNS
    c["kc"][c["tables"][0, :10].long(), :, :, 5] = -INF
    out = P._call(c, variant=variant)
    for b, own in enumerate((33, 0, 300)):
        assert bool(torch.isnan(out[b, 1::2]).all())
        if own == 0:
            assert not out[b, ::2].any()
        else:
            assert all(_near(c, out, b, h, torch.arange(160, 160 + own)) for h in range(0, 16, 2))


@pytest.mark.parametrize("top", [3, 40])
def test_sparse(top):
    c = S._case(4, 16, 8, 128, 64, 16, [500, 333], poison=True)
    c["q"][..., 5] = SIGNS
    c["kc"][c["tables"][0, 0], 3, :, 5] = INF     # the first chunk is always selected
    c["kc"][c["tables"][1, 0], 3, :, 5] = -INF
    out, selected = S._call(c, top)
    for b, bad in ((0, 0), (1, 1)):
        for h in range(16):
            if h % 2 == bad:
                assert bool(torch.isnan(out[b, h]).all()), (b, h)
                continue
            at = [t for j in selected[b, h // 2].tolist() if j >= 0 for t in range(j * 16, min(int(c["lens"][b]), j * 16 + 16)) if t != 3]
            assert _near(c, out, b, h, torch.tensor(at)), (b, h)
