"""NaN and infinite scores in ``nib_decode_attention``, both kernels: a row that meets a NaN score, or one
of +inf, is NaN as its softmax is, not zero; rows that meet none stay as they are; a score of -inf has no
weight; a row without tokens is zero. One split, a few (merged at once) and many."""

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import _cache_forms as F
from tests import test_gpu_shared_prefix as P

pytestmark = pytest.mark.gpu

VARIANTS = [ops.DECODE_CUDA_CORES, ops.DECODE_TENSOR_CORES]


def _call(c, variant, longest=0):
    return ops.decode_attention(*(c[k].cuda() for k in ("q", "kc", "vc", "lens", "tables")), c["scale"], longest, variant=variant)


def _nan_rows(out):
    some, all_ = torch.isnan(out).any(-1).cpu(), torch.isnan(out).all(-1).cpu()
    assert torch.equal(some, all_), "a row is NaN as a whole or not at all"
    return some


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 400, 3000])
def test_nan_reaches_the_rows_that_meet_it_and_no_others(variant, dim, n):
    c = P._case(n + dim, 16, 8, dim, 16, [], [n, n, 20, 0], torch.bfloat16, poison=True)
    clean = _call(c, variant, n)
    expect = torch.zeros(4, 16, dtype=torch.bool)
    c["q"][0, 7] = float("nan")
    expect[0, 7] = True
    for b, t, kvh in ((0, 0, 2), (1, n - 1, 5), (2, 11, 0)):  # the first token, the last, one in the middle
        c["kc"][c["tables"][b, t // 16], t % 16, kvh, 9] = float("nan")
        expect[b, 2 * kvh:2 * kvh + 2] = True
    out = _call(c, variant, n)
    assert torch.equal(_nan_rows(out), expect)
    assert torch.equal(out.cpu()[~expect], clean.cpu()[~expect]), "the other rows keep their bits"
    assert not out[3].any()


def test_head_dim_256():
    c = P._case(5, 8, 2, 256, 16, [], [300, 7], torch.float16, poison=True)
    c["q"][0, 1] = float("nan")
    c["kc"][c["tables"][1, 0], 3, 1, 200] = float("nan")
    expect = torch.zeros(2, 8, dtype=torch.bool)
    expect[0, 1] = True
    expect[1, 4:] = True
    assert torch.equal(_nan_rows(_call(c, ops.DECODE_AUTO)), expect)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("n,at", [(30, 3), (30, 29), (700, 650), (3000, 0)])
def test_infinite_scores(variant, n, at):
    """A key of +inf in one channel: a score of +inf for queries above 0 there, of -inf below."""
    c = P._case(n + at, 8, 4, 128, 16, [], [n], torch.bfloat16, poison=True)
    c["q"][0, :, 5] = torch.tensor([1.0, -1.0] * 4)
    c["kc"][c["tables"][0, at // 16], at % 16, :, 5] = float("inf")
    out = _call(c, variant, n)
    assert torch.equal(_nan_rows(out), torch.tensor([[True, False] * 4]))
    keep = torch.tensor([t for t in range(n) if t != at])
    page = c["tables"][0].long()[keep // 16]
    for h in range(1, 8, 2):
        e, mean = F.attention(c["q"][0, h:h + 1], c["kc"][page, keep % 16, h // 2], c["vc"][page, keep % 16, h // 2], c["scale"])
        assert bool(((out[0, h:h + 1].cpu().double() - e).abs() <= F.attention_bound(out.dtype, e, mean)).all())


def test_shared_prefix_and_dense_agree_on_nan():
    c = P._case(16, 16, 8, 128, 16, [(300, [5, 40, 3])], [20], poison=True)
    c["q"][1, 7] = float("nan")
    c["kc"][c["tables"][0, 3], 2, 5, 9] = float("nan")
    dense = [_nan_rows(_call(c, v)) for v in VARIANTS]
    shared = _nan_rows(P._call(c))
    assert torch.equal(dense[0], dense[1]) and torch.equal(dense[0], shared) and int(shared.sum()) == 7
