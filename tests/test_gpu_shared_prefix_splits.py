"""Shared-prefix decode attention where a request has much to itself: outside the groups, shorter than its
group's prefix, in a group of a short prefix, and calls without host bounds. Each such request's tokens are
split over CTAs by how many it has, whatever the bounds say."""

import ctypes

import pytest
import torch

from nano_vllm_multimodal_b200 import ops
from tests import test_gpu_shared_prefix as P

pytestmark = pytest.mark.gpu

VARIANTS = [ops.PREFIX_ROWS16, ops.PREFIX_ROWS256]


def _all_bounds(c):
    n, p = int(c["lens"].max()), int(c["prefix"].max()) if len(c["prefix"]) else 0
    return [{}, dict(max_prefix_len=p, max_context_len=n), dict(max_context_len=n), dict(max_prefix_len=max(p, 1)),
            dict(max_prefix_len=1, max_context_len=1)]


@pytest.mark.parametrize("nq,nkv,dim", [(16, 8, 128), (8, 1, 64)])
@pytest.mark.parametrize("variant", VARIANTS)
def test_own_tokens_around_the_split_sizes(nq, nkv, dim, variant):
    """Own tokens of 0, 1, and one to either side of the multiples of 256 that count the splits in use."""
    own = [0, 1, 255, 256, 257, 511, 512, 513, 1024, 1025, 2700]
    c = P._case(nq, nq, nkv, dim, 16, [(333, own)], [1, 256, 257, 3000], poison=True)
    for bounds in _all_bounds(c):
        P._check(c, P._call(c, variant=variant, **bounds), str(bounds))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("groups,alone", [
    ([], [9000, 1]),                                  # no groups
    ([(300, [20, 3])], [12000]),                      # a long request in no group
    ([(40, [9000, 5, 0]), (8000, [7, 30])], []),      # a short prefix next to a long one
    ([(0, [5000, 2]), (600, [1] * 30)], [4000, 0]),   # an empty prefix
])
def test_long_own_contexts(variant, groups, alone):
    c = P._case(len(alone) + len(groups), 16, 8, 128, 64, groups, alone, poison=True)
    for bounds in _all_bounds(c):
        out = P._call(c, variant=variant, **bounds)
        P._check(c, out, str(bounds))
        assert torch.equal(out, P._call(c, variant=variant, **bounds))


@pytest.mark.parametrize("variant", VARIANTS)
def test_a_request_shorter_than_its_groups_prefix(variant):
    c = P._case(4, 16, 8, 128, 64, [(9000, [4, 9, 30])], [], poison=False)
    c["lens"][1] = 8990
    for bounds in _all_bounds(c):
        P._check(c, P._call(c, variant=variant, **bounds), str(bounds))


def test_replayed_with_other_lengths():
    """How many splits are in use goes by the lengths on the device: one graph, short and long contexts."""
    c = P._case(6, 16, 8, 128, 64, [(500, [2500, 1, 300])], [3000], poison=False)
    d = {k: (v.cuda() if torch.is_tensor(v) else v) for k, v in c.items()}
    call = lambda: ops.shared_prefix_decode_attention(*(d[k] for k in ("q", "kc", "vc", "lens", "tables", "offsets", "prefix", "scale")))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([3000, 501, 800, 3000], [501, 501, 756, 1], [757, 500, 499, 0], [0, 0, 0, 257], [3000, 501, 800, 3000]):
        c["lens"] = torch.tensor(lens, dtype=torch.int32)
        d["lens"].copy_(c["lens"])
        graph.replay()
        torch.cuda.synchronize()
        P._check(c, out, str(lens))
    del graph


def test_splits_are_planned_for_what_a_request_may_have():
    """The workspace holds each split's partials: one request of up to 32,768 tokens, in no group or without
    host bounds, gets as many splits as the SMs take."""
    from nano_vllm_multimodal_b200 import _lib
    from tests.test_cache_operators_host import SharedPrefixArgs, _decode
    size = _lib.cdll().nib_shared_prefix_workspace_bytes
    size.restype = ctypes.c_int64
    one = 16 * (128 + 2) * 4  # a split's partials of 16 heads
    for groups in (0, 1):
        s = SharedPrefixArgs(struct_size=ctypes.sizeof(SharedPrefixArgs), attn=_decode(batch=1, max_blocks_per_seq=128),
                             num_groups=groups)
        assert size(ctypes.byref(s)) >= (30 + 30 * groups) * one
