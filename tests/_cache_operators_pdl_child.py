"""Child process of tests/test_gpu_cache_operators_pdl.py: one serving step after another through the cache
operators, each reading what the kernel before it wrote, eagerly and replayed from a CUDA graph; prints a
sha256 of every output as JSON. The parent runs it with programmatic dependent launch off and on
(``NIB_B200_PDL`` is read once per process).

A step: store a token per request, refresh the key bounds, sparse attention, shared-prefix attention by both
prefix kernels (the second launches its suffixes next to the prefixes), fork, release, compact, and the
bounds' blocks after them.

Usage: python tests/_cache_operators_pdl_child.py
"""

import hashlib
import json
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from nano_vllm_multimodal_b200 import ops  # noqa: E402

BLOCK, CHUNK, NQ, NKV, DIM = 32, 16, 16, 2, 128
REQUESTS, SPARE, WIDTH, BLOCKS, PREFIX = 24, 8, 80, 2400, 2000


def digest(tensors):
    h = hashlib.sha256()
    for t in tensors:
        h.update(t.detach().contiguous().cpu().view(torch.uint8).numpy().tobytes())
    return h.hexdigest()


def main():
    torch.cuda.set_device(0)
    g = torch.Generator().manual_seed(5)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    cache0 = torch.randn(2, BLOCKS, BLOCK, NKV, DIM, generator=g).to(torch.bfloat16).cuda()
    order = torch.randperm(BLOCKS, generator=g).tolist()
    tables = torch.full((REQUESTS + SPARE, WIDTH), -1, dtype=torch.int32)
    shared = [order.pop() for _ in range(PREFIX // BLOCK)]
    lens = torch.zeros(REQUESTS + SPARE, dtype=torch.int32)
    refs = torch.zeros(BLOCKS, dtype=torch.int32)
    for b in range(REQUESTS):
        lens[b] = PREFIX + 20 + 17 * b
        row = shared + [order.pop() for _ in range(-(-int(lens[b] + 8) // BLOCK) - len(shared))]
        tables[b, :len(row)] = torch.tensor(row)
        for p in row:
            refs[p] += 1
    tables, lens, refs = tables.cuda(), lens.cuda(), refs.cuda()
    offsets, prefix = i32([0, 10, REQUESTS]), i32([PREFIX // BLOCK * BLOCK, PREFIX // BLOCK * BLOCK])
    parents, children, gone = i32([0, 3, 3, 9]), i32([REQUESTS, REQUESTS + 2, REQUESTS + 3, REQUESTS + 5]), i32([5, 17, REQUESTS + 2])
    steps = 3
    q = torch.randn(steps, REQUESTS, NQ, DIM, generator=g).to(torch.bfloat16).cuda()
    k, v = (torch.randn(steps, REQUESTS, NKV, DIM, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    slots = []
    for s in range(steps):
        at = (lens[:REQUESTS] + s).long()
        slots.append((tables[:REQUESTS].gather(1, (at // BLOCK)[:, None])[:, 0].long() * BLOCK + at % BLOCK).to(torch.int32))
    many = [(lens[:REQUESTS] + s + 1).to(torch.int32) for s in range(steps)]
    before = [(m - 1).to(torch.int32) for m in many]
    all_lens = torch.cat([many[-1], lens[REQUESTS:]])
    cache, bounds = cache0.clone(), torch.zeros(BLOCKS, NKV, BLOCK // CHUNK, 2, DIM, dtype=torch.bfloat16, device="cuda")
    zero = torch.zeros_like(lens[:REQUESTS])

    def chain():
        cache.copy_(cache0)
        bounds.zero_()
        outs = []
        t = tables[:REQUESTS]
        ops.paged_key_bounds_(bounds, cache[0], t, zero, lens[:REQUESTS], PREFIX + 20 + 17 * REQUESTS)
        for s in range(steps):
            ops.paged_store(k[s], v[s], cache[0], cache[1], slots[s])
            ops.paged_key_bounds_(bounds, cache[0], t, before[s], many[s], 1)
            outs += ops.sparse_decode_attention(q[s], cache[0], cache[1], bounds, many[s], t, DIM ** -0.5, 24)
            for variant in (ops.PREFIX_ROWS16, ops.PREFIX_ROWS256):
                outs.append(ops.shared_prefix_decode_attention(q[s], cache[0], cache[1], many[s], t, offsets, prefix, DIM ** -0.5,
                                                               variant=variant))
            outs.append(ops.shared_prefix_decode_attention(outs[-1], cache[0], cache[1], many[s], t, offsets, prefix, DIM ** -0.5,
                                                           variant=ops.PREFIX_ROWS256))
        ft, fl, fr, copies = ops.paged_fork(cache, tables, all_lens, refs, parents, children)
        ops.paged_copy_blocks(bounds, copies[0], copies[1], block_dim=0)
        ft, fl, fr = ops.paged_free(ft, fl, fr, gone, BLOCK)
        ft, fr, live, moves = ops.paged_compact(cache, ft, fr)
        ops.paged_copy_blocks(bounds, moves[0], moves[1], block_dim=0)
        outs += ops.sparse_decode_attention(q[0], cache[0], cache[1], bounds, fl[8:], ft[8:], DIM ** -0.5, 24)
        return outs + [ft, fl, fr, live, moves, copies, cache, bounds]

    eager = [digest(chain()) for _ in range(2)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    replayed = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        replayed.append(digest(captured))
    del graph
    finite = all(bool(torch.isfinite(t).all()) for t in captured if t.is_floating_point())
    print(json.dumps({"eager": eager, "graph": replayed, "finite": finite}))


if __name__ == "__main__":
    main()
