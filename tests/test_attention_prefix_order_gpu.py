"""GPU test of the order of a shared prefix's kernels behind the stream's earlier work: the kernel of
the requests' own tokens starts while the prefix kernel runs, and reads queries, lengths, tables
and caches that were written just before the call."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from paged_reference import Cache, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True], ids=["stream", "graph"])
@pytest.mark.parametrize("d", [64, 128])
def test_reads_what_was_just_written(d, captured):
    # three sets of inputs of one shape, each of which the formula gives another result for
    batch, prefix, page = 150, 1100 * 128 // d, 32
    sets = []
    for seed in range(3):
        lengths = [(37 * i + 11 * seed) % 90 for i in range(batch)]
        cache = Cache(lengths, 2, d, page, torch.bfloat16, prefix=prefix, columns=3, seed=seed)
        sets.append((cache, queries(batch, 6, d, torch.bfloat16, seed=10 + seed).cuda()))
    pages = max(c.k.shape[0] for c, _ in sets)
    k, v = (torch.zeros((pages, 2, page, d), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.zeros((batch, 3), device="cuda", dtype=torch.int32)
    own = torch.zeros(batch, device="cuda", dtype=torch.int32)
    first = torch.zeros(-(-prefix // page), device="cuda", dtype=torch.int32)
    q = torch.zeros_like(sets[0][1])
    rows = []  # every row of a cache, which append_kv writes to the slots in order
    for cache, query in sets:
        flat = [x.transpose(1, 2).reshape(-1, 2, d) for x in (cache.k, cache.v)]
        rows.append((*flat, torch.arange(len(flat[0]), device="cuda", dtype=torch.int32),
                     cache.table.cuda(), cache.lengths.cuda(), cache.pages(), query))

    def step(i):
        ks, vs, slots, t, n, p, query = rows[i]
        for to, x in ((table, t), (own, n), (first, p), (q, query)):
            to.copy_(x)
        mfa.append_kv(ks, vs, k, v, slots)  # the launch in front of the attention's
        return mfa.shared_prefix_attention(q, k, v, first, prefix, table, own)

    want = []
    for i, (cache, query) in enumerate(sets):
        out = step(i)
        torch.cuda.synchronize()
        check(out, *cache.reference(query))
        want.append(out.clone())
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [(i % 3, step(i % 3)) for i in range(12)]
        for _ in range(8):
            graph.replay()
    else:
        outs = [(i % 3, step(i % 3)) for i in range(100)]
    for i, out in outs:
        assert torch.equal(out, want[i])
