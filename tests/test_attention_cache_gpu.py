"""GPU tests of the paged cache's extension: block tables and slots against a loop over the tokens,
the copy of k and v bit for bit, and a generation that runs prompt, cache and decoding together."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi
from window_reference import reference

pytestmark = pytest.mark.gpu


def loop(table, cached, added, free, page, capacity):
    """The contract of extend_block_tables, token by token."""
    table = [list(row) for row in table]
    slots, starts, used = [], [0], 0
    for row, c, a in zip(table, cached, added):
        c, a = max(0, c), max(0, a)
        columns = len(row)
        for column in range(min(columns, -(-c // page)), min(columns, -(-(c + a) // page))):
            row[column] = free[used] if used < len(free) else -1
            used += 1
        for p in range(c, c + a):
            at = row[p // page] if p // page < columns else -1
            slots.append(at * page + p % page if at >= 0 else -1)
        starts.append(len(slots))
    slots = (slots + [-1] * capacity)[:capacity]
    return table, slots, starts, [used]


def run_both(cached, added, page, columns, free, capacity, seed=0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randint(0, 1000, (len(cached), columns), generator=g, dtype=torch.int32)
    gpu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    mine = table.cuda()
    got = mfa.extend_block_tables(mine, gpu(cached), gpu(added), gpu(free), page, capacity)
    want = loop(table.tolist(), cached, added, free, page, capacity)
    assert mine.tolist() == want[0]
    for x, y in zip(got, want[1:]):
        assert x.dtype == torch.int32 and x.tolist() == y
    return got


@pytest.mark.parametrize("page", [1, 7, 16, 128])
@pytest.mark.parametrize("cached,added", [
    ([0], [1]), ([0], [0]), ([5], [300]), ([15, 16, 17, 0], [1, 1, 1, 1]),
    ([0, 0, 31, 200, 7], [0, 65, 1, 0, 500]), ([3] * 300, [i % 5 for i in range(300)]),
    ([i % 40 for i in range(1000)], [0] * 999 + [7]),
])
def test_extend(cached, added, page):
    total = sum(added)
    columns = max(-(-(c + a) // page) for c, a in zip(cached, added)) + 1
    free = [(37 * i) % 4001 for i in range(total + 5)]
    run_both(cached, added, page, columns, free, total)
    run_both(cached, added, page, columns, free, total + 333)


def test_extend_no_room():
    # rows that end, free pages that end, less capacity than tokens, negative counts
    run_both([10, 0, 5], [100, 50, 0], 16, 3, list(range(100)), 200)
    _, _, used = run_both([10, 0, 40], [100, 50, 30], 16, 10, [5, 6, 7], 300)
    assert used.item() > 3
    run_both([1, 2, 3], [50, 60, 70], 16, 20, list(range(40)), 77)
    run_both([-4, 3], [9, -1], 4, 5, list(range(9)), 12)
    run_both([1], [5], 16, 1, [], 5)
    run_both([], [], 16, 4, [3], 6)
    run_both([3], [0], 16, 2, [3], 0)


def test_extend_huge_pages_and_counts():
    # a slot past 32 bits is no slot; sums past 32 bits end nothing
    gpu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = gpu([[(1 << 31) - 1, 4]])
    slots, _, _ = mfa.extend_block_tables(table, gpu([3]), gpu([20]), gpu([9]), 16, 20)
    assert slots.tolist() == [-1] * 13 + [9 * 16 + i for i in range(7)]
    big = (1 << 31) - 1
    table = gpu([[1], [2], [3]])
    slots, starts, used = mfa.extend_block_tables(table, gpu([0, big, 0]), gpu([big, big, 3]),
                                                  gpu([7, 8, 9]), 16, 40)
    assert slots.tolist() == [7 * 16 + i for i in range(16)] + [-1] * 24
    assert starts.tolist() == [0, big, big, big] and used.tolist() == [2]
    assert table.tolist() == [[7], [2], [8]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,d,page", [(1, 64, 16), (3, 128, 32), (8, 64, 128), (2, 8, 5),
                                             (5, 72, 1)])
@pytest.mark.parametrize("tokens", [1, 2, 77, 700])
def test_append(tokens, kv_heads, d, page, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    new = lambda *shape: torch.randn(shape, device="cuda", generator=g).to(dtype)  # noqa: E731
    pages = -(-tokens // page) + 4
    k_cache, v_cache = (new(pages, kv_heads, page, d) for _ in range(2))
    fused = new(tokens, 2 * kv_heads + 1, d)  # k and v as slices of one projection
    k, v = fused[:, :kv_heads], fused[:, kv_heads:2 * kv_heads]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].int()
    slots[::5] = -1
    slots[3::7] = pages * page
    want_k, want_v = k_cache.clone(), v_cache.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, :, s % page] = k[t]
            want_v[s // page, :, s % page] = v[t]
    mfa.append_kv(k, v, k_cache, v_cache, slots)
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


def test_append_head_major_and_nothing():
    k = torch.randn((2, 40, 64), device="cuda").half().transpose(0, 1)  # [T, Hkv, D]
    cache = torch.zeros((3, 2, 16, 64), device="cuda", dtype=torch.float16)
    other = torch.zeros_like(cache)
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    mfa.append_kv(k, k, cache, other, slots)
    assert torch.equal(cache.transpose(1, 2).reshape(48, 2, 64)[:40], k)
    assert torch.equal(cache, other)
    mfa.append_kv(k[:0], k[:0], cache, other, slots[:0])
    assert torch.equal(cache, other)


def test_refusals():
    i = lambda *x: torch.zeros(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for call, match in (
            (lambda: mfa.extend_block_tables(i(2, 3).long(), i(2), i(2), i(5), 16, 4), "int32"),
            (lambda: mfa.extend_block_tables(i(6), i(2), i(2), i(5), 16, 4), "shape"),
            (lambda: mfa.extend_block_tables(i(2, 3), i(3), i(2), i(5), 16, 4), "one value"),
            (lambda: mfa.extend_block_tables(i(2, 3), i(2), i(2).cpu(), i(5), 16, 4), "CUDA"),
            (lambda: mfa.extend_block_tables(i(2, 6)[:, ::2], i(2), i(2), i(5), 16, 4),
             "contiguous"),
            (lambda: mfa.extend_block_tables(i(2, 3), i(2), i(2), i(5), 0, 4), "page_size"),
            (lambda: mfa.extend_block_tables(i(2, 3), i(2), i(2), i(5), 16, -1), "capacity")):
        with pytest.raises(RuntimeError, match=match):
            call()
    k = torch.zeros((4, 2, 64), device="cuda", dtype=torch.float16)
    cache = torch.zeros((3, 2, 16, 64), device="cuda", dtype=torch.float16)
    slots = i(4)
    for args, match in (
            ((k.float(), k, cache, cache, slots), "same dtype"),
            ((k, k[:3], cache, cache, slots), "one entry per token"),
            ((k, k, cache, cache, slots[:3]), "one entry per token"),
            ((k, k, cache, cache, slots.long()), "int32"),
            ((k[:, :1], k, cache, cache, slots), "shape"),
            ((k, k, cache.transpose(1, 2), cache.transpose(1, 2), slots), "contiguous"),
            ((k.transpose(1, 2).contiguous().transpose(1, 2), k, cache, cache, slots),
             "contiguous in D"),
            ((torch.zeros((4, 2, 68), device="cuda").half()[:, :, :64], k, cache, cache, slots),
             "multiples of 8"),
            ((k.reshape(-1)[4:4 + 256].reshape(2, 2, 64), k[:2], cache, cache, slots[:2]),
             "16-byte aligned"),
            ((k.cpu(), k, cache, cache, slots), "same device")):
        with pytest.raises(RuntimeError, match=match):
            mfa.append_kv(*args)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_generation(window, sinks):
    """Prompts go through the windowed forward and into the cache, then tokens are decoded one by
    one; every output against the attention of the whole sequence. The decoding step is a graph
    of table, copy and attention, replayed with new lengths. A request leaves on the way, and the
    rows behind the batch's tokens stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(5)
    batch, heads, kv_heads, d, page, steps = 3, 4, 2, 64, 16, 20
    prompts = [40, 1, 33]
    n = max(prompts) + steps
    q, k, v = (torch.randn((batch, h, n, d), device="cuda", generator=g).half()
               for h in (heads, kv_heads, kv_heads))
    whole = window or n
    want = reference(q, k, v, whole, sinks if window else 0)["out"]
    out = mfa.forward_window(q, k, v, whole, sinks if window else 0)
    assert ((out.double() - want[0]).abs() <= want[1]).all()

    columns = -(-n // page)
    free = torch.randperm(batch * columns, generator=g, device="cuda").int()
    shape = (batch * columns, kv_heads, page, d)
    k_cache, v_cache = (torch.full(shape, float("nan"), device="cuda").half() for _ in range(2))
    table = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")
    cached = torch.zeros(batch, dtype=torch.int32, device="cuda")
    added = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    rows = lambda x: torch.cat([x[b, :, :m].transpose(0, 1)  # noqa: E731
                                for b, m in enumerate(prompts)])
    capacity = sum(prompts) + 6
    pad = torch.full((6, kv_heads, d), 7.0, device="cuda").half()
    slots, starts, used = mfa.extend_block_tables(table, cached, added, free, page, capacity)
    mfa.append_kv(torch.cat((rows(k), pad)), torch.cat((rows(v), pad)), k_cache, v_cache, slots)
    assert starts.tolist() == [0, 40, 41, 74] and used.item() == 3 + 1 + 3
    assert torch.isnan(k_cache).sum().item() == (k_cache.numel()
                                                 - sum(prompts) * kv_heads * d)
    free = free[used.item():].contiguous()

    # one step: the new tokens' pages, slots and rows, then their attention
    cached = added.clone()
    ones = torch.ones_like(cached)
    rest = torch.zeros(batch * columns, dtype=torch.int32, device="cuda")
    rest[:len(free)] = free
    taken = torch.zeros(1, dtype=torch.int64, device="cuda")
    k_new, v_new = (torch.zeros((batch, kv_heads, d), device="cuda").half() for _ in range(2))
    q_new = torch.zeros((batch, heads, d), device="cuda").half()

    def step():
        mine, _, count = mfa.extend_block_tables(table, cached, ones, rest, page, batch)
        mfa.append_kv(k_new, v_new, k_cache, v_cache, mine)
        cached.add_(ones)
        # what was taken leaves the list
        at = (torch.arange(len(rest), device="cuda") + count).clamp(max=len(rest) - 1)
        rest.copy_(rest[at])
        taken.add_(count)
        return mfa.paged_attention(q_new, k_cache, v_cache, table, cached, window, sinks)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step()
    for s in range(steps):
        if s == 12:
            ones[1] = 0  # the second request is done; its length of 0 marks an idle row
            cached[1] = 0
        at = [m + s for m in prompts]
        live = [b for b in range(batch) if b != 1 or s < 12]
        q_new.copy_(torch.stack([q[b, :, i] for b, i in enumerate(at)]))
        for to, x in ((k_new, k), (v_new, v)):
            # the new tokens' rows follow one another, an idle request has none
            to[:len(live)] = torch.stack([x[b, :, at[b]] for b in live])
        graph.replay()
        for b, i in enumerate(at):
            if b not in live:
                assert (result[b] == 0).all()
                continue
            value, bound = want[0][b, :, i], want[1][b, :, i]
            over = ((result[b].double() - value).abs() - bound).max().item()
            assert over <= 0, (s, b, over)
    assert taken.item() == sum(-(-(m + (12 if b == 1 else steps)) // page) - -(-m // page)
                               for b, m in enumerate(prompts))
    assert capi.device_status(torch.cuda.current_device()) == 0
