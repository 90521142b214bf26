"""GPU tests of the attention of single tokens over a paged cache, alone (with and without a window
and sinks) and behind a shared prefix, against the formula in 64 bits. In every cache what is
not visible is NaN, and table entries of pages without visible tokens are out of range."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi
from paged_reference import Cache, check, queries

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def status_stays_clean():
    yield
    assert capi.device_status(torch.cuda.current_device()) == 0


def decode(cache, q, window=0, sinks=0):
    k, v, table, lengths = cache.tensors()
    return mfa.paged_attention(q.cuda(), k, v, table, lengths, window, sinks)


LENGTHS = {
    "one": [1], "empty": [0, 0], "tile_edges": [63, 64, 65, 0, 127, 128, 129, 1],
    "long": [5000], "ragged": [3, 900, 0, 77, 2049, 16],
}


# A table for long requests goes to the kernels that cut the work into equal shares, a narrow one
# and few requests to the one that gives a cluster of CTAs to a head of a request.
WIDE = pytest.mark.parametrize("wide", [False, True], ids=["narrow", "wide"])


def columns(lengths, page, wide):
    return max(1, *(-(-n // page) for n in lengths), 9000 // page if wide else 1)


@WIDE
@pytest.mark.parametrize("lengths", LENGTHS.values(), ids=LENGTHS.keys())
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_decode(lengths, page, d, dtype, wide):
    cache = Cache(lengths, 2, d, page, dtype, columns=columns(lengths, page, wide), seed=page + d)
    q = queries(len(lengths), 6, d, dtype)
    check(decode(cache, q), *cache.reference(q))


# windows of one token, inside a page, over pages, of whole tiles, past the sequence; sinks none,
# few, past a tile, meeting the window
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (64, 4), (100, 65), (128, 64), (500, 130),
                                          (900, 1000), (10000, 3), (63, 17)])
@pytest.mark.parametrize("page,d,dtype", [(16, 64, torch.float16), (64, 128, torch.bfloat16),
                                          (256, 64, torch.bfloat16), (16, 128, torch.float16),
                                          (16, 32, torch.bfloat16), (128, 32, torch.float16)])
@WIDE
def test_decode_window(window, sinks, page, d, dtype, wide):
    lengths = [1, 64, 100, 129, 0, 1000, 1537]
    cache = Cache(lengths, 2, d, page, dtype, window=window, sinks=sinks, seed=window,
                  columns=columns(lengths, page, wide))
    q = queries(len(lengths), 8, d, dtype)
    check(decode(cache, q, window, sinks), *cache.reference(q))


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (8, 1), (3, 2), (1, 7), (2, 16), (1, 17), (2, 33),
                                            (1, 128)])
@pytest.mark.parametrize("d", [32, 64, 128])
@WIDE
def test_decode_heads(kv_heads, group, d, wide):
    lengths = [200, 1, 333]
    cache = Cache(lengths, kv_heads, d, 32, torch.bfloat16, seed=group,
                  columns=columns(lengths, 32, wide))
    q = queries(3, kv_heads * group, d, torch.bfloat16)
    check(decode(cache, q), *cache.reference(q))


def test_decode_many_requests():
    # more requests than threads that sum their lengths, most of them short or empty
    lengths = [(7 * i) % 40 if i % 97 else 700 for i in range(500)]
    cache = Cache(lengths, 1, 64, 16, torch.float16, columns=60)
    q = queries(500, 2, 64, torch.float16)
    check(decode(cache, q), *cache.reference(q))


def test_decode_a_unit_a_cta():
    # about as many units as CTAs, of about the same length, and a table for longer ones
    lengths = [900 + 7 * i for i in range(30)]
    cache = Cache(lengths, 8, 128, 32, torch.bfloat16, columns=100)
    q = queries(30, 32, 128, torch.bfloat16)
    check(decode(cache, q), *cache.reference(q))
    cache = Cache(lengths, 8, 128, 32, torch.bfloat16, columns=100, prefix=1500)
    q = queries(30, 32, 128, torch.bfloat16)
    check(behind_prefix(cache, q), *cache.reference(q))


def test_decode_very_many_requests():
    lengths = [(13 * i) % 90 for i in range(5000)]
    cache = Cache(lengths, 1, 128, 16, torch.bfloat16)
    q = queries(5000, 1, 128, torch.bfloat16)
    check(decode(cache, q), *cache.reference(q))


def test_decode_more_units_than_ctas():
    lengths = [100 + i for i in range(90)]
    cache = Cache(lengths, 4, 64, 32, torch.float16)
    q = queries(90, 8, 64, torch.float16)
    check(decode(cache, q), *cache.reference(q))


def test_decode_clamps_lengths():
    cache = Cache([128, 0], 1, 64, 32, torch.float16)
    q = queries(2, 1, 64, torch.float16)
    k, v, table, _ = cache.tensors()
    lengths = torch.tensor([1 << 30, -7], dtype=torch.int32, device="cuda")
    check(mfa.paged_attention(q.cuda(), k, v, table, lengths), *cache.reference(q))


def test_decode_large_scores_and_infinite_keys_out_of_sight():
    cache = Cache([300, 40], 1, 64, 16, torch.float16, window=50, sinks=2)
    cache.k[torch.isnan(cache.k)] = float("inf")
    cache.v[torch.isnan(cache.v)] = -float("inf")
    q = queries(2, 4, 64, torch.float16) * 16
    value, bound = cache.reference(q)
    # scores of up to about 100: 64 products' 2^-24 relative in 32 bits, in the exponent
    check(decode(cache, q, 50, 2), value, 2 * bound)


# --------------------------------------------------------------------------- shared prefix
def behind_prefix(cache, q):
    k, v, table, own = cache.tensors()
    return mfa.shared_prefix_attention(q.cuda(), k, v, cache.pages(), cache.prefix, table, own)


# few bytes of prefix, which become each request's first tiles
@WIDE
@pytest.mark.parametrize("prefix", [1, 16, 63, 64, 65, 1000])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_prefix(prefix, page, d, dtype, wide):
    lengths = [0, 1, 65, 200, 17]
    cache = Cache(lengths, 2, d, page, dtype, prefix=prefix, seed=prefix,
                  columns=columns(lengths, page, wide))
    q = queries(5, 6, d, dtype)
    check(behind_prefix(cache, q), *cache.reference(q))


# more than 64 MB read by all requests together: the prefix has a kernel of its own
@pytest.mark.parametrize("prefix,batch", [(127, 530), (128, 530), (129, 530), (1000, 140)])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
def test_prefix_apart(prefix, batch, page, d, dtype):
    batch = batch * 128 // d
    lengths = [(7 * i) % 70 for i in range(batch)]
    cache = Cache(lengths, 2, d, page, dtype, prefix=prefix, seed=prefix)
    q = queries(batch, 6, d, dtype)
    check(behind_prefix(cache, q), *cache.reference(q))


# one tile of query rows, a tile and one row, several tiles, groups that do not divide a tile
@pytest.mark.parametrize("batch,kv_heads,group", [(1, 1, 1), (16, 2, 8), (17, 1, 8), (50, 2, 7),
                                                  (100, 1, 5), (3, 1, 128), (300, 2, 1),
                                                  (20, 1, 33)])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("long", [False, True])
def test_prefix_rows(batch, kv_heads, group, d, long):
    lengths = [(11 * i) % 30 for i in range(batch)]
    prefix = 17_000_000 // (batch * kv_heads * d) + 100 if long else 70
    cache = Cache(lengths, kv_heads, d, 32, torch.bfloat16, prefix=prefix, seed=batch)
    q = queries(batch, kv_heads * group, d, torch.bfloat16)
    check(behind_prefix(cache, q), *cache.reference(q))


@pytest.mark.parametrize("d", [32, 64, 128])
def test_prefix_several_units_a_cta(d):
    # more query tiles than CTAs: a CTA goes over several units
    lengths = [(5 * i) % 50 for i in range(320)]
    cache = Cache(lengths, 4, d, 64, torch.bfloat16, prefix=1100)
    q = queries(320, 4 * 31, d, torch.bfloat16)
    check(behind_prefix(cache, q), *cache.reference(q))


@pytest.mark.parametrize("batch,d,page", [(40, 128, 128), (150, 128, 16), (150, 64, 256),
                                           (50, 32, 64)])
def test_prefix_past_the_l2(batch, d, page):
    # a prefix of more bytes than stay in L2: the units of a head read the same keys at the same time
    prefix = 32768 * 128 // d - 5
    cache = Cache([i % 3 for i in range(batch)], 8, d, page, torch.float16, prefix=prefix)
    q = queries(batch, 64, d, torch.float16)
    check(behind_prefix(cache, q), *cache.reference(q))


def test_prefix_long_and_none():
    lengths = [5, 300]
    cache = Cache(lengths, 8, 64, 64, torch.float16, prefix=20000)
    q = queries(2, 8, 64, torch.float16)
    check(behind_prefix(cache, q), *cache.reference(q))
    cache = Cache(lengths, 8, 64, 64, torch.float16)
    k, v, table, own = cache.tensors()
    out = mfa.shared_prefix_attention(q.cuda(), k, v, cache.pages(), 0, table, own)
    check(out, *cache.reference(q))
    assert torch.equal(out, mfa.paged_attention(q.cuda(), k, v, table, own))


def test_prefix_without_own_tokens():
    cache = Cache([0, 0, 0], 2, 64, 16, torch.bfloat16, prefix=333, columns=0)
    q = queries(3, 4, 64, torch.bfloat16)
    check(behind_prefix(cache, q), *cache.reference(q))
    cache = Cache([0] * 500, 2, 64, 16, torch.bfloat16, prefix=333, columns=0)
    q = queries(500, 4, 64, torch.bfloat16)
    check(behind_prefix(cache, q), *cache.reference(q))


# ----------------------------------------------------------------------------- any caller
def test_same_result_again_on_streams_and_in_graphs():
    lengths = [700, 3, 2500, 64]
    cache = Cache(lengths, 2, 64, 16, torch.float16, prefix=500)
    q = queries(4, 8, 64, torch.float16).cuda()
    k, v, table, own = cache.tensors()
    pages = cache.pages()

    wide = torch.cat((table, torch.full((4, 600), -1, dtype=torch.int32, device="cuda")), 1)
    many = Cache([5] * 300, 2, 64, 16, torch.float16, prefix=500)
    big, big_q = many.tensors(), queries(300, 8, 64, torch.float16).cuda()
    big_pages = many.pages()

    def calls():
        return (mfa.paged_attention(q, k, v, table, own),
                mfa.paged_attention(q, k, v, wide, own),
                mfa.paged_attention(q, k, v, wide, own, 1, 0),
                mfa.shared_prefix_attention(q, k, v, pages, 500, table, own),
                mfa.shared_prefix_attention(big_q, *big[:2], big_pages, 500, *big[2:]))  # 77 MB

    want = calls()
    assert all(torch.equal(a, b) for a, b in zip(want, calls()))
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([calls() for _ in range(3)])
    torch.cuda.synchronize()
    for per_stream in got:
        for result in per_stream:
            assert all(torch.equal(a, b) for a, b in zip(want, result))
    # two graphs, replayed in turn with other lengths
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = calls()
        graphs.append((graph, result))
    for n in ([700, 3, 2500, 64], [1, 0, 1300, 30]):
        own.copy_(torch.tensor(n, dtype=torch.int32))
        want = calls()
        for graph, _ in graphs:
            graph.replay()
        for _, result in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, result))


def test_cache_past_32_bits():
    # 2^31 elements and more lie before the last pages
    page, kv_heads, d = 256, 8, 128
    pages = (1 << 31) // (kv_heads * page * d) + 3
    k = torch.zeros((pages, kv_heads, page, d), device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    n = 300
    small = Cache([n], kv_heads, d, page, torch.bfloat16)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    for at, column in ((pages - 1, 0), (pages - 2, 1)):
        k[at], v[at] = small.k[small.table[0, column]], small.v[small.table[0, column]]
    q = queries(1, kv_heads, d, torch.bfloat16)
    own = torch.tensor([n], dtype=torch.int32, device="cuda")
    check(mfa.paged_attention(q.cuda(), k, v, table, own), *small.reference(q))
    empty = torch.zeros((1,), dtype=torch.int32, device="cuda")
    out = mfa.shared_prefix_attention(q.cuda(), k, v, table[0].contiguous(), n, table, empty)
    check(out, *small.reference(q))
    new = torch.randn((2, kv_heads, d), device="cuda").bfloat16()
    slots = torch.tensor([pages * page - 1, 5], dtype=torch.int32, device="cuda")
    mfa.append_kv(new, new, k, v, slots)
    for t, (at, row) in enumerate(((pages - 1, page - 1), (0, 5))):
        assert torch.equal(k[at, :, row], new[t]) and torch.equal(v[at, :, row], new[t])


def test_bad_pages_are_reported():
    device = torch.cuda.current_device()
    cache = Cache([100, 20], 2, 64, 16, torch.float16, prefix=40)
    q = queries(2, 4, 64, torch.float16)
    k, v, table, own = cache.tensors()
    cache.shared = [x[:0] for x in cache.shared]  # its reference without the prefix
    for bad in (-1, k.shape[0], 1 << 30):
        broken = table.clone()
        broken[0, 2] = bad  # tokens 32 to 47 read as zeros
        out = mfa.paged_attention(q.cuda(), k, v, broken, own)
        assert capi.device_status(device) == capi.STATUS_BAD_PAGE
        assert capi.device_status(device) == 0
        value, bound = cache.reference(q)
        check(out[1:], value[1:], bound[1:])  # the other request is not touched by it
        pages = cache.pages()
        pages[1] = bad
        mfa.shared_prefix_attention(q.cuda(), k, v, pages, 40, table, own)
        assert capi.device_status(device) == capi.STATUS_BAD_PAGE


# q as a part of a fused projection, or with the heads outermost: bit for bit what a contiguous q
# gives, in every form of the kernel (few units, equal shares, a prefix inside and apart)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("batch,group,prefix", [(3, 3, 0), (150, 4, 0), (9, 17, 0), (5, 2, 100),
                                                (40, 5, 3000), (130, 1, 6000), (1, 2, 70), (4, 1, 0)])
@WIDE
def test_query_strides(batch, group, prefix, d, wide):
    lengths = [(37 * i) % 200 for i in range(batch)]
    cache = Cache(lengths, 2, d, 32, torch.bfloat16, prefix=prefix, seed=batch + prefix,
                  columns=columns(lengths, 32, wide))
    k, v, table, own = cache.tensors()
    heads = 2 * group
    q = queries(batch, heads, d, torch.bfloat16).cuda()
    fused = torch.full((batch, (heads + 4) * d), float("nan"), device="cuda", dtype=q.dtype)
    part = fused[:, 2 * d:(2 + heads) * d].view(batch, heads, d)
    part.copy_(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    if prefix:
        call = lambda x: mfa.shared_prefix_attention(  # noqa: E731
            x, k, v, cache.pages(), prefix, table, own)
    else:
        call = lambda x: mfa.paged_attention(x, k, v, table, own, 60, 5)  # noqa: E731
    want = call(q)
    for x in (part, turned):
        got = call(x)
        assert got.is_contiguous() and torch.equal(got, want)


def test_empty_batch():
    cache = Cache([5], 2, 64, 16, torch.float16)
    k, v, table, own = cache.tensors()
    q = queries(1, 4, 64, torch.float16).cuda()
    assert mfa.paged_attention(q[:0], k, v, table[:0], own[:0]).shape == (0, 4, 64)
    assert mfa.shared_prefix_attention(q[:0], k, v, table[0], 3, table[:0],
                                       own[:0]).shape == (0, 4, 64)


def test_refusals():
    cache = Cache([40, 5], 2, 64, 16, torch.float16, prefix=20)
    k, v, table, own = cache.tensors()
    pages, q = cache.pages(), queries(2, 4, 64, torch.float16).cuda()
    for change, match in (
            ({"q": q.bfloat16()}, "same dtype"), ({"q": q.float()}, "same dtype"),
            ({"q": q[:, :3].contiguous()}, "multiple of the k / v heads"),
            ({"q": q[:, :, :32].contiguous()}, "q must have shape"),
            ({"q": q.repeat_interleave(2, 2)[:, :, ::2]}, "q must be contiguous in D"),
            ({"q": q[:1].expand(2, 4, 64)}, "strides of q must be positive multiples of 8"),
            ({"q": torch.zeros(2, 4, 68, device="cuda").half()[:, :, :64]},
             "strides of q must be positive multiples of 8"),
            ({"q": torch.zeros(2, 4, 72, device="cuda").half()[:, :, 4:68]},
             "q must be 16-byte aligned"),
            ({"q": q.cpu()}, "CUDA tensor"),
            ({"k": k[:, :, ::2]}, "same shape"), ({"v": v[:-1]}, "same shape"),
            ({"k": k[:, :, :8].contiguous(), "v": v[:, :, :8].contiguous()}, "page size"),
            ({"k": k.transpose(1, 2), "v": v.transpose(1, 2)}, "contiguous"),
            ({"table": table.long()}, "block_table must be int32"),
            ({"table": table[:1]}, "block_table must have shape"),
            ({"own": own.long()}, "lengths must be int32"),
            ({"own": own[:1]}, "lengths must have one value"),
            ({"own": own.cpu()}, "lengths must be a CUDA tensor"),
            ({"window": -1}, "window must not be negative"),
            ({"sinks": -1}, "sinks must not be negative")):
        a = {"q": q, "k": k, "v": v, "table": table, "own": own, "window": 0, "sinks": 0} | change
        with pytest.raises(RuntimeError, match=match):
            mfa.paged_attention(a["q"], a["k"], a["v"], a["table"], a["own"], a["window"],
                                a["sinks"])
        if "window" in change or "sinks" in change:
            continue
        with pytest.raises(RuntimeError, match=match):
            mfa.shared_prefix_attention(a["q"], a["k"], a["v"], pages, 5, a["table"], a["own"])
    for call, match in (
            (lambda: mfa.shared_prefix_attention(q, k, v, pages, 33, table, own), "must hold"),
            (lambda: mfa.shared_prefix_attention(q, k, v, pages, -1, table, own), "negative"),
            (lambda: mfa.shared_prefix_attention(q, k, v, pages.long(), 5, table, own), "int32")):
        with pytest.raises(RuntimeError, match=match):
            call()
    x = torch.zeros((1, 1, 16, 48), device="cuda", dtype=torch.float16)
    with pytest.raises(RuntimeError, match="D=32, D=64 and D=128"):
        mfa.paged_attention(x[0, :, :1], x, x, table[:1], own[:1])
    # the workspace of the C entry is checked
    cache = Cache([40, 5], 2, 64, 16, torch.float16, columns=3000)
    k, v, table, own = cache.tensors()
    need = capi.paged_workspace_bytes(2, 4, 2, 64, 16, table.shape[1])
    work = torch.empty((need,), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    common = (2, 4, 2, 64, k.shape[0], 16, table.shape[1], 0.125)
    ptrs = [x.data_ptr() for x in (q, k, v, table, own, out, work)]
    with pytest.raises(capi.MfaError, match="the workspace must have"):
        capi.paged_attention(*ptrs, need - 1, *common)
    capi.paged_attention(*ptrs, need, *common, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check(out, *cache.reference(q.cpu()))
    # a call that takes none needs none
    assert capi.paged_workspace_bytes(2, 4, 2, 64, 16, 3) == 0
    ptrs[-1] = 0
    narrow = table[:, :3].contiguous()
    ptrs[3] = narrow.data_ptr()
    capi.paged_attention(*ptrs, 0, 2, 4, 2, 64, k.shape[0], 16, 3, 0.125,
                         stream=torch.cuda.current_stream().cuda_stream)
    check(out, *cache.reference(q.cpu()))
