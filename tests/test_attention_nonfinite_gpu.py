"""GPU tests of what NaN and infinities in visible places do: by the formula a row that sees a score
of NaN or +inf is NaN, a key whose score is -inf has no weight, and every other row is as without
them. In every form of the paged and shared-prefix attention (which depends on the table's width and the
prefix's bytes)."""
from __future__ import annotations

import math

import pytest
import torch

import mini_flash_attention as mfa
from paged_reference import Cache, check, queries

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
DIMS = pytest.mark.parametrize("d", [32, 64, 128])
# "few" units go to a cluster of CTAs each, with a wide table or many requests to equal shares; a
# prefix of few bytes becomes the requests' first tiles, one that the batch would read more
# than 64 MB of has its own kernel
FORMS = ["few", "wide", "inside", "inside_wide", "apart"]
NAN = float("nan")


def make(form, d, dtype):
    lengths = [300, 1, 77, 1000, 0]
    prefix = {"inside": 200, "inside_wide": 200, "apart": 1100}.get(form, 0)
    if form == "apart":
        lengths = lengths + [(7 * i) % 60 for i in range(17_000_000 // (2 * d * prefix) + 1)]
    columns = 700 if "wide" in form else None
    return Cache(lengths, 2, d, 32, dtype, prefix=prefix, columns=columns, seed=d)


def call(cache, q):
    k, v, table, lengths = cache.tensors()
    if cache.prefix:
        return mfa.shared_prefix_attention(q.cuda(), k, v, cache.pages(), cache.prefix, table,
                                           lengths)
    return mfa.paged_attention(q.cuda(), k, v, table, lengths)


def row_of(cache, request, position):
    """The cache's page and row of a request's own token (request None: the prefix's)."""
    pages = cache.prefix_pages if request is None else cache.table[request].tolist()
    return pages[position // 32], position % 32


def expect(cache, q, out, bad):
    """Rows in `bad` [B, H] are NaN in every column, the others within the formula's bounds."""
    value, bound = cache.reference(q)
    bad = bad.cuda()
    assert torch.isnan(out[bad]).all()
    check(out[~bad], value[~bad], bound[~bad])


@DTYPES
@DIMS
@pytest.mark.parametrize("form", FORMS)
def test_nan_query(form, d, dtype):
    cache = make(form, d, dtype)
    batch = len(cache.lengths)
    q = queries(batch, 6, d, dtype)
    clean = q.clone()
    q[0, 1, d - 1] = NAN   # one value of a row
    q[3, 4] = NAN          # a whole row
    q[1, 0, 0] = NAN       # a request of one token
    q[4, 5] = NAN          # sees nothing, or the prefix alone
    bad = torch.zeros((batch, 6), dtype=torch.bool)
    bad[0, 1] = bad[3, 4] = bad[1, 0] = True
    bad[4, 5] = cache.prefix > 0
    expect(cache, clean, call(cache, q), bad)


@DTYPES
@DIMS
@pytest.mark.parametrize("value", [NAN, float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("form", FORMS)
def test_key(form, value, d, dtype):
    cache = make(form, d, dtype)
    batch = len(cache.lengths)
    q = queries(batch, 6, d, dtype)
    # +inf makes the score of heads 0, 1, 2 +inf where their first column is positive, and -inf
    # where it is negative
    q[:, 0, 0], q[:, 1, 0], q[:, 2, 0] = 1.0, 0.5, -1.0
    for position in (0, 9, 17, 22, 47, 62, 85, 120, 250, 299):
        page, row = row_of(cache, 0, position)
        keep = cache.k[page, 0, row].clone()
        cache.k[page, 0, row, 0] = value
        bad = torch.zeros((batch, 6), dtype=torch.bool)
        bad[0, :2] = True
        bad[0, 2] = math.isnan(value)
        out = call(cache, q)
        if not math.isnan(value):  # the key of score -inf leaves head 2's sums
            own = cache.keys[0], cache.values[0]
            left = [j for j in range(300) if j != position]
            cache.keys[0], cache.values[0] = (x[left] for x in own)
            want = [x[0, 2] for x in cache.reference(q)]
            check(out[0, 2], *want)
            cache.keys[0], cache.values[0] = own
            bad[0, 2] = True
            out[0, 2] = NAN
        expect(cache, q, out, bad)
        cache.k[page, 0, row] = keep


@DTYPES
@DIMS
@pytest.mark.parametrize("form", ["inside", "inside_wide"])
def test_prefix_key(form, d, dtype):
    cache = make(form, d, dtype)
    batch = len(cache.lengths)
    q = queries(batch, 6, d, dtype)
    bad = torch.zeros((batch, 6), dtype=torch.bool)
    bad[:, 3:] = True
    for position in (0, 18, 54, 103, 150, 199):
        page, row = row_of(cache, None, position)
        keep = cache.k[page, 1, row].clone()
        cache.k[page, 1, row, d // 2] = NAN
        expect(cache, q, call(cache, q), bad)
        cache.k[page, 1, row] = keep


@DIMS
@pytest.mark.parametrize("form", FORMS)
def test_value(form, d):
    # v of a visible key: its column is NaN for the heads that read it
    cache = make(form, d, torch.bfloat16)
    batch = len(cache.lengths)
    q = queries(batch, 6, d, torch.bfloat16)
    value, bound = cache.reference(q)
    for position in (0, 33, 299):
        page, row = row_of(cache, 0, position)
        keep = cache.v[page, 1, row].clone()
        cache.v[page, 1, row, 5] = NAN
        out = call(cache, q)
        assert torch.isnan(out[0, 3:, 5]).all()
        out[0, 3:, 5] = value[0, 3:, 5].to(out.dtype)
        check(out, value, bound)
        cache.v[page, 1, row] = keep
