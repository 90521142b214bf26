"""GPU tests of what NaN and infinities in visible places do: by the formula a row that sees a score
of NaN or +inf is NaN, a key whose score is -inf has no weight, and every other row is as without
them. In every form of the windowed, paged and shared-prefix attention (the form of the paged
ones depends on the table's width and the prefix's bytes), at keys of many columns of a tile."""
from __future__ import annotations

import math

import pytest
import torch

import mini_flash_attention as mfa
from paged_reference import Cache, check as check_paged, queries
from window_reference import check, reference, visible

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
    check_paged(out[~bad], value[~bad], bound[~bad])


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
            check_paged(out[0, 2], *want)
            cache.keys[0], cache.values[0] = own
            bad[0, 2] = True
            out[0, 2] = NAN
        expect(cache, q, out, bad)
        cache.k[page, 0, row] = keep


@DTYPES
@DIMS
@pytest.mark.parametrize("form", ["inside", "inside_wide", "apart"])
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
        check_paged(out, value, bound)
        cache.v[page, 1, row] = keep


# ------------------------------------------------------------------------------ whole sequences
def sequence(d, dtype, n=700, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((1, h, n, d), generator=g).to(dtype).cuda() for h in (4, 2, 2, 4)]


def expect_rows(got, want, bad):
    """got, want: {name: tensor}, {name: (value, bound)}; bad [B, H, N]."""
    for name, x in got.items():
        value, bound = want[name]
        assert torch.isnan(x[bad]).all(), name
        check(name, x[~bad], value[~bad], bound[~bad])


@DTYPES
@DIMS
@pytest.mark.parametrize("window,sinks", [(700, 0), (130, 3), (64, 40)])
def test_window_query(window, sinks, d, dtype):
    q, k, v, _ = sequence(d, dtype)
    want = reference(q, k, v, window, sinks)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    for h, i in ((0, 0), (1, 130), (2, 257), (3, 699)):
        q[0, h, i, i % d] = NAN
        bad[0, h, i] = True
    out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
    expect_rows({"out": out, "lse": lse}, want, bad)
    expect_rows({"out": mfa.forward_window(q, k, v, window, sinks)}, want, bad)


@DTYPES
@DIMS
@pytest.mark.parametrize("value", [NAN, float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("window,sinks", [(700, 0), (130, 3), (64, 40)])
def test_window_key(window, sinks, value, d, dtype):
    q, k, v, _ = sequence(d, dtype)
    q[..., 0] = q[..., 0].abs() + 0.1  # q.k is +inf where k's first column is
    want = reference(q, k, v, window, sinks)
    seen = visible(700, window, sinks, "cuda")
    for position in (0, 18, 39, 86, 117, 143, 215, 400, 693, 699):
        keep = k[0, 1, position].clone()
        k[0, 1, position, 0] = value
        bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
        bad[0, 2:] = seen[:, position]
        out, lse = mfa.forward_window_lse(q, k, v, window, sinks)
        expect_rows({"out": out, "lse": lse}, want, bad)
        k[0, 1, position] = keep


@DTYPES
@DIMS
def test_window_gradients(d, dtype):
    """A query row whose score is NaN or infinite has a NaN gradient, and so have the keys that it
    sees; other heads are as without it."""
    for at, value in ((150, NAN), (300, float("inf"))):
        q, k, v, dout = sequence(d, dtype)
        want = reference(q, k, v, 200, 2, dout)
        k[0, 0, at, 1] = value
        out, lse = mfa.forward_window_lse(q, k, v, 200, 2)
        dq, dk, dv = mfa.backward_window(q, k, v, out, lse, dout, 200, 2)
        rows = torch.arange(at, at + 200, device="cuda")
        if math.isinf(value):
            rows = [r for r in rows.tolist() if (q[0, :2, r, 1] > 0).all()]
        assert torch.isnan(dq[0, :2, rows]).all()
        assert torch.isnan(dk[0, 0, at]).all() and torch.isnan(dv[0, 0, at]).all()
        for name, x, first in (("dq", dq, 2), ("dk", dk, 1), ("dv", dv, 1)):
            check(name, x[:, first:], *(t[:, first:] for t in want[name]))


# ------------------------------------------------------------------------------ without a window
@DIMS
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("h,n", [(2, 700), (1, 8200)], ids=["whole", "in_pieces"])
def test_forward(h, n, causal, d):
    """The kernel that the window and prefix variants share their steps with; few long heads are cut
    into pieces."""
    g = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn((1, h, n, d), generator=g).half().cuda() for _ in range(3))
    clean = mfa.forward(q, k, v, causal).double()
    k[0, 0, 54, 1] = NAN
    out = mfa.forward(q, k, v, causal)
    first = 54 if causal else 0
    assert torch.isnan(out[0, 0, first:]).all()
    # the others: the same formula, the reference maximum possibly raised at other steps; each weight
    # is rounded twice (2 * 2^-11) and the outputs are, of values up to |v| < 6
    rest = torch.cat((out[0, 0, :first], out[0, 1:].reshape(-1, d))).double()
    want = torch.cat((clean[0, 0, :first], clean[0, 1:].reshape(-1, d)))
    assert ((rest - want).abs() <= 4 * 2.0 ** -11 * 6).all()
