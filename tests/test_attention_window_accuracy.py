"""How exact the windowed attention's gradients are: the 64-bit formula against differences, the kernels
against the formula by norms over blocks of rows (the bounds of window_reference.py add up magnitudes
and say little where many keys are visible), and what these checks do with gradients that are wrong.

By norms: the error of dq and dk is made of three roundings of about the same size, their own, that of
dS and, through the row sums, that of the forward's weights; that of dv of two, its own and that of P. So
over a block of rows it is at most 3 ** 0.5 or 2 ** 0.5 times the rounding of the exact values alone (a
step of each value's, over 12 ** 0.5).

By chance it may be more. The D values of a row share the rounding errors of its dS, one for each key, and
of its row sum. Where rows see two keys a block of 128 rows holds 256 and 128 of them, with squares of
a kurtosis of up to 10 (products of a rounding and of a value), so a third of the error's square is off
by (10 / 256) ** 0.5 and another by (10 / 128) ** 0.5 of itself: together by 0.11 of the whole, and the
norm by half of that, 0.06. dk of keys that one row sees: twice (10 / 128) ** 0.5 of a third, 0.07; dv
of those: (10 / 128) ** 0.5 of a half, 0.07. The largest of some hundreds is at four times that."""
from __future__ import annotations

import math

import pytest
import torch

import mini_flash_attention as mfa
from window_reference import check, half_step, reference, visible

CHANCE = 1.3
MOST = {"dq": 3 ** 0.5 * CHANCE, "dk": 3 ** 0.5 * CHANCE, "dv": 2 ** 0.5 * CHANCE}
NAMES = tuple(MOST)


def ratios(x, value, dtype, rows=128):
    """Norms of x - value over what rounding value is off by on average, [B, H, blocks of rows] (a last
    block of fewer than 64 rows is a part of the one before)."""
    n, info = value.shape[2], torch.finfo(dtype)
    ends = [e for e in range(rows, n + 1, rows) if n - e >= 64 or e == n]
    ends = ends if ends and ends[-1] == n else [*ends, n]
    step = torch.exp2(torch.floor(torch.log2(value.abs().clamp(min=info.tiny)))) * info.eps
    got, first = [], 0
    for end in ends:
        error = (x[:, :, first:end].double() - value[:, :, first:end]).flatten(2).norm(dim=2)
        got.append(error / (step[:, :, first:end].flatten(2).norm(dim=2) / 12 ** 0.5))
        first = end
    return torch.stack(got, 2)


def inputs(b, h, hk, n, d, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((b, x, n, d), generator=g).to(dtype).to(device) for x in (h, hk, hk, h)]


def loss_along(x, direction, window, sinks, dout):
    """The formula's loss, written apart from reference(), at `step` along the direction."""
    group, d, n = x[0].shape[1] // x[1].shape[1], x[0].shape[3], x[0].shape[2]

    def loss(step):
        q, k, v = (t.detach().double() + step * w for t, w in zip(x, direction))
        k, v = (t.repeat_interleave(group, 1) for t in (k, v))
        s = torch.einsum("bhid,bhjd->bhij", q, k) / math.sqrt(d)
        s = s.masked_fill(~visible(n, window, sinks, q.device), -math.inf)
        return (torch.softmax(s, -1) @ v * dout.double()).sum()

    return loss


def directions(x, seed, count):
    g = torch.Generator().manual_seed(seed)
    return [[torch.randn(t.shape, generator=g, dtype=torch.float64).to(t.device) for t in x]
            for _ in range(count)]


# --------------------------------------------------------------------- the formula, on the CPU
@pytest.mark.parametrize("b,h,hk,n,d,window,sinks", [
    (1, 1, 1, 1, 32, 1, 0), (1, 2, 1, 40, 32, 5, 0), (2, 6, 2, 50, 64, 50, 0), (1, 4, 4, 61, 128, 9, 7),
    (1, 3, 1, 70, 64, 1, 1),
])
def test_formula_against_differences(b, h, hk, n, d, window, sinks):
    x = inputs(b, h, hk, n, d, torch.float16, seed=n, device="cpu")
    *x, dout = x
    want = reference(*x, window, sinks, dout)
    for direction in directions(x, n + 1, 4):
        loss = loss_along(x, direction, window, sinks, dout)
        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        ours = sum((want[m][0] * w).sum() for m, w in zip(NAMES, direction))
        size = sum((want[m][0] * w).square().sum() for m, w in zip(NAMES, direction)).sqrt()
        # a difference is off by 1e-8 times a third derivative, which is of the slope's size here
        assert abs(ours - slope) <= 1e-6 * size + 1e-9, (ours.item(), slope.item())


def test_checks_reject_wrong_gradients():
    """Rounded exact gradients pass the check by norms; without one block of queries, without one of
    the group's heads, with a tenth of the row sums gone or a hundredth too large they don't."""
    dtype, window, sinks = torch.float16, 300, 2
    *x, dout = inputs(1, 4, 1, 520, 32, dtype, seed=5, device="cpu")
    want = {m: t for m, (t, _) in reference(*x, window, sinks, dout).items()}
    exact = {m: want[m] for m in NAMES}

    def passes(grads):
        return {m for m in grads if ratios(grads[m].to(dtype), exact[m], dtype).max() <= MOST[m]}

    assert passes(exact) == set(NAMES)
    assert passes({m: 1.01 * t for m, t in exact.items()}) == set()
    part = dout.clone()
    part[:, :, 256:384] = 0
    less = reference(*x, window, sinks, part)
    assert passes({m: less[m][0] for m in NAMES}) == set()
    part = dout.clone()
    part[:, 3] = 0
    less = reference(*x, window, sinks, part)
    assert passes({m: less[m][0] for m in ("dk", "dv")}) == set()
    q, k, v = (t.double() for t in x)
    k, v = (t.repeat_interleave(4, 1) for t in (k, v))
    s = (q @ k.transpose(-1, -2) / 32 ** 0.5).masked_fill(~visible(520, window, sinks, "cpu"), -math.inf)
    p = torch.softmax(s, -1)
    ds = p * (dout.double() @ v.transpose(-1, -2) - 0.9 * (dout.double() * want["out"]).sum(-1, True))
    wrong = {"dq": ds @ k / 32 ** 0.5,
             "dk": (ds.transpose(-1, -2) @ q / 32 ** 0.5).sum(1, keepdim=True)}
    assert passes(wrong) == set()


# ------------------------------------------------------------------------ the kernels, on the GPU
# long windows, groups, units in pieces, sinks that the whole sequence sees, both sides of 1024
CASES = [(1, 1, 1, 4096, 4096, 0), (1, 8, 1, 2048, 2048, 0), (1, 4, 1, 3000, 128, 200),
         (1, 16, 2, 2500, 300, 4), (2, 2, 2, 4000, 1, 1), (1, 4, 2, 1024, 1024, 0),
         (1, 4, 2, 1025, 1025, 0), (2, 6, 2, 777, 128, 4), (2, 32, 8, 1100, 256, 4),
         # rows of few keys that lie in several blocks: a sink and the row's own, windows over a
         # block's end
         (1, 4, 2, 1500, 2, 1), (1, 4, 1, 1500, 5, 2), (2, 2, 1, 1500, 40, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("b,h,hk,n,window,sinks", CASES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradients_by_norm(b, h, hk, n, window, sinks, d, dtype):
    *x, dout = inputs(b, h, hk, n, d, dtype, seed=n + d, device="cuda")
    leaves = [t.requires_grad_() for t in x]
    grads = torch.autograd.grad(mfa.window_attention(*leaves, window, sinks), leaves, dout)
    for i in range(b):
        part = [t[i:i + 1].detach() for t in x]
        want = reference(*part, window, sinks, dout[i:i + 1])
        for name, grad in zip(NAMES, grads):
            worst = ratios(grad[i:i + 1], want[name][0], dtype).max().item()
            assert worst <= MOST[name], (name, worst)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradients_against_differences(d, dtype):
    """Projections of the gradients on random directions against differences of the formula. A
    projection is a sum of independent rounding errors, each about one half step of a gradient's value
    (three roundings of half_step / 3 ** 0.5 rms), so six times the root of their squares bound it; no
    gradient at all is off by hundreds of that."""
    window, sinks = 50, 2
    *x, dout = inputs(1, 4, 2, 300, d, dtype, seed=d, device="cuda")
    leaves = [t.requires_grad_() for t in x]
    grads = torch.autograd.grad(mfa.window_attention(*leaves, window, sinks), leaves, dout)
    slopes, rooms = [], []
    for direction in directions(x, 2 * d, 8):
        loss = loss_along(x, direction, window, sinks, dout)
        slopes.append(((loss(1e-4) - loss(-1e-4)) / 2e-4).item())
        ours = sum((g.double() * w).sum() for g, w in zip(grads, direction)).item()
        size = sum((g.double() * w).square().sum() for g, w in zip(grads, direction)).sqrt().item()
        rooms.append(6 * half_step(dtype) * size)
        assert abs(ours - slopes[-1]) <= rooms[-1], (ours, slopes[-1], rooms[-1])
    far = 100 if dtype == torch.float16 else 12  # 0.3 of a projection's size
    assert max(abs(s) / r for s, r in zip(slopes, rooms)) > far


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
def test_gradients_of_large_scores(rest):
    # scores of hundreds: weights of 0 and 1, hardly any between
    *x, dout = inputs(1, 2, 1, 700, 64, torch.float16, seed=7, device="cuda")
    q, k, v = x[0] * 8, x[1] * 8, x[2]
    want = reference(q, k, v, 150, 3, dout)
    out, lse, *more = mfa.forward_window_lse(q, k, v, 150, 3, rest=rest)
    grads = mfa.backward_window(q, k, v, out, lse, dout, 150, 3, *more)
    # a score of up to about 500 is off by up to 64 products' 2^-24 relative in 32 bits, and its
    # logarithm base 2 by one more step: at most 4 * 2e-4 in the exponent, which is DELTA five times
    for name, x in zip(NAMES, grads):
        value, bound = want[name]
        check(name, x, value, 5 * bound)
