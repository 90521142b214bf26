"""How exact the windowed attention's gradients are: the kernels against the formula by norms over blocks
of rows (the bounds of window_reference.py add up magnitudes and say little where many keys are
visible).

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

import pytest
import torch

import mini_flash_attention as mfa
from window_reference import reference

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


# ------------------------------------------------------------------------ the kernels, on the GPU
# rows of few keys that lie in several blocks: a sink and the row's own, windows over a block's end
CASES = [(2, 2, 2, 4000, 1, 1), (1, 4, 2, 1500, 2, 1), (1, 4, 1, 1500, 5, 2), (2, 2, 1, 1500, 40, 3)]


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
