"""The windowed attention and its gradients in 64 bits, with bounds for what the kernels may be off.

Let u be half a step of the type (2^-11 for fp16, 2^-8 for bf16). The kernels hold scores, row
maxima, sums and accumulators in 32 bits and round to the type

* the weights p (before the division by their sum, at most 2^8 and at least one of them 1) for
  the product with v, by u relative or, in fp16 below its normal range, by 2^-25;
* dS = p (dP - D) likewise for dq and dk, and p for dv;
* every output once, by u relative.

Exponentials are off by at most 7.5e-5 relative (the polynomial; the unit's are far below), and
the sums of 32-bit terms and the saved log-sum-exp by less than that again, so a weight is
off by delta = 2e-4 relative besides its rounding. With the sums of magnitudes in place of the
sums this gives the bounds below, none of which is a measured number.
"""
from __future__ import annotations

import math

import torch

DELTA = 2e-4
TINY = 1e-6  # 32-bit noise of values that cancel to nothing


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def visible(n: int, window: int, sinks: int, device) -> torch.Tensor:
    i = torch.arange(n, device=device)[:, None]
    j = torch.arange(n, device=device)[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks))


def reference(q, k, v, window, sinks, dout=None):
    """{name: (value, bound)} for out, lse and, with dout, dq, dk, dv, on [B, H, N, D] tensors."""
    u = half_step(q.dtype)
    floor = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    group, scale = q.shape[1] // k.shape[1], q.shape[-1] ** -0.5
    x, y, z = q.double(), *(t.double().repeat_interleave(group, 1) for t in (k, v))
    seen = visible(q.shape[2], window, sinks, q.device)
    s = (x @ y.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = p @ z
    seen = seen.double()
    out_bound = u * out.abs() + (u + DELTA) * (p @ z.abs()) + floor * (seen @ z.abs()) + TINY
    got = {"out": (out, out_bound), "lse": (lse, torch.full_like(lse, DELTA))}
    if dout is None:
        return got
    do = dout.double()
    dp = do @ z.transpose(-1, -2)
    row = (do * out).sum(-1, keepdim=True)
    row_bound = (do.abs() * out_bound).sum(-1, keepdim=True)
    ds = p * (dp - row)
    ds_bound = (u + DELTA) * ds.abs() + p * (row_bound + TINY) + floor * seen
    p_bound = (u + DELTA) * p + floor * seen
    shared = lambda t: t.reshape(k.shape[0], k.shape[1], group, *t.shape[2:]).sum(2)  # noqa: E731
    t = lambda a: a.transpose(-1, -2)  # noqa: E731
    for name, value, bound in (
            ("dq", ds @ y * scale, ds_bound @ y.abs() * scale),
            ("dk", shared(t(ds) @ x) * scale, shared(t(ds_bound) @ x.abs()) * scale),
            ("dv", shared(t(p) @ do), shared(t(p_bound) @ do.abs()))):
        got[name] = (value, u * value.abs() + bound + TINY)
    return got


def check(name, ours, value, bound):
    assert ours.shape == value.shape, name
    assert torch.isfinite(ours).all(), name
    over = (ours.double() - value).abs() - bound
    worst = over.max().item()
    assert worst <= 0, f"{name}: {worst:.3g} over the bound at {int(over.argmax())}"
