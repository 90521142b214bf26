"""A paged cache for the tests, and the attention over it in 64 bits with the bounds that
window_reference.py derives: weights rounded to the type before the product with v, exponentials
and 32-bit sums off by at most DELTA together, one rounding of the output."""
from __future__ import annotations

import torch

from window_reference import DELTA, TINY, half_step


def seen_positions(n: int, window: int, sinks: int) -> list[int]:
    return [j for j in range(n) if not window or j >= n - window or j < sinks]


class Cache:
    """A cache in which only what the requests see is finite, and a table in which only what they
    look up is a page; everything else is NaN or out of range."""

    def __init__(self, lengths, kv_heads, d, page, dtype, *, window=0, sinks=0, prefix=0, columns=None,
                 seed=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lengths]
        shared = -(-prefix // page)
        total = sum(need) + shared + 3
        order = torch.randperm(total, generator=g).tolist()
        self.prefix, self.prefix_pages = prefix, order[:shared]
        columns = max(1, max(need, default=0)) if columns is None else columns
        self.table = torch.full((len(lengths), columns), 1 << 30, dtype=torch.int32)
        self.keys, self.values = [], []
        shape = (total, kv_heads, page, d)
        k, v = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))

        def fill(pages, positions):
            at = torch.tensor(positions, dtype=torch.long)
            rows = torch.tensor(pages, dtype=torch.long)[at // page] if positions else at
            new = [torch.randn((len(positions), kv_heads, d), generator=g).to(dtype)
                   for _ in range(2)]
            k[rows, :, at % page], v[rows, :, at % page] = new
            return [x.cuda().double() for x in new]

        self.shared = fill(self.prefix_pages, list(range(prefix)))
        at = shared
        for r, n in enumerate(lengths):
            pages, at = order[at:at + need[r]], at + need[r]
            seen = seen_positions(n, window, sinks)
            for j in seen:
                self.table[r, j // page] = pages[j // page]
            x, y = fill(pages, seen)
            self.keys.append(x)
            self.values.append(y)
        self.k, self.v = k.cuda(), v.cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32)
        self.dtype = dtype

    def tensors(self):
        return self.k, self.v, self.table.cuda(), self.lengths.cuda()

    def pages(self):
        return torch.tensor(self.prefix_pages, dtype=torch.int32, device="cuda")

    def reference(self, q):
        """(value, bound) of the attention of q [B, H, D]."""
        u, q = half_step(self.dtype), q.cuda()
        floor = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        value = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        bound = torch.full_like(value, TINY)
        for r, (k, v) in enumerate(zip(self.keys, self.values)):
            k, v = (torch.cat((a, b)) for a, b in zip(self.shared, (k, v)))
            if not len(k):
                continue
            hk, d = k.shape[1:]
            x = q[r].double().reshape(hk, -1, d)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", x, k) * d ** -0.5, -1)
            out = torch.einsum("hgn,nhd->hgd", p, v)
            size = torch.einsum("hgn,nhd->hgd", p, v.abs())
            most = v.abs().sum(0)[:, None]
            value[r] = out.reshape(q[r].shape)
            bound[r] += (u * out.abs() + (u + DELTA) * size + floor * most).reshape(q[r].shape)
        return value, bound


def queries(batch, heads, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((batch, heads, d), generator=g).to(dtype)


def check(out, value, bound):
    assert out.shape == value.shape
    assert torch.isfinite(out).all()
    worst = ((out.double() - value).abs() - bound).max().item() if out.numel() else 0.0
    assert worst <= 0, f"{worst:.3g} over the bound"
