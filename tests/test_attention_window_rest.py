"""The rest of the windowed attention's output (what its rounding left) of the first rows only, which is
what window_attention keeps: the rows that see few keys are as exact in long sequences as in short
ones."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi
from window_reference import check, reference

FAKE = 0x10000  # never dereferenced


@pytest.mark.parametrize("rows", [-1, 257, 1 << 40])
def test_refused(rows):
    for call, count, more in ((capi.fwd_window, 4, (0,)), (capi.bwd_window, 9, ())):
        with pytest.raises(capi.MfaError, match="rest_rows must be within") as e:
            call(*[FAKE] * count, *more, 1, 4, 2, 256, 64, 16, 0, 0.125, rest_ptr=FAKE, rest_rows=rows)
        assert e.value.code == capi.MFA_ERR_INVALID_ARGUMENT


def test_misaligned():
    with pytest.raises(capi.MfaError, match="out_rest must be 16-byte aligned"):
        capi.fwd_window(*[FAKE] * 4, 0, 1, 4, 2, 256, 64, 16, 0, 0.125, rest_ptr=FAKE + 2, rest_rows=5)
    # without rows it is not looked at: the next check answers
    with pytest.raises(capi.MfaError, match="null q"):
        capi.fwd_window(0, *[FAKE] * 3, 0, 1, 4, 2, 256, 64, 16, 0, 0.125, rest_ptr=FAKE + 2,
                        rest_rows=0)


def inputs(b, h, hk, n, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((b, x, n, d), generator=g).to(dtype).cuda() for x in (h, hk, hk, h)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("n,window", [(1024, 1024), (1025, 1025), (1500, 64), (1500, 1500)])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_few_keys(n, window, d, dtype):
    """dq of the rows that see two to four keys, up to 16 and up to 64. Three roundings of about the
    same size make up the error: that of dq, that of dS and, through the row sums, that of the
    forward's weights, so it is at most 3 ** 0.5 times that of the first alone; the smallest group
    is 6144 values or more, whose norms are within 3 in 100 of that by chance. The output's rounding
    would make it 2.2 (D = 128: 1.86) in the first group."""
    q, k, v, dout = inputs(1, 32, 32, n, d, dtype, seed=n + window)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    dq = torch.autograd.grad(mfa.window_attention(*leaves, window), leaves, dout)[0]
    want = reference(*(x.detach() for x in leaves), window, 0, dout)["dq"][0]
    for first, last in ((1, 4), (4, 16), (16, 64)):
        value, x = want[:, :, first:last], dq[:, :, first:last]
        error = (x.double() - value).norm() / (value.to(dtype).double() - value).norm()
        assert error <= 3 ** 0.5 * 1.03, (first, error.item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("turned", [False, True], ids=["bhnd", "bnhd"])
def test_first_rows(turned, d, dtype):
    """The rest of the first rows is a part of the whole one, and each row's dq is the one with or
    without it."""
    b, h, hk, n, window, sinks = 2, 4, 2, 300, 130, 3
    x = inputs(b, h, hk, n, d, dtype, seed=d)
    want = reference(*x[:3], window, sinks, x[3])
    if turned:
        x = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in x]
    q, k, v, dout = x
    out, lse, rest = mfa.forward_window_lse(q, k, v, window, sinks, rest=True)
    whole = mfa.backward_window(q, k, v, out, lse, dout, window, sinks, rest)
    none = mfa.backward_window(q, k, v, out, lse, dout, window, sinks)
    for rows in (0, 1, 100, 128, 299, 300):
        part = rest[:, :, :rows]
        got = mfa.backward_window(q, k, v, out, lse, dout, window, sinks, part)
        assert torch.equal(got[0][:, :, :rows], whole[0][:, :, :rows])
        assert torch.equal(got[0][:, :, rows:], none[0][:, :, rows:])
        for name, g in zip(("dq", "dk", "dv"), got):
            check(name, g, *want[name])
        again = mfa.backward_window(q, k, v, out, lse, dout, window, sinks, part.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    # the entry of the C library, in memory that must not be written behind the rows
    layout = capi.LAYOUT_BNHD if turned else capi.LAYOUT_BHND
    flat = [t.transpose(1, 2).contiguous() if turned else t for t in (q, k, v)]
    for rows in (1, 100, 300):
        shape = (b, rows, h, d) if turned else (b, h, rows, d)
        size = b * h * rows * d
        room = torch.full((size + 512,), 7.0, device="cuda", dtype=dtype)
        mine, mine_lse = torch.empty_like(q), torch.empty_like(lse)
        capi.fwd_window(*(t.data_ptr() for t in flat), mine.data_ptr(), mine_lse.data_ptr(), b, h, hk,
                        n, d, window, sinks, d ** -0.5,
                        capi.DTYPE_BF16 if dtype == torch.bfloat16 else capi.DTYPE_FP16, layout,
                        torch.cuda.current_stream().cuda_stream, rest_ptr=room.data_ptr(),
                        rest_rows=rows)
        got = room[:size].view(shape)
        assert torch.equal(got.transpose(1, 2) if turned else got, rest[:, :, :rows])
        assert (room[size:] == 7).all() and torch.equal(mine_lse, lse)
    for bad in (rest[:, :1], torch.cat((rest, rest), 2), rest[0], rest[..., :16]):
        with pytest.raises(RuntimeError, match="rest must have"):
            mfa.backward_window(q, k, v, out, lse, dout, window, sinks, bad)


@pytest.mark.gpu
def test_kept_memory():
    """A long sequence keeps the output, its log-sum-exp and 1024 rows."""
    q, k, v, _ = inputs(1, 8, 2, 8192, 64, torch.bfloat16, seed=1)
    q.requires_grad_()
    out = mfa.window_attention(q, k, v, 2048)
    del out
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = mfa.window_attention(q, k, v, 2048)
    whole = 8 * 8192 * 64 * 2
    assert torch.cuda.memory_allocated() - before <= whole + 8 * 8192 * 4 + whole // 8 + 4096
    assert out.shape == q.shape
