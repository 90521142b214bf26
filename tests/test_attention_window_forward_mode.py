"""window_attention refuses forward-mode derivatives, with and without reverse-mode gradients; a tangent
dropped without a word would read as a derivative of 0."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import mini_flash_attention as mfa


def refused(device):
    new = lambda h: torch.randn((1, h, 100, 64), device=device).half()  # noqa: E731
    for which in range(3):
        for requires_grad, mode in ((False, torch.enable_grad), (True, torch.enable_grad),
                                    (False, torch.no_grad)):
            x = [new(4), new(2), new(2)]
            x[(which + 1) % 3].requires_grad_(requires_grad)
            with fwAD.dual_level(), mode():
                x[which] = fwAD.make_dual(x[which], torch.randn_like(x[which]))
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    mfa.window_attention(*x, 20, 1)


def test_refused_cpu():
    refused("cpu")


@pytest.mark.gpu
def test_refused_gpu():
    refused("cuda")
    # inside a level, tensors without a tangent are as ever
    q, k = torch.randn((1, 4, 100, 64), device="cuda").half(), torch.randn((1, 2, 100, 64),
                                                                           device="cuda").half()
    want = mfa.forward_window(q, k, k, 20, 1)
    with fwAD.dual_level():
        assert torch.equal(mfa.window_attention(q, k, k, 20, 1), want)
        leaf = q.clone().requires_grad_()
        mfa.window_attention(leaf, k, k, 20, 1).sum().backward()
    assert leaf.grad is not None
