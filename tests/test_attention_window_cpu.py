"""CPU tests of the windowed attention's argument checks: no case reaches a launch."""
from __future__ import annotations

import inspect

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi

FAKE = 0x10000  # never dereferenced


def call(direction="fwd", ptr=FAKE, batch=1, heads=4, kv_heads=2, n=256, d=64, window=16, sinks=0,
         scale=0.125, dtype=capi.DTYPE_FP16, layout=capi.LAYOUT_BHND, strides=None):
    fn, count = (capi.fwd_window, 4) if direction == "fwd" else (capi.bwd_window, 9)
    more = (0,) if direction == "fwd" else ()
    fn(*[ptr] * count, *more, batch, heads, kv_heads, n, d, window, sinks, scale, dtype, layout,
       strides=strides)


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("change,code,text", [
    ({"d": 48}, capi.MFA_ERR_HEAD_DIM, "D=32, D=64 and D=128"),
    ({"window": 0}, capi.MFA_ERR_INVALID_ARGUMENT, "window must be at least 1"),
    ({"window": -5}, capi.MFA_ERR_INVALID_ARGUMENT, "window must be at least 1"),
    ({"sinks": -1}, capi.MFA_ERR_INVALID_ARGUMENT, "sinks must not be negative"),
    ({"kv_heads": 3}, capi.MFA_ERR_INVALID_ARGUMENT, "multiple of the k / v heads"),
    ({"kv_heads": 0}, capi.MFA_ERR_INVALID_ARGUMENT, "multiple of the k / v heads"),
    ({"n": -1}, capi.MFA_ERR_INVALID_ARGUMENT, "negative extent"),
    ({"n": 1 << 31}, capi.MFA_ERR_INVALID_ARGUMENT, "N is too large"),
    ({"batch": 1 << 30}, capi.MFA_ERR_INVALID_ARGUMENT, "B \\* H is too large"),
    ({"n": 1 << 30, "batch": 1 << 20}, capi.MFA_ERR_INVALID_ARGUMENT, "N is too large"),
    ({"scale": 0.0}, capi.MFA_ERR_INVALID_ARGUMENT, "scale must be positive"),
    ({"scale": float("nan")}, capi.MFA_ERR_INVALID_ARGUMENT, "scale must be positive"),
    ({"dtype": 7}, capi.MFA_ERR_INVALID_ARGUMENT, "dtype must be"),
    ({"layout": 7}, capi.MFA_ERR_INVALID_ARGUMENT, "layout must be"),
    ({"strides": (1 << 16, 1 << 14, 0) * 3}, capi.MFA_ERR_INVALID_ARGUMENT, "strides of q, k"),
    ({"strides": (1 << 16, -64, 64) * 3}, capi.MFA_ERR_INVALID_ARGUMENT, "strides of q, k"),
    ({"batch": 2, "strides": (1 << 38, 64, 512) * 3}, capi.MFA_ERR_INVALID_ARGUMENT, "strides of"),
    ({"strides": (1 << 16, 64, 512) * 2 + (1 << 16, 64, 516)}, capi.MFA_ERR_INVALID_ARGUMENT,
     "strides of q, k"),
    ({"strides": (-1, 64, 512) * 3, "ptr": 0}, capi.MFA_ERR_INVALID_ARGUMENT, "null q"),
    ({"ptr": 0}, capi.MFA_ERR_INVALID_ARGUMENT, "null q"),
    ({"ptr": FAKE + 8}, capi.MFA_ERR_INVALID_ARGUMENT, "16-byte aligned"),
])
def test_refused(direction, change, code, text):
    with pytest.raises(capi.MfaError, match=text) as e:
        call(direction, **change)
    assert e.value.code == code


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("change", [{"batch": 0}, {"n": 0}, {"heads": 0}])
def test_nothing_to_do(direction, change):
    call(direction, ptr=0, **change)


def test_cpu_tensors_refused_and_signatures():
    q = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    for fn in (mfa.forward_window, mfa.forward_window_lse, mfa.window_attention):
        with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
            fn(q, q, q, 4)
        params = inspect.signature(fn).parameters
        more = ["rest"] if fn is mfa.forward_window_lse else []
        assert list(params) == ["q", "k", "v", "window", "sinks", *more]
        assert params["sinks"].default == 0 and all(not params[x].default for x in more)
