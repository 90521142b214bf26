"""CPU tests of the argument checks of the paged cache's entry points: no case reaches a launch."""
from __future__ import annotations

import pytest
import torch

import mini_flash_attention as mfa
from mini_flash_attention import capi

FAKE = 0x10000  # never dereferenced
INVALID = capi.MFA_ERR_INVALID_ARGUMENT


def attend(shared=False, ptr=FAKE, out=None, batch=2, heads=8, kv_heads=2, d=64, pages=10,
           page_size=16, columns=4, window=0, sinks=0, prefix=50, scale=0.125,
           dtype=capi.DTYPE_FP16, q_strides=None):
    out = ptr if out is None else out
    if shared:
        capi.shared_prefix_attention(ptr, ptr, ptr, ptr, prefix, ptr, ptr, out, ptr, 1 << 30, batch,
                                     heads, kv_heads, d, pages, page_size, columns, scale, dtype,
                                     q_strides=q_strides)
    else:
        capi.paged_attention(ptr, ptr, ptr, ptr, ptr, out, ptr, 1 << 30, batch, heads, kv_heads, d,
                             pages, page_size, columns, scale, window, sinks, dtype,
                             q_strides=q_strides)


COMMON = [
    ({"d": 48}, capi.MFA_ERR_HEAD_DIM, "D=32, D=64 and D=128"),
    ({"dtype": 2}, INVALID, "dtype must be"),
    ({"scale": -1.0}, INVALID, "scale must be positive"),
    ({"page_size": 8}, INVALID, "page size"),
    ({"page_size": 48}, INVALID, "page size"),
    ({"page_size": 512}, INVALID, "page size"),
    ({"kv_heads": 3}, INVALID, "multiple of the k / v heads"),
    ({"heads": 258}, INVALID, "at most 128 query heads"),
    ({"batch": -1}, INVALID, "negative extent"),
    ({"columns": -1}, INVALID, "negative extent"),
    ({"batch": 1 << 30}, INVALID, "B \\* H is too large"),
    ({"pages": 1 << 28}, INVALID, "too many tokens"),
    ({"columns": 1 << 28}, INVALID, "too many columns"),
    ({"batch": 1 << 20, "columns": 1 << 16}, INVALID, "batch \\* heads \\* tokens"),
    ({"q_strides": (0, 64)}, INVALID, "strides of q must be positive multiples of 8"),
    ({"q_strides": (512, -64)}, INVALID, "strides of q must be positive multiples of 8"),
    ({"q_strides": (516, 64)}, INVALID, "strides of q must be positive multiples of 8"),
    ({"q_strides": (1 << 31, 64)}, INVALID, "strides of q .* below 2\\^31"),
    ({"q_strides": (3, 64), "batch": 1, "pages": 0}, INVALID, "the cache has no pages"),
    ({"pages": 0}, INVALID, "the cache has no pages"),
    ({"ptr": 0}, INVALID, "null q"),
    ({"ptr": FAKE + 4}, INVALID, "q must be 16-byte aligned"),
    ({"out": FAKE + 2}, INVALID, "out must be 16-byte aligned"),
]


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("change,code,text", COMMON)
def test_attention_refused(shared, change, code, text):
    with pytest.raises(capi.MfaError, match=text) as e:
        attend(shared, **change)
    assert e.value.code == code


def test_window_and_prefix_refused():
    for change, text in (({"window": -1}, "window must not be negative"),
                         ({"sinks": -1}, "sinks must not be negative")):
        with pytest.raises(capi.MfaError, match=text):
            attend(**change)
    for change, text in (({"prefix": -1}, "negative extent"),
                         ({"prefix": 1 << 31}, "prefix is too long")):
        with pytest.raises(capi.MfaError, match=text):
            attend(True, **change)


@pytest.mark.parametrize("shared", [False, True])
def test_attention_of_nobody(shared):
    attend(shared, ptr=0, batch=0)
    attend(shared, ptr=0, heads=0)


def extend(ptr=FAKE, batch=2, columns=3, free=5, page_size=16, capacity=10):
    capi.extend_block_tables(*[ptr] * 7, batch, columns, free, page_size, capacity)


@pytest.mark.parametrize("change,text", [
    ({"batch": -1}, "negative extent"), ({"capacity": -1}, "negative extent"),
    ({"page_size": 0}, "page_size must be positive"), ({"free": 1 << 31}, "32 bits"),
    ({"capacity": 1 << 31}, "32 bits"), ({"ptr": 0}, "null block_table"),
    ({"ptr": FAKE + 2}, "4-byte aligned"),
])
def test_extend_refused(change, text):
    with pytest.raises(capi.MfaError, match=text) as e:
        extend(**change)
    assert e.value.code == INVALID


def append(ptr=FAKE, slots=FAKE, tokens=4, kv_heads=2, d=64, k_strides=(128, 64),
           v_strides=(128, 64), pages=3, page_size=16):
    capi.append_kv(ptr, ptr, ptr, ptr, slots, tokens, kv_heads, d, k_strides, v_strides, pages,
                   page_size)


@pytest.mark.parametrize("change,text", [
    ({"tokens": -1}, "negative extent"), ({"d": 60}, "multiple of 8"),
    ({"k_strides": (128, 60)}, "multiples of 8"), ({"v_strides": (4, 64)}, "multiples of 8"),
    ({"page_size": 0}, "page_size must be positive"), ({"pages": 1 << 28}, "too many tokens"),
    ({"tokens": 1 << 31}, "too large"), ({"kv_heads": 1 << 16}, "too large"),
    ({"ptr": 0}, "null k"), ({"ptr": FAKE + 8}, "16-byte aligned"), ({"slots": 0}, "null slots"),
    ({"slots": FAKE + 1}, "4-byte aligned"),
])
def test_append_refused(change, text):
    with pytest.raises(capi.MfaError, match=text) as e:
        append(**change)
    assert e.value.code == INVALID


def test_append_of_nothing():
    append(ptr=0, slots=0, tokens=0)
    append(ptr=0, slots=0, pages=0)


def test_workspace_query_refused():
    with pytest.raises(capi.MfaError, match="page size"):
        capi.paged_workspace_bytes(1, 4, 2, 64, 24, 4)
    assert capi.paged_workspace_bytes(0, 4, 2, 64, 16, 4) == 0


def test_cpu_tensors_refused():
    x = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    i = torch.zeros((2, 3), dtype=torch.int32)
    for call in (lambda: mfa.paged_attention(x[0], x, x, i, i[:, 0]),
                 lambda: mfa.shared_prefix_attention(x[0], x, x, i[0], 4, i, i[:, 0]),
                 lambda: mfa.append_kv(x[0], x[0], x, x, i[0]),
                 lambda: mfa.extend_block_tables(i, i[:, 0], i[:, 0], i[0], 16, 4)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
