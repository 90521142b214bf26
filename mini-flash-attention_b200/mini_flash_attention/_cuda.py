"""Extension loader and Python entry points.

Mirrors src/mini_flash_attention/_cuda.py:8-45 of the reference: a module-level cache of the
compiled extension and two thin wrappers that forward ``causal`` to it. Unlike the reference,
nothing is JIT-compiled at call time: the sm_100a library and its binding are built ahead of
time (``python -m mini_flash_attention._build``) into this package directory, and a missing
build is an error, never a fallback.
"""
import ctypes
from pathlib import Path

import torch

_EXTENSION = None
_PKG_DIR = Path(__file__).resolve().parent


def _load_extension():
    global _EXTENSION

    if _EXTENSION is not None:
        return _EXTENSION
    try:
        # The binding links libmfa_b200.so by soname; load that first from this directory.
        ctypes.CDLL(str(_PKG_DIR / "libmfa_b200.so"), mode=ctypes.RTLD_GLOBAL)
        from . import mfa_b200_C as ext  # noqa: PLC0415  (built in-tree)
    except (ImportError, OSError) as exc:
        raise RuntimeError(
            "mini_flash_attention: the sm_100a extension is not built in "
            f"{_PKG_DIR} ({exc}); run `python -m mini_flash_attention._build`"
        ) from exc
    _EXTENSION = ext
    return _EXTENSION


def forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False) -> torch.Tensor:
    """softmax(q k^T / sqrt(D)) v on [B, H, N, D] (or [B*H, N, D]) tensors: fp16 or bf16,
    D = 32, 64 or 128, any N; causal=True masks key index > query index."""
    return _load_extension().forward(q, k, v, causal)


def forward_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                causal: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """forward plus the row log-sum-exp ln(sum_k exp(q.k / sqrt(D))) as fp32 of shape q.shape[:-1]."""
    out, lse = _load_extension().forward_lse(q, k, v, causal)
    return out, lse


def backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
             lse: torch.Tensor, dout: torch.Tensor,
             causal: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of forward(q, k, v, causal) for the output gradient dout, given
    the forward's out and lse (forward_lse). D = 64, fp16 or bf16."""
    dq, dk, dv = _load_extension().backward(q, k, v, out, lse, dout.contiguous(), causal)
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal):
        out, lse = forward_lse(q, k, v, causal)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.causal = causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = backward(q, k, v, out, lse, dout, ctx.causal)
        return dq, dk, dv, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              causal: bool = False) -> torch.Tensor:
    """Differentiable forward: the tcgen05 forward kernel, with the tcgen05 backward kernels as
    its autograd backward (D = 64 for gradients)."""
    return _Attention.apply(q, k, v, causal)


def forward_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                   sinks: int = 0) -> torch.Tensor:
    """Attention in which a token sees the ``window`` newest tokens up to itself and the ``sinks``
    first ones of its sequence: query i sees key j if j <= i and (j > i - window or j < sinks).
    q is [B, H, N, D]; k and v are [B, Hkv, N, D], Hkv a divisor of H (query head h reads k / v
    head h // (H // Hkv)). fp16 or bf16, D = 32, 64 or 128, any N, scale 1/sqrt(D). Blocks of
    keys that no query of a block sees are skipped. A batch padded behind its sequences needs no
    mask: no token sees a later one (the padding has to be finite; a visible score of NaN or infinity
    makes its row NaN).

    q, k and v may be views, as of a fused projection: contiguous in D, other strides multiples of
    8. The output lies in memory as q does, [B, H, N, D] or (``x.view(B, N, H, D).transpose(1, 2)``)
    [B, N, H, D], and the gradients with it."""
    return _load_extension().forward_window(q, k, v, int(window), int(sinks), False, 0)[0]


def forward_window_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                       sinks: int = 0, rest: bool = False) -> tuple[torch.Tensor, ...]:
    """forward_window plus the row log-sum-exp over the visible keys as fp32 [B, H, N] and, with
    ``rest``, what the rounding of the output left, in its type and shape (see backward_window)."""
    return tuple(_load_extension().forward_window(q, k, v, int(window), int(sinks), True,
                                                  -1 if rest else 0))


def backward_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                    lse: torch.Tensor, dout: torch.Tensor, window: int, sinks: int = 0,
                    rest: torch.Tensor | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of forward_window for the output gradient dout, given its out and
    lse (forward_window_lse); dk and dv of a shared head are summed over its query heads. The types,
    head dims and views of forward_window; out, rest and dout in another layout are copied.

    With the output's ``rest`` its rounding does not reach dq and dk: with few visible keys it would
    be their largest error (without it 2.2 times that of their own rounding in rows that see two to
    four keys, 1.6 at 4 to 16, 1.49 at 16 to 64, 1.45 from there on; with it 1.48, 1.46, 1.45 and
    1.44). ``rest[:, :, :r]``, that of the first rows, helps those; the others count as without."""
    dq, dk, dv = _load_extension().backward_window(q, k, v, out, lse, dout, int(window),
                                                   int(sinks), rest)
    return dq, dk, dv


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                     sinks: int = 0) -> torch.Tensor:
    """Differentiable forward_window (gradients can be taken once: a gradient of a gradient
    raises, and so does a forward-mode derivative). It keeps q, k, v, the output and its log-sum-exp,
    and the output's rest (backward_window) of the first 1024 rows, below a window of 64 of all."""
    return _load_extension().window_attention(q, k, v, int(window), int(sinks))


def extend_block_tables(block_table: torch.Tensor, cached: torch.Tensor, added: torch.Tensor,
                        free_pages: torch.Tensor, page_size: int,
                        capacity: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages and slots for new tokens of a paged cache, without a word from the host.

    Request r has cached[r] tokens, token i in row i % page_size of page block_table[r, i //
    page_size], and gets added[r] more (int32 CUDA tensors, block_table [B, columns]). The pages
    that it needs beyond its ceil(cached / page_size) are the next ones of ``free_pages``, request
    after request; they are written into block_table in place, other entries stay. Returns

    * slots, int32 [capacity]: page * page_size + row of every new token, request after request,
      -1 behind the last one (``capacity`` is what the caller's k and v are padded to);
    * starts, int32 [B + 1]: where each request's tokens start in slots;
    * used, int32 [1]: how many of free_pages are taken. More than there are: pages were missing.

    Tokens without a page (the list or the table's row ends) have the slot -1, too.
    """
    slots, starts, used = _load_extension().extend_block_tables(
        block_table, cached, added, free_pages, int(page_size), int(capacity))
    return slots, starts, used


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              slots: torch.Tensor) -> None:
    """Copies the rows of k and v ([T, Hkv, D]; the token and head strides may be those of a fused
    projection) to their slots (int32 [T], extend_block_tables) of the caches [pages, Hkv,
    page_size, D], in place. Tokens whose slot is negative or past the cache are skipped; a slot
    may occur only once, and k and v must not be parts of the caches."""
    _load_extension().append_kv(k, v, k_cache, v_cache, slots)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, lengths: torch.Tensor, window: int = 0,
                    sinks: int = 0) -> torch.Tensor:
    """Attention of one token per request over a paged cache (the decoding form of
    forward_window): q [B, H, D], caches [pages, Hkv, page_size, D], block_table int32 [B,
    columns], lengths int32 [B], the query's own token among them; q's strides but that of D may be
    those of a fused projection. With ``window`` the ``window``
    newest tokens and the ``sinks`` first are visible, otherwise all. fp16 or bf16, D = 32, 64 or 128,
    page sizes 16 to 256 (powers of two), H a multiple of Hkv (up to 128 heads a k / v head),
    scale 1/sqrt(D). A request of length 0 gets 0. Lengths and table are read on the GPU: a
    captured call may be replayed with others of the same shape. Pages without visible tokens are
    not looked up, and rows that are not visible may hold anything.

    The table's width bounds the lengths and selects the kernel: few requests and a narrow table take
    one launch (1000 tokens of one request 7.3 us with 63 columns, 8.6 with 2048), so a program that
    knows its longest request passes the columns that it needs."""
    return _load_extension().paged_attention(q, k_cache, v_cache, block_table, lengths,
                                             int(window), int(sinks))


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            prefix_pages: torch.Tensor, prefix_length: int,
                            block_table: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
    """paged_attention for a batch whose requests share their first ``prefix_length`` tokens,
    stored once in the pages ``prefix_pages`` (int32) of the cache. block_table and lengths
    describe what each request has of its own behind the prefix (a length of 0: nothing). The
    prefix is read once and meets the queries of all requests in one matrix product."""
    return _load_extension().shared_prefix_attention(q, k_cache, v_cache, prefix_pages,
                                                     int(prefix_length), block_table, lengths)


def forward_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_begin: int, q_end: int,
                 out: torch.Tensor | None = None, causal: bool = False) -> torch.Tensor:
    """Forward of the query rows [q_begin, q_end) of every head, each against all N keys (with
    ``causal``, the keys up to its own index; the range must then start at a multiple of 256
    rows), written into ``out`` (same shape as q; a new tensor if None) and nowhere else: the
    per-GPU call of the query-row sharding used when B*H is smaller than the number of GPUs
    (every GPU holds the whole k and v)."""
    if out is None:
        out = torch.empty_like(q)
    _load_extension().forward_rows(q, k, v, out, int(q_begin), int(q_end), bool(causal))
    return out


def forward_bnhd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 causal: bool = False) -> torch.Tensor:
    """forward on [B, N, H, D] tensors (the flash-attn layout); the output has that layout."""
    return _load_extension().forward_bnhd(q, k, v, causal)


def forward_wmma(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False) -> torch.Tensor:
    return _load_extension().forward_wmma(q, k, v, causal)


def pinned_chunk_bounds(rows: int, chunks: int) -> list[int]:
    """Row bounds of the pieces of ``forward_pinned``: ``chunks`` pieces of decreasing size
    (weights 2^(c-2), ..., 2, 1, 1), every piece at least one row. The copy-in of all pieces
    bounds the pipeline; small last pieces keep short the compute and copy-out that follow
    it."""
    chunks = max(1, min(chunks, rows))
    weights = [2 ** (chunks - 2 - i) for i in range(chunks - 1)] + [1] if chunks > 1 else [1]
    total = sum(weights)
    bounds, acc = [0], 0
    for i, w in enumerate(weights):
        acc += w
        b = rows * acc // total
        b = max(b, bounds[-1] + 1)               # at least one row per piece
        b = min(b, rows - (chunks - 1 - i))      # leave a row for every later piece
        bounds.append(b)
    bounds[-1] = rows
    return bounds


def forward_pinned(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False,
                   out: torch.Tensor | None = None, chunks: int = 4,
                   device: torch.device | int | None = None) -> torch.Tensor:
    """Attention forward on host tensors: fp16 / bf16 q, k, v in (preferably pinned) CPU
    memory, result written to a host tensor (``out`` or a new pinned one).

    The batch*head rows are cut into ``chunks`` pieces of decreasing size
    (``pinned_chunk_bounds``) that move through three CUDA streams: piece i+1 is copied in
    while piece i is computed and piece i-1 is copied back, so the host<->device transfers
    overlap the kernels. The pipeline runs in the C++ extension (one call, no per-piece Python
    work). Synchronous: returns when the result is in ``out``. Same shape / dtype / error
    contract as ``forward``.
    """
    if q.is_cuda or k.is_cuda or v.is_cuda:
        raise RuntimeError("forward_pinned expects host tensors; use forward for CUDA tensors")
    if not (q.shape == k.shape == v.shape):
        raise RuntimeError("k must have the same shape as q")
    if q.dim() not in (3, 4):
        raise RuntimeError("q must have shape [B, H, N, D]")
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else
                       (device if isinstance(device, int) else device.index or 0))
    n, d = q.shape[-2], q.shape[-1]
    bh = q.numel() // (n * d) if n * d else 0
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, pin_memory=True)
    if bh == 0 or n == 0:
        return out
    if not out.is_contiguous():
        raise RuntimeError("out must be contiguous")
    q3, k3, v3 = (x.contiguous().reshape(bh, n, d) for x in (q, k, v))
    o3 = out.reshape(bh, n, d)
    _load_extension().forward_pinned(q3, k3, v3, o3, causal, pinned_chunk_bounds(bh, chunks),
                                     dev.index)
    return out
