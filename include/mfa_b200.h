/*
 * mini-flash-attention for B200 (sm_100a) -- C ABI of the attention forward.
 *
 * Plain pointers and sizes only; no torch or C++ types cross this boundary, and no call
 * throws. Every entry point returns MFA_OK (0) or an MFA_ERR_* code; the message of the last
 * failure on the calling thread is available from mfa_last_error_string().
 *
 * Tensor contract (identical to the reference binding, src/mini_flash_attention/flash_attn.cpp:
 * 45-109): q, k, v and out are device pointers to contiguous fp16 arrays laid out [BH, N, D]
 * (BH = batch * heads), D = 64, out is written completely by the kernel. Launches are
 * asynchronous on `stream` (a cudaStream_t; NULL = legacy default stream) and on the device
 * that is current for the calling thread, exactly like the reference launchers.
 */
#ifndef MFA_B200_H
#define MFA_B200_H

#include <stdint.h>

#if defined(__GNUC__)
#define MFA_API __attribute__((visibility("default")))
#else
#define MFA_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum mfa_status_code {
  MFA_OK = 0,
  MFA_ERR_INVALID_ARGUMENT = 1, /* null / misaligned pointer, negative or oversized extent */
  MFA_ERR_HEAD_DIM = 2,         /* unsupported D (64 only, or 32 / 64 / 128 for mfa_fwd) */
  MFA_ERR_SEQ_LEN = 3,          /* N not a multiple of 64 (mfa_fwd_simple_f16 only) */
  MFA_ERR_CAUSAL = 4,           /* reserved: causal masking is supported by every entry point */
  MFA_ERR_CUDA = 5,             /* CUDA runtime or driver error; message has the details */
  MFA_ERR_DEVICE = 6            /* current device is not an sm_100 (B200-class) GPU */
};

/*
 * Attention forward, tcgen05 kernel with two query tiles (256 rows) per CTA.
 * Replaces the reference launcher launch_flash_attn_forward
 * (src/mini_flash_attention/flash_attn_cuda.cu:370-420): same arguments, the same D == 64 check
 * and message; any N >= 1 (the reference requires N % 128 == 0, flash_attn_cuda.cu:402-407).
 * `scale` multiplies q.k before the softmax (the reference binding passes 1/sqrt(D),
 * flash_attn.cpp:94); it must be positive and finite (MFA_ERR_INVALID_ARGUMENT otherwise).
 * q, k, v and out must be memory of the current device (checked: other pointers return
 * MFA_ERR_INVALID_ARGUMENT before any launch). causal != 0 masks
 * key index > query index (the reference launcher rejects causal, flash_attn_cuda.cu:408-410;
 * the mask is the one its test and benchmark build, tests/test_forward.py:30-32).
 * bh == 0 or n == 0 is a no-op that returns MFA_OK.
 */
MFA_API int mfa_fwd_f16(const void* q, const void* k, const void* v, void* out, int64_t bh, int64_t n,
                int32_t d, float scale, int32_t causal, void* stream);

/*
 * Attention forward, single-query-tile tcgen05 kernel (128 rows per CTA, 2-stage K/V ring).
 * Replaces the reference's WMMA launcher, declared as launch_flash_attn_forward_wmma
 * (src/mini_flash_attention/flash_attn.cpp:21-31) and implemented at
 * src/mini_flash_attention/flash_attn_wmma_cuda.cu:253-289: checks D == 64 and N % 64 == 0
 * with that launcher's messages; causal != 0 masks key index > query index (that launcher
 * rejects causal, flash_attn_wmma_cuda.cu:275-277).
 */
MFA_API int mfa_fwd_simple_f16(const void* q, const void* k, const void* v, void* out, int64_t bh,
                       int64_t n, int32_t d, float scale, int32_t causal, void* stream);

/* Element type and memory layout of mfa_fwd's q, k, v and out. */
enum mfa_dtype { MFA_DTYPE_FP16 = 0, MFA_DTYPE_BF16 = 1 };
enum mfa_layout {
  MFA_LAYOUT_BHND = 0, /* [B, H, N, D] contiguous: the reference's layout */
  MFA_LAYOUT_BNHD = 1  /* [B, N, H, D] contiguous: the flash-attn style layout */
};

/*
 * General forward: `dtype` (fp16 or bf16; out has the same type), `layout` (above), B = batch
 * and H = heads given separately, head dim d = 32, 64 or 128 (others: MFA_ERR_HEAD_DIM, "This
 * kernel supports only D=32, D=64 and D=128"), any N, same causal semantics as mfa_fwd_f16; bf16 rounds P to bf16 for the P.V product, as fp16
 * inputs round it to fp16. No counterpart in the reference launchers, which take fp16
 * [B*H, N, D] only; its benchmark exposes bf16 and converts to [B, N, H, D] for flash-attn
 * (benchs/benchmark_forward.py:162-167, 188, 210-215). mfa_fwd_f16(q, k, v, out, bh, ...)
 * equals mfa_fwd(q, k, v, out, 1, bh, ..., MFA_DTYPE_FP16, MFA_LAYOUT_BHND, stream).
 */
MFA_API int mfa_fwd(const void* q, const void* k, const void* v, void* out, int64_t batch,
                    int64_t heads, int64_t n, int32_t d, float scale, int32_t causal,
                    int32_t dtype, int32_t layout, void* stream);

/*
 * mfa_fwd restricted to the query rows [q_begin, q_end) of every head: q, k, v and out are the
 * whole tensors (as for mfa_fwd), every query row in the range attends to all N keys, and only
 * those rows of out are written. For multi-GPU sharding when B*H is smaller than the number of
 * GPUs: each GPU holds the whole k and v and takes a range of query rows. causal != 0 masks
 * key index > query index as in mfa_fwd (absolute indices); a causal range must start at a
 * multiple of 256 rows (MFA_ERR_INVALID_ARGUMENT otherwise). 0 <= q_begin <= q_end <= N.
 * No counterpart in the reference, which has no multi-GPU mode.
 */
MFA_API int mfa_fwd_rows(const void* q, const void* k, const void* v, void* out, int64_t batch,
                         int64_t heads, int64_t n, int64_t q_begin, int64_t q_end, int32_t d,
                         float scale, int32_t causal, int32_t dtype, int32_t layout,
                         void* stream);

/*
 * mfa_fwd that also writes the row log-sum-exp of the scaled scores,
 * lse[bh * N + row] = ln(sum over keys of exp(scale * q.k)), fp32 [B*H, N] whatever the
 * layout: the state the backward pass needs. No counterpart in the reference (no backward).
 */
MFA_API int mfa_fwd_lse(const void* q, const void* k, const void* v, void* out, float* lse,
                        int64_t batch, int64_t heads, int64_t n, int32_t d, float scale,
                        int32_t causal, int32_t dtype, int32_t layout, void* stream);

/*
 * Backward pass (D = 64, fp16 or bf16, either layout, any N, optional causal mask): from q,
 * k, v, the forward output `out`, its gradient `dout` and `lse` of mfa_fwd_lse (same scale and
 * causal), writes dq, dk, dv (type and layout of q). dV = P^T dout, dS = P * (dout v^T - D)
 * with D = rowsum(dout * out), dq = scale * dS k, dk = scale * dS^T q. Two tcgen05 passes
 * (dq; dk and dv) and a small row pass; a stream-ordered scratch of 8 bytes per row from the
 * library's pool. Other D: MFA_ERR_HEAD_DIM "The backward pass supports only D=64". No
 * counterpart in the reference: its README lists the backward pass as future work
 * (README.md:125).
 */
MFA_API int mfa_bwd(const void* q, const void* k, const void* v, const void* out,
                    const void* dout, const float* lse, void* dq, void* dk, void* dv,
                    int64_t batch, int64_t heads, int64_t n, int32_t d, float scale,
                    int32_t causal, int32_t dtype, int32_t layout, void* stream);

/*
 * Attention with a sliding window and sink tokens, and k / v heads shared by groups of query
 * heads: query i sees key j if j <= i and (j > i - window or j < sinks); query head h reads k / v
 * head h / (heads / kv_heads). q and out have `heads` heads, k and v `kv_heads` (a divisor of
 * heads); d = 32, 64 or 128, any n, window >= 1 (at n or more: causal attention), sinks >= 0.
 * lse (may be NULL): the row log-sum-exp over the visible keys, fp32 [B*H, N]. out_rest (may be
 * NULL): what the rounding of out left, in its type and shape, for mfa_bwd_window. Key blocks that
 * no row of a query block sees are neither read nor computed. k and v must be finite also where
 * they are masked, as for mfa_fwd; a visible score of NaN or +inf makes its row NaN. `strides` (NULL: those of `layout`) are the element strides of
 * q's, k's and v's batch, head and token dimension, nine values in that order: positive multiples
 * of 8 (any value for a dimension of one element), as of the parts of a fused projection. The
 * other tensors are contiguous in `layout`. No counterpart in the reference.
 */
MFA_API int mfa_fwd_window(const void* q, const void* k, const void* v, void* out, float* lse,
                           void* out_rest, int64_t batch, int64_t heads, int64_t kv_heads,
                           int64_t n, int32_t d, int64_t window, int64_t sinks, float scale,
                           int32_t dtype, int32_t layout, const int64_t* strides, void* stream);

/*
 * mfa_fwd_window with an out_rest of the first rest_rows rows of every head only: its extents are
 * [batch, heads, rest_rows, d], its memory order that of `layout`, 0 <= rest_rows <= n. The first rows of a
 * sequence see few keys whatever its length. No counterpart in the reference.
 */
MFA_API int mfa_fwd_window_rest(const void* q, const void* k, const void* v, void* out, float* lse,
                                void* out_rest, int64_t rest_rows, int64_t batch, int64_t heads,
                                int64_t kv_heads, int64_t n, int32_t d, int64_t window,
                                int64_t sinks, float scale, int32_t dtype, int32_t layout,
                                const int64_t* strides, void* stream);

/*
 * Backward of mfa_fwd_window, of the same types and head dims: dq, dk, dv from q, k, v, out, lse,
 * dout. dk and dv of a shared head are the sum over its query heads, in a fixed order. With out_rest
 * (may be NULL) the rounding of out does not reach dq and dk; where rows see few keys it would be
 * their largest error (without it 2.2 times that of their own rounding in rows that see two to four
 * keys, 1.49 at 16 to 64, 1.45 from there on; with it 1.48, 1.45 and 1.44). Takes 8 bytes per query row and up to a few hundred partial sums of 64 KB (D =
 * 128: 128 KB; of key blocks that many queries see) from the library's stream-ordered pool. No
 * counterpart in the reference.
 */
MFA_API int mfa_bwd_window(const void* q, const void* k, const void* v, const void* out,
                           const void* dout, const float* lse, const void* out_rest, void* dq,
                           void* dk, void* dv, int64_t batch, int64_t heads, int64_t kv_heads,
                           int64_t n, int32_t d, int64_t window, int64_t sinks, float scale,
                           int32_t dtype, int32_t layout, const int64_t* strides, void* stream);

/* mfa_bwd_window with the out_rest of mfa_fwd_window_rest. No counterpart in the reference. */
MFA_API int mfa_bwd_window_rest(const void* q, const void* k, const void* v, const void* out,
                                const void* dout, const float* lse, const void* out_rest,
                                int64_t rest_rows, void* dq, void* dk, void* dv, int64_t batch,
                                int64_t heads, int64_t kv_heads, int64_t n, int32_t d,
                                int64_t window, int64_t sinks, float scale, int32_t dtype,
                                int32_t layout, const int64_t* strides, void* stream);

/*
 * Paged key / value cache. k_cache and v_cache are contiguous [pages, kv_heads, page_size, d]
 * arrays of 16-bit elements; request r's token at position i is row i % page_size of page
 * block_table[r][i / page_size] (int32 [batch, columns]); slot s is row s % page_size of page
 * s / page_size. No counterpart in the reference, which has no cache.
 *
 * mfa_extend_block_tables makes room for added[r] tokens behind the cached[r] ones of every
 * request (both int32 [batch]; negative counts as 0). Columns from ceil(cached / page_size) on are
 * filled with the next entries of free_pages, request after request; slots[0..capacity) gets the
 * slots of the new tokens, request after request, and -1 behind the last; starts[batch + 1] the
 * requests' first indices in slots; *used the number of pages taken. A token whose page would be
 * behind the row's last column or the last free page has the slot -1 (*used counts the pages past
 * free_count, so used > free_count says that pages are missing). Tokens past `capacity` get pages
 * but no slot. Entries of block_table in other columns are left as they are. page_size >= 1.
 */
MFA_API int mfa_extend_block_tables(int32_t* block_table, const int32_t* cached,
                                    const int32_t* added, const int32_t* free_pages,
                                    int32_t* slots, int32_t* starts, int32_t* used, int64_t batch,
                                    int64_t columns, int64_t free_count, int64_t page_size,
                                    int64_t capacity, void* stream);

/*
 * Copies token t's rows of k and v ([tokens, kv_heads, d]; token and head strides in elements,
 * multiples of 8; d a multiple of 8) to slot slots[t]; tokens whose slot is outside the cache are
 * skipped. A slot may occur once in a call: of two tokens with one slot either may stay, also
 * in parts. k and v must not overlap the caches.
 */
MFA_API int mfa_append_kv(const void* k, const void* v, void* k_cache, void* v_cache,
                          const int32_t* slots, int64_t tokens, int64_t kv_heads, int64_t d,
                          int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                          int64_t v_head_stride, int64_t pages, int64_t page_size, void* stream);

/*
 * Attention of one query token per request over the cache: q and out are [batch, heads, d], q with
 * element strides that are positive multiples of 8 (any value for a dimension of one element), d =
 * 32, 64 or 128, heads a multiple of kv_heads (at most 128 query heads a k / v head), page_size 16, 32,
 * 64, 128 or 256. Request r has lengths[r] tokens (int32; clamped to [0, columns * page_size]), the
 * query's own among them; visible are all of them, or with window > 0 those in the newest
 * `window` positions and the first `sinks`. out is 0 for a request that sees nothing. Only pages
 * with visible tokens are looked up and read, and what else their rows hold (NaN too) does not
 * matter. A looked-up page outside the cache reads as zeros and sets the device status word
 * (mfa_device_status) to 0x200. A visible score of NaN or +inf makes its row of out NaN. `columns`
 * selects the kernel: few requests of a narrow table take one launch and no workspace, the same
 * requests with a wide table two launches. The workspace (256-byte aligned, mfa_paged_workspace_bytes) must
 * not be shared by calls that may overlap; nothing in it has to be kept between calls.
 */
MFA_API int mfa_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                                const int32_t* block_table, const int32_t* lengths, void* out,
                                void* workspace, uint64_t workspace_bytes, int64_t batch,
                                int64_t heads, int64_t kv_heads, int32_t d, int64_t q_batch_stride,
                                int64_t q_head_stride, int64_t pages, int64_t page_size,
                                int64_t columns, int64_t window, int64_t sinks, float scale,
                                int32_t dtype, void* stream);

/*
 * The same for requests that share their first prefix_length tokens, in the pages prefix_pages
 * (int32, ceil(prefix_length / page_size) of them) of the same cache; block_table and lengths
 * tell each request's own tokens behind them. The prefix is read once for the whole batch.
 */
MFA_API int mfa_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache,
                                        const int32_t* prefix_pages, int64_t prefix_length,
                                        const int32_t* block_table, const int32_t* lengths,
                                        void* out, void* workspace, uint64_t workspace_bytes,
                                        int64_t batch, int64_t heads, int64_t kv_heads, int32_t d,
                                        int64_t q_batch_stride, int64_t q_head_stride,
                                        int64_t pages, int64_t page_size, int64_t columns,
                                        float scale, int32_t dtype, void* stream);

/* Workspace, in bytes, of mfa_paged_attention (prefix_length 0) or mfa_shared_prefix_attention on
 * the current device; launches and allocates nothing. */
MFA_API int mfa_paged_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int32_t d,
                                      int64_t page_size, int64_t columns, int64_t prefix_length,
                                      uint64_t* bytes);

/*
 * Device scratch, in bytes, that one call of mfa_fwd (or mfa_fwd_f16 / mfa_fwd_lse, and with d
 * = 64 and fp16 mfa_fwd_f16_noalloc) takes on the current device for these extents: 0 when
 * whole query blocks fill the SMs evenly, else the split plan's partial-result slots (2 x
 * (256 rows x (D + 2) floats) per CTA, one CTA per SM). dtype and layout do not change it.
 * Nothing is launched or allocated. The allocating entry points take it from a stream-ordered
 * pool of the library (outside any framework allocator) and return it on the same stream;
 * the output tensor is the caller's. No counterpart in the reference, whose launchers need
 * no scratch (its benchmark reports the allocator's peak over the calls,
 * benchs/benchmark_forward.py:266-289).
 */
MFA_API int mfa_fwd_workspace_bytes(int64_t batch, int64_t heads, int64_t n, int32_t d,
                                    int32_t causal, uint64_t* bytes);

/* Size of the static device scratch array used by mfa_fwd_f16_noalloc (20 MiB). */
#define MFA_NOALLOC_SCRATCH_BYTES 20971520u

/*
 * Allocation-free variant of mfa_fwd_f16: same kernels, arguments, checks, messages and
 * results, but it calls no cudaMalloc / cudaFree / stream-ordered or library allocator.
 * No counterpart in the reference (whose launchers need no scratch at all).
 *
 * For callers that cannot allocate device memory on this path: an engine or framework that
 * reserves the device's memory for its own allocator at start-up (a further allocation may
 * fail or fragment its pool), and code that must not enter the CUDA allocator in the middle
 * of a step (an allocation there can block or fail at a point the caller cannot recover from).
 *
 * When B*H*(N/256) does not fill the GPU evenly, the key dimension is split and partial
 * results are merged; mfa_fwd_f16 takes that scratch from a stream-ordered pool, this entry
 * point from one file-scope device array of MFA_NOALLOC_SCRATCH_BYTES in the library's device
 * image (2 x 67,584 bytes per CTA: enough for up to 155 SMs; a B200 has 148). A launch that
 * would need more returns MFA_ERR_INVALID_ARGUMENT with the required size in the message.
 *   - Nothing in the scratch has to start at zero: every part a call reads, it first writes.
 *   - The array is shared by every call on a device: calls that overlap on the GPU (issued
 *     on different streams without ordering between them) race on it and may return wrong
 *     results. Serialise them, e.g. by issuing them on one stream.
 *   - The first call on each device runs its one-time set-up (device checks, kernel
 *     attributes, cudaGetSymbolAddress of the scratch); make that first call before any
 *     stream capture. If the set-up fails with a CUDA error, the call returns MFA_ERR_CUDA
 *     and the next call tries the set-up again; only a device of the wrong architecture
 *     fails every call.
 *   - Memory cost to every user of the library: the array belongs to the library's device
 *     image, so each device on which any kernel of this library is loaded holds
 *     MFA_NOALLOC_SCRATCH_BYTES for it until the process exits, whether or not this entry
 *     point is ever called.
 */
MFA_API int mfa_fwd_f16_noalloc(const void* q, const void* k, const void* v, void* out, int64_t bh,
                        int64_t n, int32_t d, float scale, int32_t causal, void* stream);

/* Message of the last failing call made by this thread ("" if none). Replaces the
 * std::runtime_error text of the reference launchers and check_cuda
 * (src/mini_flash_attention/utils.cuh:15-21). */
MFA_API const char* mfa_last_error_string(void);

/*
 * Reads the device-side status word of `device` (synchronises that device first).
 * 0 = every kernel finished normally; 0x100 + site = a bounded mbarrier wait in some CTA
 * expired and that CTA unwound without writing its output tile; 0x200 = a block table named a
 * page outside its cache. If `reset` is non-zero the
 * word is cleared afterwards. No reference counterpart: the reference kernels have no
 * bounded waits.
 */
MFA_API int mfa_device_status(int device, int* status, int reset);

/* Per-wait watchdog limit in nanoseconds used by later launches (default 2 s, min 1 ms).
 * No reference counterpart. */
MFA_API int mfa_set_watchdog_ns(uint64_t ns);

/*
 * Self-test of the watchdog path: launches a one-CTA kernel on `stream` that allocates TMEM,
 * waits on an mbarrier that nothing arrives at with the given limit, records the expiry in
 * its own status word, frees TMEM and returns. *status_out receives that word (0x100 + site
 * when the wait expired as designed). Synchronises `stream`. No reference counterpart.
 */
MFA_API int mfa_watchdog_selftest(void* stream, uint64_t timeout_ns, int* status_out);

/* Library version string. */
MFA_API const char* mfa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MFA_B200_H */
