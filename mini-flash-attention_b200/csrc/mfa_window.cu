// C-ABI launchers of the windowed attention (sliding window with sink tokens, grouped k / v heads):
// forward and backward. Query i sees key j if j <= i and (j > i - window or j < sinks); query head
// h reads k / v head h / (heads / kv_heads). The kernels are the window variants of the forward and
// backward kernels (mfa_fwd_kernel.cuh, mfa_bwd_kernel.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/mfa_b200.h"
#include "mfa_bwd_kernel.cuh"
#include "mfa_fwd_kernel.cuh"
#include "mfa_host.h"

namespace mfa {
namespace {

// The head dim's tile count and ring depth are the causal forward's.
template <bool kBF16, int D>
using Window = FwdConfig<D == 128 ? 1 : 2, D == 128 ? 2 : 3, true, kBF16, D, true, true>;

template <class Cfg>
auto* window_kernel() {
  return &mfa_fwd_kernel<Cfg::NQ, Cfg::STAGES, true, Cfg::kBF16, Cfg::kHeadDim, true, true>;
}

template <bool kBF16>
constexpr int window_bwd_smem() {
  using CQ = BwdConfig<false, true, kBF16, true>;
  using CK = BwdConfig<true, true, kBF16, true>;
  return CQ::kSmemBytes > CK::kSmemBytes ? CQ::kSmemBytes : CK::kSmemBytes;
}

template <bool kBF16>
constexpr int window_bwd128_smem() {
  constexpr int kv = BwdDK128<kBF16>::kSmemBytes > BwdDV128<kBF16>::kSmemBytes
                         ? BwdDK128<kBF16>::kSmemBytes
                         : BwdDV128<kBF16>::kSmemBytes;
  return kv > BwdDQ128<kBF16>::kSmemBytes ? kv : BwdDQ128<kBF16>::kSmemBytes;
}

template <bool kBF16>
cudaError_t set_attributes() {
  const auto smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(window_kernel<Window<kBF16, 32>>(), smem,
                                       Window<kBF16, 32>::kSmemBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(window_kernel<Window<kBF16, 64>>(), smem,
                             Window<kBF16, 64>::kSmemBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(window_kernel<Window<kBF16, 128>>(), smem,
                             Window<kBF16, 128>::kSmemBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(mfa_bwd_window_kernel<kBF16>, smem, window_bwd_smem<kBF16>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(mfa_bwd_window128_kernel<kBF16>, smem, window_bwd128_smem<kBF16>());
  return e;
}

int prepare(int dev) {
  static host::SetUp set_up[host::kMaxDevices];
  return set_up[dev]([]() -> int {
    cudaError_t e = set_attributes<false>();
    if (e == cudaSuccess) e = set_attributes<true>();
    return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "window kernel set-up");
  });
}

// The arguments of both directions, checked.
struct Problem {
  int64_t batch, heads, kv_heads, n, window, sinks;
  int32_t d, dtype, layout;
  float scale;
  int64_t rest_rows;  // of the output's rest, if it is given
  host::Strides q, k, v;
};

// Strides of q, k and v: those of the layout, or the caller's {batch, head, token} of each.
int set_strides(Problem& w, const int64_t* strides) {
  const struct {
    host::Strides* to;
    int64_t heads;
  } tensors[3] = {{&w.q, w.heads}, {&w.k, w.kv_heads}, {&w.v, w.kv_heads}};
  for (int i = 0; i < 3; ++i) {
    *tensors[i].to = host::strides_of(w.layout, tensors[i].heads, w.n, w.d);
    if (!strides) continue;
    const int64_t extents[3] = {w.batch, tensors[i].heads, w.n};
    int64_t* const to[3] = {&tensors[i].to->b, &tensors[i].to->h, &tensors[i].to->n};
    for (int x = 0; x < 3; ++x) {
      const int64_t s = strides[3 * i + x];
      if (extents[x] <= 1) {
        *to[x] = w.d;  // a dimension of one element may have any stride
      } else if (s <= 0 || s % 8 != 0 || s >= int64_t{1} << 38) {
        return host::fail(MFA_ERR_INVALID_ARGUMENT,
                          "the strides of q, k and v must be positive multiples of 8 elements");
      } else {
        *to[x] = s;
      }
    }
  }
  return MFA_OK;
}

int check(Problem& w) {
  if (w.batch < 0 || w.heads < 0 || w.kv_heads < 0 || w.n < 0)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "negative extent");
  if (w.d != 32 && w.d != 64 && w.d != 128)
    return host::fail(MFA_ERR_HEAD_DIM, "This kernel supports only D=32, D=64 and D=128");
  if (w.dtype != MFA_DTYPE_FP16 && w.dtype != MFA_DTYPE_BF16)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "dtype must be MFA_DTYPE_FP16 or MFA_DTYPE_BF16");
  if (w.layout != MFA_LAYOUT_BHND && w.layout != MFA_LAYOUT_BNHD)
    return host::fail(MFA_ERR_INVALID_ARGUMENT,
                      "layout must be MFA_LAYOUT_BHND or MFA_LAYOUT_BNHD");
  if (!(w.scale > 0.0f) || !std::isfinite(w.scale))
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if (w.window < 1) return host::fail(MFA_ERR_INVALID_ARGUMENT, "window must be at least 1");
  if (w.sinks < 0) return host::fail(MFA_ERR_INVALID_ARGUMENT, "sinks must not be negative");
  if (w.heads > 0 && (w.kv_heads == 0 || w.heads % w.kv_heads != 0))
    return host::fail(MFA_ERR_INVALID_ARGUMENT,
                      "the number of query heads must be a multiple of the k / v heads");
  // blocks, units and steps are counted in 32 bits
  if (w.n > 0x7fff0000LL) return host::fail(MFA_ERR_INVALID_ARGUMENT, "N is too large");
  if (w.heads > 0 && w.batch > 0x7fffffffLL / w.heads)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "B * H is too large");
  const int64_t blocks = (w.n + 127) / 128;
  if (static_cast<double>(blocks) * static_cast<double>(w.batch * w.heads) > 0x3fff0000)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "B * H * N is too large");
  // beyond the sequence both mean the same
  if (w.window >= w.n) {
    w.window = w.n > 0 ? w.n : 1;
    w.sinks = 0;
  }
  if (w.sinks > w.n) w.sinks = w.n;
  if (w.rest_rows < 0 || w.rest_rows > w.n)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "rest_rows must be within [0, N]");
  return MFA_OK;
}

template <class Cfg>
int launch_forward(const void* q, const void* k, const void* v, void* out, float* lse,
                   void* rest, const Problem& w, const host::Device& dev, cudaStream_t stream) {
  FwdParams p = {};
  const bool bf16 = Cfg::kBF16;
  const host::Strides st = host::strides_of(w.layout, w.heads, w.n, w.d);
  int rc = host::encode_heads(&p.tm_q, q, w.batch, w.heads, w.n, w.d, w.q, bf16);
  if (rc == MFA_OK) rc = host::encode_heads(&p.tm_k, k, w.batch, w.kv_heads, w.n, w.d, w.k, bf16);
  if (rc == MFA_OK) rc = host::encode_heads(&p.tm_v, v, w.batch, w.kv_heads, w.n, w.d, w.v, bf16);
  if (rc == MFA_OK)
    rc = host::encode_heads(&p.tm_o, out, w.batch, w.heads, w.n, w.d, st, bf16);
  if (rc != MFA_OK) return rc;
  p.n = p.nq = static_cast<int>(w.n);
  p.heads = static_cast<int>(w.heads);
  p.sc = make_schedule(w.batch * w.heads, w.n, w.n, Cfg::kRowsPerUnit, Cfg::kKeys, true);
  p.scale_log2 = w.scale * 1.4426950408889634f;
  p.timeout_ns = dev.timeout_ns;
  p.status = dev.status;
  p.lse = lse;
  const host::Strides rs = host::strides_of(w.layout, w.heads, w.rest_rows, w.d);
  p.rest = static_cast<uint16_t*>(rest);
  p.rest_rows = static_cast<int>(w.rest_rows);
  p.rest_b = rs.b;
  p.rest_h = rs.h;
  p.rest_n = rs.n;
  p.window = static_cast<int>(w.window);
  p.sinks = static_cast<int>(w.sinks);
  p.sink_blocks = static_cast<int>((w.sinks + 127) / 128);
  p.kv_group = static_cast<int>(w.heads / w.kv_heads);
  // Rows of few keys in several blocks follow their maximum exactly: the weight of the key that
  // dominates a row is then 1, without a rounding that would reach the row sums of the
  // backward (dP - D is a difference, and D has the whole of it). A row that sees itself and one
  // sink: dq 1.48 times as far off as its own rounding, 1.9 times at the other threshold. It costs a
  // rescale in most steps: 33.5 us for 32.1 at 16 heads x 8192, window 32, 4 sinks. Where many keys are
  // seen it would cost 10% (window 2048: 120 us for 110) and change nothing with normal inputs; with
  // queries four times as large, dq 1.77 times its own rounding to 1.50.
  p.rescale_threshold = w.window < 64 ? 0.0f : Cfg::kRescaleThreshold;
  // Query blocks of two tiles that would fill at most half of the SMs, or of the last wave, are
  // done tile by tile.
  const int64_t units = static_cast<int64_t>(p.sc.q_blocks) * p.sc.bh, over = units % dev.sms;
  const int64_t whole = Cfg::NQ == 2 && 2 * over <= dev.sms ? units - over : units;
  const int64_t items = 2 * units - whole;
  p.whole_units = static_cast<int>(whole);
  const cudaError_t e =
      host::launch({items < dev.sms ? items : dev.sms, Cfg::kThreads, Cfg::kSmemBytes, stream},
                   window_kernel<Cfg>(), p);
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "window forward launch");
}

// How the dK/dV pass cuts its units into pieces (BwdWindowCursor). `span_steps` is the number of
// (key block, query block) pairs of one head that hold a visible (key, query) pair: every pass
// walks all of them; `passes` is what they cost together, in dQ steps (D = 64: the dK/dV step is
// about 1.05 of one; D = 128: the dV step, with two products for three, is taken as 0.85).
struct Pieces {
  int chunk_sink, pieces_sink, chunk_rest, pieces_rest;
};

Pieces plan_pieces(int64_t blocks, int64_t sink_blocks, int64_t span, int64_t span_steps,
                   int64_t kv_rows, int64_t group, int64_t sms, double passes) {
  const double share = passes * static_cast<double>(span_steps) *
                       static_cast<double>(kv_rows * group) / static_cast<double>(sms);
  // A unit of `len` steps stays whole while it is not the longest thing a CTA does: up to
  // three quarters of a CTA's share of the work (units are claimed longest first). Longer ones
  // are cut to a third of it, but to no less than 16 steps: writing a piece's 64 KB of sums and
  // reading them back costs as much as about three steps.
  const auto cut = [&](int64_t len, int& chunk, int& pieces) {
    int64_t c = len;
    if (static_cast<double>(len) > 0.75 * share) {
      c = static_cast<int64_t>(std::ceil(share / 3));
      if (c < 16) c = 16;
      if (c > len) c = len;
    }
    pieces = static_cast<int>((len + c - 1) / c);
    chunk = static_cast<int>((len + pieces - 1) / pieces);
  };
  Pieces out;
  cut(blocks * group, out.chunk_sink, out.pieces_sink);
  cut(span * group, out.chunk_rest, out.pieces_rest);
  return out;
}

// The map of a tensor of the gradients: D = 32 runs as D = 64 with boxes that reach past its
// columns, where loads read zeros, which change no sum, and stores write nothing.
int encode_gradient(CUtensorMap* map, const void* base, int64_t batch, int64_t heads, int64_t n,
                    int64_t d, const host::Strides& st, bool bf16) {
  if (d >= 64) return host::encode_heads(map, base, batch, heads, n, d, st, bf16);
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(n),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(st.n) * 2, static_cast<uint64_t>(st.h) * 2,
                               static_cast<uint64_t>(st.b) * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  return host::encode_map(map, base, 4, dims, strides, box, bf16);
}

template <bool kBF16>
auto* prep_kernel(int32_t d) {
  return d == 32   ? &mfa_bwd_prep_kernel<kBF16, true, 32>
         : d == 64 ? &mfa_bwd_prep_kernel<kBF16, true, 64>
                   : &mfa_bwd_prep_kernel<kBF16, true, 128>;
}

// D: the kernel's head dim, at least w.d
template <bool kBF16, int D>
int launch_backward(const void* q, const void* k, const void* v, const void* out,
                    const void* dout, const float* lse, const void* rest, void* dq, void* dk,
                    void* dv, const Problem& w, const host::Device& dev, cudaStream_t stream) {
  const int64_t blocks = (w.n + 127) / 128, bh = w.batch * w.heads, bhk = w.batch * w.kv_heads;
  const int64_t group = w.heads / w.kv_heads, sb = (w.sinks + 127) / 128;
  // (key block, query block) pairs of one head: `reach` later query blocks see a key block
  // that holds no sinks, all later ones one that does
  const int64_t reach = (126 + w.window) >> 7;
  const int64_t span = reach + 1 < blocks ? reach + 1 : blocks;
  const int64_t others = blocks - sb, short_ones = reach < others ? reach : others;
  const int64_t span_steps = sb * blocks - sb * (sb - 1) / 2 + (others - short_ones) * span +
                             short_ones * (short_ones + 1) / 2;
  const Pieces pc = plan_pieces(blocks, sb, span, span_steps, bhk, group, dev.sms,
                                D == 64 ? 2.05 : 2.85);
  const int64_t sink_units = bhk * sb * pc.pieces_sink;
  const int64_t kv_units = sink_units + bhk * others * pc.pieces_rest, q_units = bh * blocks;
  if (kv_units > 0x3fff0000LL || blocks * group > 0x3fff0000LL)
    return host::fail(MFA_ERR_INVALID_ARGUMENT, "B * H * N is too large");
  const int64_t slots = pc.pieces_rest > 1 ? kv_units : pc.pieces_sink > 1 ? sink_units : 0;

  // L2 and D of every row, the counters, the pieces' sums (256-byte aligned): at D = 64 a slot
  // holds dK and dV, at D = 128 all slots of dK come first
  constexpr int64_t kTile = 128 * D;
  const size_t rows = static_cast<size_t>(q_units) * 128;
  const size_t floats = 2 * rows + 64 + static_cast<size_t>(slots * 2 * kTile);
  float* ws = nullptr;
  cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&ws), floats * sizeof(float),
                                          dev.pool, stream);
  if (e != cudaSuccess) return host::fail_cuda(e, "cudaMallocFromPoolAsync (backward workspace)");
  float* lse2 = ws;
  float* di = ws + rows;
  int* counters = reinterpret_cast<int*>(ws + 2 * rows);
  float* sums = ws + 2 * rows + 64;

  BwdParams pkv = {};
  pkv.n = static_cast<int>(w.n);
  pkv.blocks = static_cast<int>(blocks);
  pkv.scale = w.scale;
  pkv.scale_log2 = w.scale * 1.4426950408889634f;
  pkv.lse2 = lse2;
  pkv.di = di;
  pkv.timeout_ns = dev.timeout_ns;
  pkv.status = dev.status;
  pkv.window = static_cast<int>(w.window);
  pkv.sinks = static_cast<int>(w.sinks);
  pkv.sink_blocks = static_cast<int>(sb);
  pkv.group = static_cast<int>(group);
  pkv.chunk_sink = pc.chunk_sink;
  pkv.pieces_sink = pc.pieces_sink;
  pkv.chunk_rest = pc.chunk_rest;
  pkv.pieces_rest = pc.pieces_rest;
  pkv.partials = sums;
  BwdParams pq = pkv;
  pkv.heads = static_cast<int>(w.kv_heads);
  pkv.bh = static_cast<int>(bhk);
  pkv.units = static_cast<int>(kv_units);
  pkv.claimed = counters;
  pq.heads = static_cast<int>(w.heads);
  pq.bh = static_cast<int>(bh);
  pq.units = static_cast<int>(q_units);
  pq.claimed = counters + 1;

  struct Map {
    CUtensorMap* to;
    const void* base;
    int64_t heads;
    const host::Strides& strides;
  };
  const host::Strides st = host::strides_of(w.layout, w.heads, w.n, w.d);  // out, dout, dq
  const host::Strides kv = host::strides_of(w.layout, w.kv_heads, w.n, w.d);  // dk, dv
  // dQ: q, dO resident; k, v streamed. dK, dV: k, v resident; q, dO streamed.
  const Map maps[] = {{&pq.tm_x, q, w.heads, w.q},      {&pq.tm_y, dout, w.heads, st},
                      {&pq.tm_s0, k, w.kv_heads, w.k},  {&pq.tm_s1, v, w.kv_heads, w.v},
                      {&pq.tm_o0, dq, w.heads, st},     {&pkv.tm_o0, dk, w.kv_heads, kv},
                      {&pkv.tm_o1, dv, w.kv_heads, kv}};
  int rc = MFA_OK;
  for (const Map& m : maps) {
    rc = encode_gradient(m.to, m.base, w.batch, m.heads, w.n, w.d, m.strides, kBF16);
    if (rc != MFA_OK) break;
  }
  pq.tm_o1 = pq.tm_o0;
  pkv.tm_x = pq.tm_s0;
  pkv.tm_y = pq.tm_s1;
  pkv.tm_s0 = pq.tm_x;
  pkv.tm_s1 = pq.tm_y;
  if (rc == MFA_OK) {
    const int64_t need = static_cast<int64_t>(rows) * w.d / 2048;  // 16 bytes a thread
    const int64_t most = static_cast<int64_t>(dev.sms) * 16;
    const host::Strides rs = host::strides_of(w.layout, w.heads, w.rest_rows, w.d);
    // the kernels wait for the stream's earlier work themselves and may be set up while it ends
    e = host::launch({need < most ? need : most, 256, 0, stream}, prep_kernel<kBF16>(w.d), out,
                     dout, lse, lse2, di, static_cast<int>(bh), static_cast<int>(w.n),
                     static_cast<int>(w.heads), static_cast<long long>(st.b),
                     static_cast<long long>(st.h), static_cast<long long>(st.n),
                     static_cast<int>(blocks), counters, rest,
                     static_cast<int>(rest ? w.rest_rows : 0), static_cast<long long>(rs.b),
                     static_cast<long long>(rs.h), static_cast<long long>(rs.n));
    const int64_t units = kv_units > q_units ? kv_units : q_units;
    const int64_t ctas = units < dev.sms ? units : dev.sms;
    if constexpr (D == 64) {
      if (e == cudaSuccess)
        e = host::launch({ctas, BwdConfig<true, true, kBF16, true>::kThreads,
                          window_bwd_smem<kBF16>(), stream},
                         &mfa_bwd_window_kernel<kBF16>, pq, pkv);
    } else {
      auto set_grad = [](BwdParams& to, void* grad, const host::Strides& g) {
        to.grad = static_cast<uint16_t*>(grad);
        to.grad_b = g.b;
        to.grad_h = g.h;
        to.grad_n = g.n;
      };
      set_grad(pq, dq, st);
      BwdParams pv = pkv;  // pkv: dK
      set_grad(pkv, dk, kv);
      set_grad(pv, dv, kv);
      pv.claimed = counters + 2;
      pv.partials = sums + slots * kTile;
      if (e == cudaSuccess)
        e = host::launch({ctas, BwdDQ128<kBF16>::kThreads, window_bwd128_smem<kBF16>(), stream},
                         &mfa_bwd_window128_kernel<kBF16>, pq, pkv, pv);
    }
    if (e == cudaSuccess && slots > 0) {
      const int64_t pairs = bhk * (pc.pieces_rest > 1 ? blocks : sb);
      const long long slot_floats = D == 64 ? 2 * kTile : kTile;
      e = host::launch({pairs * D / 8, 256, 0, stream}, &mfa_bwd_reduce_kernel<kBF16, D>, pkv, sums,
                       sums + (D == 64 ? kTile : slots * kTile), slot_floats, w.d,
                       static_cast<uint16_t*>(dk), static_cast<uint16_t*>(dv),
                       static_cast<long long>(kv.b), static_cast<long long>(kv.h),
                       static_cast<long long>(kv.n));
    }
  }
  const cudaError_t ef = cudaFreeAsync(ws, stream);
  if (rc != MFA_OK) return rc;
  if (e == cudaSuccess) e = ef;
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "window backward launch");
}

template <bool kBF16>
int forward_d(const void* q, const void* k, const void* v, void* out, float* lse, void* rest,
              const Problem& w, const host::Device& dev, cudaStream_t s) {
  if (w.d == 32) return launch_forward<Window<kBF16, 32>>(q, k, v, out, lse, rest, w, dev, s);
  if (w.d == 64) return launch_forward<Window<kBF16, 64>>(q, k, v, out, lse, rest, w, dev, s);
  return launch_forward<Window<kBF16, 128>>(q, k, v, out, lse, rest, w, dev, s);
}

int forward(const void* q, const void* k, const void* v, void* out, float* lse, void* rest,
            Problem& w, const int64_t* strides, void* stream) {
  int rc = check(w);
  if (rc != MFA_OK || w.batch * w.heads == 0 || w.n == 0) return rc;
  if (w.rest_rows == 0) rest = nullptr;
  if ((rc = set_strides(w, strides)) != MFA_OK) return rc;
  host::Pointer ptrs[6] = {{q, "q", 16}, {k, "k", 16}, {v, "v", 16}, {out, "out", 16}};
  int count = 4;
  if (rest) ptrs[count++] = {rest, "out_rest", 16};
  if (lse) ptrs[count++] = {lse, "lse", 4};
  if ((rc = host::check_pointers(ptrs, count, -1)) != MFA_OK) return rc;
  host::Device dev;
  if ((rc = host::open_device(&dev)) != MFA_OK || (rc = prepare(dev.index)) != MFA_OK) return rc;
  if ((rc = host::check_pointers(ptrs, count, dev.index)) != MFA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w.dtype == MFA_DTYPE_BF16 ? forward_d<true>(q, k, v, out, lse, rest, w, dev, s)
                                   : forward_d<false>(q, k, v, out, lse, rest, w, dev, s);
}

int backward(const void* q, const void* k, const void* v, const void* out, const void* dout,
             const float* lse, const void* rest, void* dq, void* dk, void* dv, Problem& w,
             const int64_t* strides, void* stream) {
  int rc = check(w);
  if (rc != MFA_OK || w.batch * w.heads == 0 || w.n == 0) return rc;
  if (w.rest_rows == 0) rest = nullptr;
  if ((rc = set_strides(w, strides)) != MFA_OK) return rc;
  const host::Pointer ptrs[] = {{q, "q", 16}, {k, "k", 16}, {v, "v", 16},
                                {out, "out", 16}, {dout, "dout", 16}, {lse, "lse", 4},
                                {dq, "dq", 16}, {dk, "dk", 16}, {dv, "dv", 16},
                                {rest, "out_rest", 16}};
  const int count = rest ? 10 : 9;
  if ((rc = host::check_pointers(ptrs, count, -1)) != MFA_OK) return rc;
  host::Device dev;
  if ((rc = host::open_device(&dev)) != MFA_OK || (rc = prepare(dev.index)) != MFA_OK) return rc;
  if ((rc = host::check_pointers(ptrs, count, dev.index)) != MFA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w.dtype == MFA_DTYPE_BF16)
    return w.d <= 64
               ? launch_backward<true, 64>(q, k, v, out, dout, lse, rest, dq, dk, dv, w, dev, s)
               : launch_backward<true, 128>(q, k, v, out, dout, lse, rest, dq, dk, dv, w, dev, s);
  return w.d <= 64
             ? launch_backward<false, 64>(q, k, v, out, dout, lse, rest, dq, dk, dv, w, dev, s)
             : launch_backward<false, 128>(q, k, v, out, dout, lse, rest, dq, dk, dv, w, dev, s);
}

}  // namespace
}  // namespace mfa

using namespace mfa;

extern "C" int mfa_fwd_window(const void* q, const void* k, const void* v, void* out, float* lse,
                              void* rest, int64_t batch, int64_t heads, int64_t kv_heads, int64_t n,
                              int32_t d, int64_t window, int64_t sinks, float scale,
                              int32_t dtype, int32_t layout, const int64_t* strides, void* stream) {
  return mfa_fwd_window_rest(q, k, v, out, lse, rest, n > 0 ? n : 0, batch, heads, kv_heads, n, d,
                             window, sinks, scale, dtype, layout, strides, stream);
}

extern "C" int mfa_fwd_window_rest(const void* q, const void* k, const void* v, void* out,
                                   float* lse, void* rest, int64_t rest_rows, int64_t batch,
                                   int64_t heads, int64_t kv_heads, int64_t n, int32_t d,
                                   int64_t window, int64_t sinks, float scale, int32_t dtype,
                                   int32_t layout, const int64_t* strides, void* stream) {
  Problem w{batch, heads, kv_heads, n, window, sinks, d, dtype, layout, scale, rest_rows, {}, {}, {}};
  return forward(q, k, v, out, lse, rest, w, strides, stream);
}

extern "C" int mfa_bwd_window(const void* q, const void* k, const void* v, const void* out,
                              const void* dout, const float* lse, const void* rest, void* dq,
                              void* dk, void* dv, int64_t batch, int64_t heads,
                              int64_t kv_heads, int64_t n, int32_t d, int64_t window,
                              int64_t sinks, float scale, int32_t dtype, int32_t layout,
                              const int64_t* strides, void* stream) {
  return mfa_bwd_window_rest(q, k, v, out, dout, lse, rest, n > 0 ? n : 0, dq, dk, dv, batch, heads,
                             kv_heads, n, d, window, sinks, scale, dtype, layout, strides, stream);
}

extern "C" int mfa_bwd_window_rest(const void* q, const void* k, const void* v, const void* out,
                                   const void* dout, const float* lse, const void* rest,
                                   int64_t rest_rows, void* dq, void* dk, void* dv, int64_t batch,
                                   int64_t heads, int64_t kv_heads, int64_t n, int32_t d,
                                   int64_t window, int64_t sinks, float scale, int32_t dtype,
                                   int32_t layout, const int64_t* strides, void* stream) {
  Problem w{batch, heads, kv_heads, n, window, sinks, d, dtype, layout, scale, rest_rows, {}, {}, {}};
  return backward(q, k, v, out, dout, lse, rest, dq, dk, dv, w, strides, stream);
}
