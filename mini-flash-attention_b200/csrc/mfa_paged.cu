// C-ABI launchers of the paged key / value cache: its extension (block tables, slots, the copy of
// k and v) and the attention of single tokens over it, alone or behind a shared prefix.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/mfa_b200.h"
#include "mfa_cache_kernel.cuh"
#include "mfa_fwd_kernel.cuh"
#include "mfa_host.h"
#include "mfa_paged_kernel.cuh"

namespace mfa {
namespace {

constexpr int64_t kMost = 0x7fffff00LL;  // 32-bit counters with room for a tile

// The prefix variant of the forward kernel. D = 64 has two query tiles a CTA as the forward does,
// or, when all rows fit one, one tile and a deeper ring (a prefix read for so few rows is bound
// by HBM: 5 stages are 160 KB in flight on an SM); D = 128 one tile, as the forward, and three
// stages of 64 KB.
template <bool kBF16, int D, int NQ>
using Prefix = FwdConfig<NQ, D == 64 && NQ == 1 ? 5 : 3, false, kBF16, D, false, false, true>;

template <class Cfg>
auto* prefix_kernel() {
  return &mfa_fwd_kernel<Cfg::NQ, Cfg::STAGES, false, Cfg::kBF16, Cfg::kHeadDim, false, false, true>;
}

template <class Cfg>
cudaError_t set_prefix() {
  return cudaFuncSetAttribute(prefix_kernel<Cfg>(), cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Cfg::kSmemBytes);
}

template <int D, bool kBF16>
cudaError_t set_paged() {
  constexpr int kSmem = PagedConfig<D, kBF16>::kSmemBytes;
  constexpr auto kAttr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(mfa_paged_kernel<D, kBF16>, kAttr, kSmem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(mfa_paged_cluster_kernel<D, kBF16>, kAttr, kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(mfa_paged_cluster_kernel<D, kBF16>,
                             cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <bool kBF16>
cudaError_t set_attributes() {
  cudaError_t e = set_paged<64, kBF16>();
  if (e == cudaSuccess) e = set_paged<128, kBF16>();
  if (e == cudaSuccess) e = set_prefix<Prefix<kBF16, 64, 1>>();
  if (e == cudaSuccess) e = set_prefix<Prefix<kBF16, 64, 2>>();
  if (e == cudaSuccess) e = set_prefix<Prefix<kBF16, 128, 1>>();
  return e;
}

int prepare(int dev) {
  static host::SetUp set_up[host::kMaxDevices];
  return set_up[dev]([]() -> int {
    cudaError_t e = set_attributes<false>();
    if (e == cudaSuccess) e = set_attributes<true>();
    return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "paged kernel set-up");
  });
}

int invalid(const std::string& msg) { return host::fail(MFA_ERR_INVALID_ARGUMENT, msg); }

using host::Pointer;
template <int kCount>
int check_pointers(const Pointer (&ptrs)[kCount], int dev) {
  return host::check_pointers(ptrs, kCount, dev);
}

constexpr int64_t kInlinePrefixBytes = 64 << 20;

// The arguments of the two attentions.
struct Problem {
  int64_t batch, heads, kv_heads;
  int32_t d;
  int64_t q_request, q_head;  // element strides of q
  int64_t pages, page_size, columns, window, sinks;
  int64_t prefix;  // tokens of the shared prefix
  float scale;
  int32_t dtype;

  int64_t group() const { return heads / kv_heads; }
  int kernel_d() const { return d == 128 ? 128 : 64; }  // see PagedConfig
  int64_t row_tiles() const { return (group() + 15) / 16; }
  int64_t units() const { return batch * kv_heads * row_tiles(); }
  int64_t slot_rows() const { return group() < 16 ? group() : 16; }
  int shift() const {
    int s = 0;
    while ((int64_t{1} << s) < page_size) ++s;
    return s;
  }
  // requests of a 128-row query tile of the prefix, tiles of a k / v head
  int64_t tile_batch() const { return 128 / group(); }
  int64_t tiles() const { return (batch + tile_batch() - 1) / tile_batch(); }
  int tiles_a_unit() const { return d == 128 || tiles() == 1 ? 1 : 2; }
  // A prefix that costs less to read for every request (from L2) than its own kernel and the
  // joining of its pieces: it becomes the first tiles of each request. (Of 64 requests, 8 heads of
  // 128: 67 MB 16.7 us either way, 134 MB 21.6 us inline and 17.2 apart; of 4 requests, 66 MB 13.3
  // and 16.3, 16 MB 7.8 and 10.5; of 200 requests, 2 heads of 64: 52 MB 12.9 and 14.7, 102 MB 17.7
  // and 15.7.)
  bool prefix_inline() const {
    return static_cast<double>(batch) * static_cast<double>(prefix) *
               static_cast<double>(kv_heads * row_tiles() * d * 4) <= kInlinePrefixBytes;
  }
  bool prefix_apart() const { return prefix > 0 && !prefix_inline(); }
  int64_t prefix_tiles() const { return prefix_apart() ? 0 : (prefix + 63) / 64; }
  // Tiles of the longest request.
  int64_t most_tiles() const {
    const int64_t t = (columns * page_size + 63) / 64 + prefix_tiles();
    return t > 0 ? t : 1;
  }
};

int check(Problem& w) {
  if (w.batch < 0 || w.heads < 0 || w.kv_heads < 0 || w.pages < 0 || w.columns < 0 || w.prefix < 0)
    return invalid("negative extent");
  if (w.d != 32 && w.d != 64 && w.d != 128)
    return host::fail(MFA_ERR_HEAD_DIM, "This kernel supports only D=32, D=64 and D=128");
  if (w.dtype != MFA_DTYPE_FP16 && w.dtype != MFA_DTYPE_BF16)
    return invalid("dtype must be MFA_DTYPE_FP16 or MFA_DTYPE_BF16");
  if (!(w.scale > 0.0f) || !std::isfinite(w.scale))
    return invalid("scale must be positive and finite");
  if (w.page_size < 16 || w.page_size > 256 || (w.page_size & (w.page_size - 1)))
    return invalid("the page size must be 16, 32, 64, 128 or 256 tokens");
  if (w.window < 0) return invalid("window must not be negative");
  if (w.sinks < 0) return invalid("sinks must not be negative");
  if (w.heads > 0 && (w.kv_heads == 0 || w.heads % w.kv_heads != 0))
    return invalid("the number of query heads must be a multiple of the k / v heads");
  if (w.heads > 0 && w.group() > 128) return invalid("at most 128 query heads may share a k / v head");
  if (w.heads > 0x7fffffffLL || (w.heads > 0 && w.batch > 0x7fffffffLL / w.heads))
    return invalid("B * H is too large");
  if (w.pages > 0x7fffffffLL / w.page_size) return invalid("the cache has too many tokens");
  if (w.columns > kMost / w.page_size) return invalid("the block table has too many columns");
  if (w.prefix > kMost) return invalid("the prefix is too long");
  if (w.heads == 0 || w.batch == 0) return MFA_OK;
  // a dimension of one element may have any stride
  if (w.heads == 1) w.q_head = w.d;
  if (w.batch == 1) w.q_request = w.d;
  for (const int64_t s : {w.q_request, w.q_head})
    if (s <= 0 || s % 8 != 0 || s >= int64_t{1} << 31)
      return invalid("the strides of q must be positive multiples of 8 elements below 2^31");
  // steps of a launch are counted in 32 bits
  const double tiles = static_cast<double>(w.most_tiles() + kPagedUnitSteps);
  if (tiles * static_cast<double>(w.units()) > 0x7fffff00 ||
      static_cast<double>(w.prefix / 128 + 1) * static_cast<double>(w.kv_heads * w.tiles()) >
          0x7fffff00)
    return invalid("batch * heads * tokens is too large");
  const int64_t most = w.columns * w.page_size;
  if (w.window >= most) w.window = 0;  // the same
  if (w.window == 0) w.sinks = 0;
  if (w.sinks > most) w.sinks = most;
  return MFA_OK;
}

// Parts of the workspace, in floats from its start (256-byte aligned parts).
struct Layout {
  int cluster;          // CTAs a unit of the cluster kernel; 0: the paged and combine kernels
  int64_t ctas;         // of the paged kernel
  int64_t prefix_ctas, splits;  // of the prefix kernel
  int64_t slots, prefix_slots, pieces, bytes;
};

Layout lay_out(const Problem& w, int64_t sms) {
  const auto whole = [](int64_t floats) { return (floats + 63) / 64 * 64; };
  Layout l = {};
  const int64_t full =
      sms * (w.kernel_d() == 64 ? PagedConfig<64, false>::kCtas : PagedConfig<128, false>::kCtas);
  const int64_t most = w.most_tiles();
  if (!w.prefix_apart() && w.units() <= full) {
    // CTAs a unit: as many as can be resident, up to 16, but two tiles each at least (at 16 tiles
    // 8 CTAs measured 5.7 us and 16 6.0, at 2 tiles one 4.6 and two 4.9); if one would have
    // more than eight tiles, the work is better cut evenly (see the cluster kernel).
    int size = 1;
    while (size < 16 && w.units() * size * 2 <= full && size * 4 <= most) size *= 2;
    if (most <= 8 * size) {
      l.cluster = size;
      l.ctas = w.units() * size;
      return l;
    }
  }
  // All that are resident at once, but no more than there can be steps.
  const int64_t steps = w.units() * (most + kPagedUnitSteps);
  l.ctas = steps < full ? steps : full;
  const bool shared = w.prefix_apart();
  const int64_t slots = shared ? l.ctas + w.units() : 2 * l.ctas;
  const int64_t entries = shared ? w.units() : l.ctas;
  l.slots = 0;
  l.pieces = whole(slots * paged_slot_floats(static_cast<int>(w.slot_rows()), w.kernel_d()));
  l.prefix_slots = l.pieces + whole(entries * static_cast<int64_t>(sizeof(PagedPieces)) / 4);
  int64_t end = l.prefix_slots;
  if (shared) {
    const int nq = w.tiles_a_unit();
    const int64_t units = (w.tiles() + nq - 1) / nq * w.kv_heads;
    const int64_t blocks = (w.prefix + 127) / 128;
    // As many ranges a unit as finish first: waves of items times their steps, each with about
    // two steps' time more for its queries, first scores and result; and every range is one
    // more piece for the combine kernel to read.
    double best = 1e300;
    for (int64_t s = 1; s <= blocks && (s == 1 || s * units <= 3 * sms); ++s) {
      const int64_t waves = (units * s + sms - 1) / sms;
      const double cost = static_cast<double>(waves * ((blocks + s - 1) / s + 2)) + 0.1 * s;
      if (cost < best) {
        best = cost;
        l.splits = s;
      }
    }
    l.prefix_ctas = units * l.splits < sms ? units * l.splits : sms;
    end += units * l.splits * (128 * nq * (w.kernel_d() + 2));
  }
  l.bytes = end * 4;
  return l;
}

int encode_cache(CUtensorMap* map, const void* base, const Problem& w, int64_t most_rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(w.d), static_cast<uint64_t>(w.page_size),
                            static_cast<uint64_t>(w.kv_heads), static_cast<uint64_t>(w.pages)};
  const uint64_t row = static_cast<uint64_t>(w.d) * 2;
  const uint64_t strides[3] = {row, row * dims[1], row * dims[1] * dims[2]};
  const uint32_t box[4] = {64, static_cast<uint32_t>(w.page_size < most_rows ? w.page_size : most_rows),
                           1, 1};
  return host::encode_map(map, base, 4, dims, strides, box, w.dtype == MFA_DTYPE_BF16);
}

struct Arrays {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int* prefix_pages;
  const int* block_table;
  const int* lengths;
  void* out;
  float* workspace;
};

template <class Cfg>
int launch_prefix(const Arrays& x, const Problem& w, const Layout& l, const host::Device& dev,
                  cudaStream_t stream, PrefixPieces* pp) {
  FwdParams p = {};
  const uint64_t dims[4] = {static_cast<uint64_t>(w.d), static_cast<uint64_t>(w.group()),
                            static_cast<uint64_t>(w.batch), static_cast<uint64_t>(w.kv_heads)};
  const uint64_t row = static_cast<uint64_t>(w.q_head) * 2;
  const uint64_t strides[3] = {row, static_cast<uint64_t>(w.q_request) * 2, row * dims[1]};
  const uint32_t box[4] = {64, static_cast<uint32_t>(w.group()),
                           static_cast<uint32_t>(w.tile_batch()), 1};
  int rc = host::encode_map(&p.tm_q, x.q, 4, dims, strides, box, Cfg::kBF16);
  if (rc == MFA_OK) rc = encode_cache(&p.tm_k, x.k_cache, w, 128);
  if (rc == MFA_OK) rc = encode_cache(&p.tm_v, x.v_cache, w, 128);
  if (rc != MFA_OK) return rc;
  p.n = static_cast<int>(w.prefix);
  p.heads = static_cast<int>(w.kv_heads);
  p.sc = make_schedule(w.kv_heads, w.tiles() * 128, w.prefix, Cfg::kRowsPerUnit, Cfg::kKeys, false);
  p.splits = static_cast<int>(l.splits);
  p.scale_log2 = w.scale * 1.4426950408889634f;
  p.timeout_ns = dev.timeout_ns;
  p.status = dev.status;
  p.workspace = x.workspace + l.prefix_slots;
  p.tile_batch = static_cast<int>(w.tile_batch());
  p.tile_rows = static_cast<int>(w.tile_batch() * w.group());
  p.prefix_pages = x.prefix_pages;
  p.page_shift = w.shift();
  p.pages = static_cast<int>(w.pages);
  *pp = {p.workspace, p.splits, p.sc.q_blocks, Cfg::kRowsPerUnit, p.tile_batch};
  const cudaError_t e = host::launch({l.prefix_ctas, Cfg::kThreads, Cfg::kSmemBytes, stream},
                                     prefix_kernel<Cfg>(), p);
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "prefix attention launch");
}

template <int D, bool kBF16>
int launch_paged(const Arrays& x, const Problem& w, const host::Device& dev, cudaStream_t stream) {
  using Cfg = PagedConfig<D, kBF16>;
  const Layout l = lay_out(w, dev.sms);
  const bool shared = w.prefix_apart();
  CombineParams cp = {};
  int rc = MFA_OK;
  if (shared) {
    if (w.tiles_a_unit() == 2)
      rc = launch_prefix<Prefix<kBF16, 64, 2>>(x, w, l, dev, stream, &cp.prefix);
    else
      rc = launch_prefix<Prefix<kBF16, D, 1>>(x, w, l, dev, stream, &cp.prefix);
    if (rc != MFA_OK) return rc;
  }
  PagedParams p = {};
  if ((rc = encode_cache(&p.tm_k, x.k_cache, w, 64)) != MFA_OK ||
      (rc = encode_cache(&p.tm_v, x.v_cache, w, 64)) != MFA_OK)
    return rc;
  p.q = static_cast<const uint16_t*>(x.q);
  p.q_request = w.q_request;
  p.q_head = w.q_head;
  p.cols = w.d;
  p.out = static_cast<uint16_t*>(x.out);
  p.block_table = x.block_table;
  p.lengths = x.lengths;
  p.batch = static_cast<int>(w.batch);
  p.kv_heads = static_cast<int>(w.kv_heads);
  p.group = static_cast<int>(w.group());
  p.row_tiles = static_cast<int>(w.row_tiles());
  p.columns = static_cast<int>(w.columns);
  p.page_shift = w.shift();
  p.pages = static_cast<int>(w.pages);
  p.window = static_cast<int>(w.window);
  p.sinks = static_cast<int>(w.sinks);
  p.pieces_only = shared ? 1 : 0;
  p.prefix_pages = x.prefix_pages;
  p.prefix = static_cast<int>(shared ? 0 : w.prefix);
  p.prefix_tiles = static_cast<int>(w.prefix_tiles());
  p.scale_log2 = w.scale * 1.4426950408889634f;
  p.slots = x.workspace + l.slots;
  p.pieces = reinterpret_cast<PagedPieces*>(x.workspace + l.pieces);
  p.timeout_ns = dev.timeout_ns;
  p.status = dev.status;
  if (l.cluster > 0) {
    const cudaError_t ec =
        host::launch({l.ctas, Cfg::kThreads, Cfg::kSmemBytes, stream, l.cluster},
                     &mfa_paged_cluster_kernel<D, kBF16>, p);
    return ec == cudaSuccess ? MFA_OK : host::fail_cuda(ec, "paged attention launch");
  }
  cudaError_t e = host::launch({l.ctas, Cfg::kThreads, Cfg::kSmemBytes, stream},
                               &mfa_paged_kernel<D, kBF16>, p);
  if (e != cudaSuccess) return host::fail_cuda(e, "paged attention launch");
  cp.pieces = p.pieces;
  cp.slots = p.slots;
  cp.out = p.out;
  cp.kv_heads = p.kv_heads;
  cp.group = p.group;
  cp.row_tiles = p.row_tiles;
  cp.cols = p.cols;
  cp.pieces_only = p.pieces_only;
  e = shared ? host::launch({w.units(), 128, 0, stream},
                            &mfa_paged_combine_kernel<D, kBF16, true>, cp)
             : host::launch({l.ctas, 128, 0, stream}, &mfa_paged_combine_kernel<D, kBF16, false>, cp);
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "paged combine launch");
}

int attend(const Arrays& x, uint64_t workspace_bytes, Problem& w, void* stream) {
  int rc = check(w);
  if (rc != MFA_OK || w.batch == 0 || w.heads == 0) return rc;
  // a call without own tokens may have no table, one without a prefix no prefix pages: a valid
  // pointer stands in, which nothing reads
  Arrays a = x;
  if (w.columns == 0) a.block_table = a.lengths;
  if (w.prefix == 0) a.prefix_pages = a.lengths;
  const Pointer ptrs[] = {{a.q, "q", 16},
                          {a.k_cache, "k_cache", 16},
                          {a.v_cache, "v_cache", 16},
                          {a.prefix_pages, "prefix_pages", 4},
                          {a.block_table, "block_table", 4},
                          {a.lengths, "lengths", 4},
                          {a.out, "out", 16}};
  const Pointer work[] = {{a.workspace, "workspace", 256}};
  if ((rc = check_pointers(ptrs, -1)) != MFA_OK) return rc;
  if (w.pages == 0) return invalid("the cache has no pages");
  host::Device dev;
  if ((rc = host::open_device(&dev)) != MFA_OK || (rc = prepare(dev.index)) != MFA_OK) return rc;
  if ((rc = check_pointers(ptrs, dev.index)) != MFA_OK) return rc;
  const int64_t need = lay_out(w, dev.sms).bytes;
  if (workspace_bytes < static_cast<uint64_t>(need))
    return invalid("the workspace must have " + std::to_string(need) + " bytes");
  if (need > 0 && ((rc = check_pointers(work, -1)) != MFA_OK ||
                   (rc = check_pointers(work, dev.index)) != MFA_OK))
    return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = w.dtype == MFA_DTYPE_BF16;
  if (w.kernel_d() == 64)
    return bf16 ? launch_paged<64, true>(a, w, dev, s) : launch_paged<64, false>(a, w, dev, s);
  return bf16 ? launch_paged<128, true>(a, w, dev, s) : launch_paged<128, false>(a, w, dev, s);
}

}  // namespace
}  // namespace mfa

using namespace mfa;

extern "C" int mfa_extend_block_tables(int32_t* block_table, const int32_t* cached,
                                       const int32_t* added, const int32_t* free_pages,
                                       int32_t* slots, int32_t* starts, int32_t* used,
                                       int64_t batch, int64_t columns, int64_t free_count,
                                       int64_t page_size, int64_t capacity, void* stream) {
  if (batch < 0 || columns < 0 || free_count < 0 || capacity < 0) return invalid("negative extent");
  if (page_size < 1) return invalid("page_size must be positive");
  if (batch > kMost || columns > kMost || free_count > kMost || capacity > kMost ||
      page_size > kMost)
    return invalid("extents must fit in 32 bits");
  // arrays that have no elements need no pointer
  const int32_t* any = starts;
  const Pointer ptrs[] = {{batch > 0 && columns > 0 ? block_table : any, "block_table", 4},
                          {batch > 0 ? cached : any, "cached", 4},
                          {batch > 0 ? added : any, "added", 4},
                          {free_count > 0 ? free_pages : any, "free_pages", 4},
                          {capacity > 0 ? slots : any, "slots", 4},
                          {starts, "starts", 4},
                          {used, "used", 4}};
  int rc = check_pointers(ptrs, -1);
  if (rc != MFA_OK) return rc;
  host::Device dev;
  if ((rc = host::open_device(&dev)) != MFA_OK) return rc;
  if ((rc = check_pointers(ptrs, dev.index)) != MFA_OK) return rc;
  ExtendParams p = {};
  p.table = block_table;
  p.cached = cached;
  p.added = added;
  p.free_pages = free_pages;
  p.batch = static_cast<int>(batch);
  p.columns = static_cast<int>(columns);
  p.free_count = static_cast<int>(free_count);
  p.page_size = static_cast<int>(page_size);
  p.slots = slots;
  p.capacity = static_cast<int>(capacity);
  p.starts = starts;
  p.used = used;
  // a token a thread, two CTAs an SM at most (each scans all requests)
  const int64_t need = (capacity + kExtendThreads - 1) / kExtendThreads;
  const int64_t grid = need < 1 ? 1 : need < 2 * dev.sms ? need : 2 * dev.sms;
  const cudaError_t e = host::launch({grid, kExtendThreads, 0, static_cast<cudaStream_t>(stream)},
                                     &mfa_extend_kernel, p);
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "block table launch");
}

extern "C" int mfa_append_kv(const void* k, const void* v, void* k_cache, void* v_cache,
                             const int32_t* slots, int64_t tokens, int64_t kv_heads, int64_t d,
                             int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                             int64_t v_head_stride, int64_t pages, int64_t page_size,
                             void* stream) {
  if (tokens < 0 || kv_heads < 0 || d < 0 || pages < 0) return invalid("negative extent");
  if (page_size < 1) return invalid("page_size must be positive");
  if (d % 8 != 0) return invalid("D must be a multiple of 8");
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 != 0)
    return invalid("token and head strides must be multiples of 8 elements");
  if (tokens > kMost || kv_heads > 65535 || d > 65536 || kv_heads * d > (1 << 24))
    return invalid("tokens, heads or D are too large");
  if (page_size > 0x7fffffffLL || pages > 0x7fffffffLL / page_size)
    return invalid("the cache has too many tokens");
  if (tokens == 0 || kv_heads == 0 || d == 0 || pages == 0) return MFA_OK;
  const Pointer ptrs[] = {{k, "k", 16},
                          {v, "v", 16},
                          {k_cache, "k_cache", 16},
                          {v_cache, "v_cache", 16},
                          {slots, "slots", 4}};
  int rc = check_pointers(ptrs, -1);
  if (rc != MFA_OK) return rc;
  host::Device dev;
  if ((rc = host::open_device(&dev)) != MFA_OK) return rc;
  if ((rc = check_pointers(ptrs, dev.index)) != MFA_OK) return rc;
  AppendParams p = {};
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.k_cache = static_cast<uint16_t*>(k_cache);
  p.v_cache = static_cast<uint16_t*>(v_cache);
  p.slots = slots;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.tokens = static_cast<int>(tokens);
  p.kv_heads = static_cast<int>(kv_heads);
  p.d = static_cast<int>(d);
  p.page_size = static_cast<int>(page_size);
  p.slot_count = pages * page_size;
  p.by_chunks.set(d / 8);
  p.by_heads.set(kv_heads);
  p.by_page.set(page_size);
  // four 16-byte pieces of k and v a thread, fewer when that leaves SMs without a block
  const int64_t a_token = kv_heads * (d / 8);
  int64_t per = (4 * 256 + a_token - 1) / a_token;
  const int64_t spread = (tokens + 2 * dev.sms - 1) / (2 * dev.sms);
  if (per > spread) per = spread;
  p.tokens_a_block = static_cast<int>(per);
  const cudaError_t e =
      host::launch({(tokens + per - 1) / per, 256, 0, static_cast<cudaStream_t>(stream)},
                   &mfa_append_kernel, p);
  return e == cudaSuccess ? MFA_OK : host::fail_cuda(e, "append launch");
}

extern "C" int mfa_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                                   const int32_t* block_table, const int32_t* lengths, void* out,
                                   void* workspace, uint64_t workspace_bytes, int64_t batch,
                                   int64_t heads, int64_t kv_heads, int32_t d,
                                   int64_t q_batch_stride, int64_t q_head_stride, int64_t pages,
                                   int64_t page_size, int64_t columns, int64_t window,
                                   int64_t sinks, float scale, int32_t dtype, void* stream) {
  Problem w{batch, heads,     kv_heads, d,      q_batch_stride, q_head_stride,
            pages, page_size, columns,  window, sinks,          0,
            scale, dtype};
  return attend({q, k_cache, v_cache, nullptr, block_table, lengths, out,
                 static_cast<float*>(workspace)},
                workspace_bytes, w, stream);
}

extern "C" int mfa_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache,
                                           const int32_t* prefix_pages, int64_t prefix_length,
                                           const int32_t* block_table, const int32_t* lengths,
                                           void* out, void* workspace, uint64_t workspace_bytes,
                                           int64_t batch, int64_t heads, int64_t kv_heads,
                                           int32_t d, int64_t q_batch_stride,
                                           int64_t q_head_stride, int64_t pages,
                                           int64_t page_size, int64_t columns, float scale,
                                           int32_t dtype, void* stream) {
  Problem w{batch, heads,     kv_heads, d, q_batch_stride, q_head_stride,
            pages, page_size, columns,  0, 0,              prefix_length,
            scale, dtype};
  return attend({q, k_cache, v_cache, prefix_pages, block_table, lengths, out,
                 static_cast<float*>(workspace)},
                workspace_bytes, w, stream);
}

extern "C" int mfa_paged_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int32_t d,
                                         int64_t page_size, int64_t columns,
                                         int64_t prefix_length, uint64_t* bytes) {
  if (!bytes) return invalid("bytes must not be null");
  *bytes = 0;
  Problem w{batch, heads,     kv_heads, d, 8, 8,
            1,     page_size, columns,  0, 0, prefix_length,
            1.0f,  MFA_DTYPE_FP16};
  const int rc = check(w);
  if (rc != MFA_OK || batch == 0 || heads == 0) return rc;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return host::fail_cuda(e, "cudaDeviceGetAttribute (multiprocessor count)");
  *bytes = static_cast<uint64_t>(lay_out(w, sms).bytes);
  return MFA_OK;
}
