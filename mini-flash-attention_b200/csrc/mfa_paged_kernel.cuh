// Attention of single query tokens over a paged key / value cache, and the kernels that extend the
// cache. A cache is [pages, kv_heads, page_size, D] (k and v apart); request b's token at position
// i lies in page block_table[b][i / page_size], row i % page_size.
//
// For the query head h of request b (k / v head h / group, n = lengths[b] tokens, the query's own
// one among them):  out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  over the visible
// positions j < n with window == 0 or j >= n - window or j < sinks; 0 where none is visible.
//
// Every visible k and v row is read once and meets `group` query rows: 4 D bytes against 4 D group
// operations, so HBM bounds it (up to 16 rows of a group at once, mma.sync m16n8k16: a padded tile
// of 16 rows takes 8192 operations a key at D = 128, a key's 512 bytes take an SM 21 cycles, and
// 390 operations a cycle are well inside what the warp-level tensor instruction gives; tcgen05
// would pad the rows to 64 or 128 and bring the scores through tensor memory for nothing).
//
// Two CTAs per SM, each of four consumer warps and one producer warp, walk a common list of steps:
// a step is one 64-key tile of one unit, a unit one (request, k / v head, 16 query rows). The
// lengths are known to the GPU only, so every CTA sums them and takes an equal share of the
// steps. Tiles arrive by TMA, one box a page, in a ring of 96 KB (two CTAs: 192 KB in flight on
// an SM). In a tile each warp takes 16 keys with a running maximum of its own; at the end of a
// unit the four warps' states meet in shared memory. What a CTA's share cuts off goes to a slot
// of the workspace as unnormalised 32-bit sums, which the combine kernel joins in CTA order.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "mfa_common.cuh"
#include "mfa_ptx.cuh"
#include "mfa_schedule.cuh"

namespace mfa {

// A piece of a unit: its first slot, and the CTAs that hold the others.
struct PagedPieces {
  int count;  // 0: nothing to combine
  int first;  // slot of the first piece
  int cta;    // CTA of the first piece; piece i > 0 is CTA cta + i's first segment
  int unit;
};

// Floats of a slot: rows x (D sums, then the maxima, then the sums of p), whole float4s.
__host__ __device__ constexpr int paged_slot_floats(int rows, int d) {
  return (rows * (d + 2) + 3) & ~3;
}

struct PagedParams {
  CUtensorMap tm_k, tm_v;  // {D, page_size, kv_heads, pages}, box {64, min(page_size, 64), 1, 1}
  const uint16_t* q;       // [batch, kv_heads * group, D]
  uint16_t* out;
  const int* block_table;  // [batch, columns]
  const int* lengths;      // [batch]
  int batch, kv_heads, group;
  int row_tiles;           // 16-row tiles of a group
  int columns;
  int page_shift;          // page_size = 1 << page_shift, 16 to 256
  int pages;
  int window, sinks;       // window 0: everything is visible
  int pieces_only;         // every unit goes to slots (its result meets that of a prefix)
  float scale_log2;
  float* slots;            // of min(group, 16) rows each
  PagedPieces* pieces;     // [CTA], or [unit] if pieces_only
  unsigned long long timeout_ns;
  int* status;
};

template <int D_, bool BF16_>
struct PagedConfig {
  static constexpr int kD = D_;
  static constexpr bool kBF16 = BF16_;
  static constexpr int kKeys = 64;  // keys of a tile
  static constexpr int kRows = 16;  // query rows of a unit
  static constexpr int kWarps = 4;
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kBoxes = kD / 64;
  static constexpr int kBoxBytes = kKeys * 128;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kStages = 98304 / (2 * kTileBytes);
  static constexpr int kMergeCols = kD + 8;  // floats a row: lanes of 4 rows hit different banks
  static constexpr int kMergeOff = kStages * 2 * kTileBytes;
  static constexpr int kStatsOff = kMergeOff + kRows * kMergeCols * 4;  // [2][kWarps][kRows]
  static constexpr int kBarOff = kStatsOff + 2 * kWarps * kRows * 4;
  static constexpr int kBarFull = 0, kBarEmpty = kStages;
  static constexpr int kScanOff = kBarOff + 2 * kStages * 8;  // warp sums, start
  static constexpr int kAbortOff = kScanOff + 4 * (kWarps + 1 + 3);
  static constexpr int kSmemBytes = kAbortOff + 4 + 1024;
};

// Tiles of a request of n tokens: those that hold sinks before the window, then the window's.
struct PagedSpan {
  int n, tiles, sinks, skip;
  __device__ void set(const PagedParams& p, int request) {
    const int most = p.columns << p.page_shift;  // < 2^31 (checked by the launcher)
    n = p.lengths[request];
    n = n < 0 ? 0 : n < most ? n : most;
    const int last = n > 0 ? (n - 1) >> 6 : 0;  // an empty request has one step, which sees nothing
    const int w0 = p.window > 0 && n > p.window ? (n - p.window) >> 6 : 0;
    const int sb = (p.sinks >> 6) + ((p.sinks & 63) != 0);
    sinks = sb < w0 ? sb : w0;
    skip = w0 - sinks;
    tiles = last + 1 - skip;
  }
  __device__ int tile(int t) const { return t < sinks ? t : t + skip; }
  __device__ bool visible(const PagedParams& p, int key) const {
    return key < n && (p.window == 0 || key >= n - p.window || key < p.sinks);
  }
};

// CTA of step s when CTA c of `ctas` has the steps [c * total / ctas, (c + 1) * total / ctas).
__device__ __forceinline__ int cta_of_step(long long s, long long total, int ctas) {
  return static_cast<int>(((s + 1) * ctas - 1) / total);
}

// Where a CTA's share of the steps starts, found by all its threads.
struct PagedShare {
  int total;    // steps of the whole call
  int ctas;     // CTAs that get a share
  int begin, end;
  int request;  // of step `begin`
  int before;   // steps of the requests before it
};

// The walk over a CTA's share, by segments (the part of one unit that it holds).
struct PagedCursor {
  PagedSpan span;
  int request, unit_row;  // unit_row: k / v head * row_tiles + row tile
  int t;                  // next tile of the unit
  int left;               // steps left in the share
  int first;              // step of the unit's first tile
  __device__ void init(const PagedParams& p, const PagedShare& sh) {
    left = sh.end - sh.begin;
    if (left <= 0) return;
    request = sh.request;
    span.set(p, request);
    const int in = sh.begin - sh.before;
    unit_row = in / span.tiles;
    t = in - unit_row * span.tiles;
    first = sh.begin - t;
  }
  __device__ int segment() const { return span.tiles - t < left ? span.tiles - t : left; }
  __device__ void advance(const PagedParams& p, int steps) {
    left -= steps;
    t += steps;
    if (t < span.tiles || left == 0) return;
    first += span.tiles;
    t = 0;
    if (++unit_row == p.kv_heads * p.row_tiles) {
      unit_row = 0;
      span.set(p, ++request);
    }
  }
};

template <class Cfg>
__device__ __forceinline__ PagedShare paged_share(const PagedParams& p, int* scan) {
  // Each thread sums the tiles of a run of requests; the block's exclusive sums tell the one
  // whose run holds the share's first step.
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + Cfg::kThreads - 1) / Cfg::kThreads;
  const int r0 = tid * per < p.batch ? tid * per : p.batch;
  const int r1 = r0 + per < p.batch ? r0 + per : p.batch;
  int mine = 0;
  PagedSpan span;
  for (int r = r0; r < r1; ++r) {
    span.set(p, r);
    mine += span.tiles;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int tiles = 0, before = upto - mine;
#pragma unroll
  for (int w = 0; w <= Cfg::kWarps; ++w) {
    const int x = scan[w];
    if (w < warp) before += x;
    tiles += x;
  }
  const int heads = p.kv_heads * p.row_tiles;
  PagedShare sh;
  sh.total = tiles * heads;
  sh.ctas = static_cast<int>(gridDim.x) < sh.total ? static_cast<int>(gridDim.x) : sh.total;
  const int c = static_cast<int>(blockIdx.x);
  sh.begin = sh.end = 0;
  if (c < sh.ctas) {
    sh.begin = static_cast<int>(static_cast<long long>(c) * sh.total / sh.ctas);
    sh.end = static_cast<int>(static_cast<long long>(c + 1) * sh.total / sh.ctas);
  }
  if (before * heads <= sh.begin && sh.begin < (before + mine) * heads) {
    int r = r0;
    for (span.set(p, r); (before + span.tiles) * heads <= sh.begin; span.set(p, r)) {
      before += span.tiles;
      ++r;
    }
    scan[Cfg::kWarps + 1] = r;
    scan[Cfg::kWarps + 2] = before * heads;
  }
  __syncthreads();
  sh.request = scan[Cfg::kWarps + 1];
  sh.before = scan[Cfg::kWarps + 2];
  return sh;
}

// Producer warp: the tiles of the share, a box for every page that holds a visible key. The page
// numbers of the next tile are read while this one waits for its stage.
template <class Cfg>
__device__ __forceinline__ void paged_load_role(const PagedParams& p, const PagedShare& sh,
                                                uint32_t smem, uint32_t bars,
                                                const Watchdog& wd) {
  const int lane = threadIdx.x & 31;
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  const int box_shift = p.page_shift < 6 ? p.page_shift : 6;  // rows of a box
  const int boxes = Cfg::kKeys >> box_shift;                  // pages of a tile (at most four)
  const uint32_t box_bytes = 128u << box_shift;
  if (lane == 0) {
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  PagedCursor cur;
  cur.init(p, sh);
  // lane i: the page of box i of a tile, or -1 if nothing in it is visible
  auto page_of = [&]() -> int {
    if (lane >= boxes) return -1;
    const int key0 = cur.span.tile(cur.t) * Cfg::kKeys + (lane << box_shift);
    const int n = cur.span.n;
    bool any = key0 < n;
    if (p.window > 0)
      any = any && (key0 + (1 << box_shift) > n - p.window || key0 < p.sinks);
    if (!any) return -1;
    const int page = p.block_table[static_cast<size_t>(cur.request) * p.columns +
                                   (key0 >> p.page_shift)];
    // an out-of-range page is out of the tensor map's range too: the copy fills zeros
    return page < 0 || page >= p.pages ? p.pages : page;
  };
  int page = cur.left > 0 ? page_of() : -1;
  int g = 0;
  while (cur.left > 0) {
    const int now = page;
    const int head = cur.unit_row / p.row_tiles;
    const int row0 = cur.span.tile(cur.t) * Cfg::kKeys & ((1 << p.page_shift) - 1);
    cur.advance(p, 1);
    if (cur.left > 0) page = page_of();
    const int st = g % Cfg::kStages;
    const uint32_t ph = static_cast<uint32_t>(g / Cfg::kStages) & 1u;
    if (!wait_warp(bar(Cfg::kBarEmpty + st), ph ^ 1u, wd, kSiteLoadKEmpty)) break;
    const uint32_t have = __ballot_sync(0xffffffffu, now >= 0);
    const bool bad = now == p.pages;
    if (bad) atomicCAS(p.status, 0, kStatusBadPage);
    if (lane == 0)
      mbar_arrive_expect_tx(bar(Cfg::kBarFull + st),
                            2 * Cfg::kBoxes * box_bytes * __popc(have));
    __syncwarp();
    const uint32_t k_dst = smem + st * 2 * Cfg::kTileBytes, v_dst = k_dst + Cfg::kTileBytes;
    for (int i = 0; i < boxes; ++i) {
      const int pg = __shfl_sync(0xffffffffu, now, i);
      if (pg < 0 || lane != 0) continue;
#pragma unroll
      for (int x = 0; x < Cfg::kBoxes; ++x) {
        const uint32_t off = x * Cfg::kBoxBytes + i * box_bytes;
        tma_load_4d(k_dst + off, &p.tm_k, bar(Cfg::kBarFull + st), 64 * x, row0, head, pg);
        tma_load_4d(v_dst + off, &p.tm_v, bar(Cfg::kBarFull + st), 64 * x, row0, head, pg);
      }
    }
    ++g;
  }
  if (*wd.abort && lane == 0) {
    // unwinding: shared memory must outlive the copies in flight
    for (int st = 0; st < Cfg::kStages; ++st) {
      int last = -1;
      for (int x = st; x < g; x += Cfg::kStages) last = x;
      if (last >= 0)
        drain_wait(bar(Cfg::kBarFull + st), static_cast<uint32_t>(last / Cfg::kStages) & 1u);
    }
  }
}

// The same keys' 8x8 blocks of 16-bit values, as they stand and transposed.
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c (16 x 8, fp32) += a (16 x 16) b (16 x 8)
template <bool kBF16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  if (kBF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Consumer warp. Fragments: lane 4 g + q holds rows g and g + 8 of the 16 query rows and, of
// every 8 keys (scores) or 8 columns (out), the two at 2 q.
template <class Cfg>
__device__ __forceinline__ void paged_consume_role(const PagedParams& p, const PagedShare& sh,
                                                   uint8_t* smem_ptr, uint32_t bars,
                                                   const Watchdog& wd) {
  constexpr int D = Cfg::kD;
  constexpr int kKSteps = D / 16;
  constexpr float kRescaleThreshold = 8.0f;  // as in the forward kernel
  const uint32_t smem = smem_addr(smem_ptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gq = lane >> 2, q = lane & 3;
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  float* merge = reinterpret_cast<float*>(smem_ptr + Cfg::kMergeOff);
  float* stat_m = reinterpret_cast<float*>(smem_ptr + Cfg::kStatsOff);
  float* stat_l = stat_m + Cfg::kWarps * Cfg::kRows;
  const int slot_rows = p.group < Cfg::kRows ? p.group : Cfg::kRows;
  const int heads = p.kv_heads * p.group;

  // ldmatrix row addresses inside a tile: this lane's key row and the 16-byte chunk, which the
  // 128-byte swizzle moves to chunk ^ (row % 8)
  const int mat = lane >> 3, mrow = lane & 7;
  const uint32_t k_row = (warp * 16 + (mat >> 1) * 8 + mrow) * 128;
  const uint32_t v_row = (warp * 16 + (mat & 1) * 8 + mrow) * 128;
  auto chunk_off = [&](int chunk) -> uint32_t {
    return (chunk >> 3) * Cfg::kBoxBytes + (((chunk & 7) ^ mrow) << 4);
  };

  PagedCursor cur;
  cur.init(p, sh);
  int g = 0;
  bool ok = true, wrote = false;
  while (cur.left > 0) {
    const int seg = cur.segment();
    const int kv_head = cur.unit_row / p.row_tiles;
    const int tile_row0 = (cur.unit_row - kv_head * p.row_tiles) * Cfg::kRows;
    const int rows = p.group - tile_row0 < Cfg::kRows ? p.group - tile_row0 : Cfg::kRows;
    const size_t q_row0 =
        static_cast<size_t>(cur.request) * heads + kv_head * p.group + tile_row0;
    uint32_t qf[kKSteps][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t* src =
          reinterpret_cast<const uint32_t*>(p.q + (q_row0 + gq + 8 * r) * D) + q;
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        qf[kk][r] = gq + 8 * r < rows ? src[8 * kk] : 0u;
        qf[kk][2 + r] = gq + 8 * r < rows ? src[8 * kk + 4] : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int i = 0; i < seg; ++i, ++g) {
      const int st = g % Cfg::kStages;
      if (ok) ok = wait_warp(bar(Cfg::kBarFull + st),
                             static_cast<uint32_t>(g / Cfg::kStages) & 1u, wd, kSiteSoftSFull);
      if (!ok) continue;  // unwinding: only the barriers below are still kept
      const uint32_t k_tile = smem + st * 2 * Cfg::kTileBytes;
      const uint32_t v_tile = k_tile + Cfg::kTileBytes;
      float s[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        uint32_t b[4];
        ldmatrix_x4(k_tile + k_row + chunk_off(2 * kk + (mat & 1)), b);
        mma_16x8x16<Cfg::kBF16>(s[0], qf[kk], b[0], b[1]);
        mma_16x8x16<Cfg::kBF16>(s[1], qf[kk], b[2], b[3]);
      }
      // Keys that are not visible, and rows of the tile that were never loaded: their scores
      // become -inf whatever they are, and their v rows 0 (0 * NaN would not be 0).
      const int key0 = cur.span.tile(cur.t + i) * Cfg::kKeys;
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // v rows 2 q, 2 q + 1 (+ 8 for the second)
      const bool edge = key0 + Cfg::kKeys > cur.span.n ||
                        (p.window > 0 && key0 < cur.span.n - p.window &&
                         key0 + Cfg::kKeys > p.sinks);
      if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + warp * 16 + 8 * h + 2 * q;
          const bool a = cur.span.visible(p, key), b = cur.span.visible(p, key + 1);
          keep[h] = (a ? 0xffffu : 0u) | (b ? 0xffff0000u : 0u);
          if (!a) s[h][0] = s[h][2] = -INFINITY;
          if (!b) s[h][1] = s[h][3] = -INFINITY;
        }
      }
      // The running maximum is raised only when a row of the warp grows past the threshold.
      const float c = p.scale_log2;
      float top[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])) * c;
      if (__any_sync(0xffffffffu, top[0] > m[0] + kRescaleThreshold ||
                                      top[1] > m[1] + kRescaleThreshold)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          const float next = fmaxf(m[r], top[r]);
          const float alpha = next == -INFINITY ? 1.0f : ex2_approx(m[r] - next);
          m[r] = next;
          l[r] *= alpha;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            o[d][2 * r] *= alpha;
            o[d][2 * r + 1] *= alpha;
          }
        }
      }
      uint32_t pf[4];  // P as the left operand: rows g, g + 8 by keys 2 q, then keys 2 q + 8
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float sub = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = ex2_approx(fmaf(s[h][2 * r], c, -sub));
          const float b = ex2_approx(fmaf(s[h][2 * r + 1], c, -sub));
          l[r] += a + b;
          pf[2 * h + r] = pack_pair<Cfg::kBF16>(a, b);
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldmatrix_x4_trans(v_tile + v_row + chunk_off(2 * d + (mat >> 1)), b);
        mma_16x8x16<Cfg::kBF16>(o[2 * d], pf, b[0] & keep[0], b[1] & keep[1]);
        mma_16x8x16<Cfg::kBF16>(o[2 * d + 1], pf, b[2] & keep[0], b[3] & keep[1]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Cfg::kBarEmpty + st));
    }

    // ---- the segment's end: the four warps' states to one, in warp 0
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (q == 0) {
        stat_m[warp * Cfg::kRows + gq + 8 * r] = m[r];
        stat_l[warp * Cfg::kRows + gq + 8 * r] = l[r];
      }
    }
    named_bar_sync(1, 32 * Cfg::kWarps);
    float m_all[2], l_all[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m_all[r] = -INFINITY;
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w)
        m_all[r] = fmaxf(m_all[r], stat_m[w * Cfg::kRows + gq + 8 * r]);
      const float sub = m_all[r] == -INFINITY ? 0.0f : m_all[r];
      l_all[r] = 0.0f;
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w)
        l_all[r] += stat_l[w * Cfg::kRows + gq + 8 * r] *
                    ex2_approx(stat_m[w * Cfg::kRows + gq + 8 * r] - sub);
      const float f = ex2_approx(m[r] - sub);
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        o[d][2 * r] *= f;
        o[d][2 * r + 1] *= f;
      }
    }
#pragma unroll
    for (int w = Cfg::kWarps - 1; w > 0; --w) {
      // warp w adds what the warps after it have left, and leaves the sum for warp w - 1
      if (warp == w) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float* at = merge + (gq + 8 * r) * Cfg::kMergeCols + 2 * q;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            float2* to = reinterpret_cast<float2*>(at + 8 * d);
            float2 x = make_float2(o[d][2 * r], o[d][2 * r + 1]);
            if (w < Cfg::kWarps - 1) {
              const float2 y = *to;
              x.x += y.x;
              x.y += y.y;
            }
            *to = x;
          }
        }
      }
      named_bar_sync(1, 32 * Cfg::kWarps);
    }
    const bool whole = cur.t == 0 && seg == cur.span.tiles;
    const bool to_slot = p.pieces_only || !whole;
    const int unit = cur.request * p.kv_heads * p.row_tiles + cur.unit_row;
    const int slot = p.pieces_only ? static_cast<int>(blockIdx.x) + unit
                                   : 2 * static_cast<int>(blockIdx.x) + (wrote ? 1 : 0);
    if (warp == 0 && ok) {
      float* to = p.slots + static_cast<size_t>(slot) * paged_slot_floats(slot_rows, D);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = gq + 8 * r;
        if (row >= rows) continue;
        const float* from = merge + row * Cfg::kMergeCols + 2 * q;
        const float inv = l_all[r] > 0.0f ? 1.0f / l_all[r] : 0.0f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          const float2 y = *reinterpret_cast<const float2*>(from + 8 * d);
          const float a = o[d][2 * r] + y.x, b = o[d][2 * r + 1] + y.y;
          if (to_slot)
            *reinterpret_cast<float2*>(to + row * D + 8 * d + 2 * q) = make_float2(a, b);
          else
            *reinterpret_cast<uint32_t*>(p.out + (q_row0 + row) * D + 8 * d + 2 * q) =
                pack_pair<Cfg::kBF16>(a * inv, b * inv);
        }
        if (to_slot && q == 0) {
          to[slot_rows * D + row] = m_all[r];
          to[slot_rows * (D + 1) + row] = l_all[r];
        }
      }
    }
    if (warp == 0 && lane == 0 && to_slot && cur.t == 0) {
      // the unit starts here: its pieces run to the CTA of its last step (said also when
      // unwinding: the combine kernel reads it in any case)
      const int last = cta_of_step(cur.first + cur.span.tiles - 1, sh.total, sh.ctas);
      PagedPieces out;
      out.count = last - static_cast<int>(blockIdx.x) + 1;
      out.first = slot;
      out.cta = static_cast<int>(blockIdx.x);
      out.unit = unit;
      p.pieces[p.pieces_only ? unit : static_cast<int>(blockIdx.x)] = out;
    }
    if (!whole) wrote = true;
    cur.advance(p, seg);
  }
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(PagedConfig<D, kBF16>::kThreads, 2)
    mfa_paged_kernel(const __grid_constant__ PagedParams p) {
  using Cfg = PagedConfig<D, kBF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t bars = smem_addr(smem + Cfg::kBarOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kAbortOff);
  // the combine kernel may be scheduled; it waits for this grid before it reads
  if (threadIdx.x == 0) grid_dependents_launch();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(bars + 8 * (Cfg::kBarFull + s), 1);
      mbar_init(bars + 8 * (Cfg::kBarEmpty + s), Cfg::kWarps);
    }
    mbar_init_fence();
  }
  grid_dependency_wait();  // nothing above touches global memory
  const PagedShare sh = paged_share<Cfg>(p, reinterpret_cast<int*>(smem + Cfg::kScanOff));
  // no piece to combine, unless a consumer below says so (only warp 0's lane 0 writes it)
  if (threadIdx.x == 0 && !p.pieces_only) p.pieces[blockIdx.x].count = 0;
  const Watchdog wd{abort_flag, p.status, p.timeout_ns};
  if (threadIdx.x < 32 * Cfg::kWarps)
    paged_consume_role<Cfg>(p, sh, smem, bars, wd);
  else
    paged_load_role<Cfg>(p, sh, smem_addr(smem), bars, wd);
}

// ---------------------------------------------------------------- combine
// What a prefix that all requests share adds: slots of the forward kernel's prefix variant.
struct PrefixPieces {
  const float* slots;   // [slot][unit_rows] x (D sums, then maxima, then sums of p)
  long long total;      // steps of the prefix launch
  int ctas;
  int steps;            // steps of one of its units
  int q_blocks;         // units of a k / v head
  int unit_rows;        // rows of a unit, 128 a tile
  int tile_batch;       // requests of a 128-row tile
};

struct CombineParams {
  const PagedPieces* pieces;
  const float* slots;
  uint16_t* out;
  int kv_heads, group, row_tiles;
  int pieces_only;
  PrefixPieces prefix;
};

// One CTA per entry of `pieces`; one float4 of a row a thread, all pieces in order.
template <int D, bool kBF16, bool kPrefix>
__global__ void __launch_bounds__(128) mfa_paged_combine_kernel(const CombineParams cp) {
  grid_dependency_wait();
  const PagedPieces pc = cp.pieces[blockIdx.x];
  if (pc.count == 0) return;
  const int unit_rows16 = cp.kv_heads * cp.row_tiles;
  const int request = pc.unit / unit_rows16, unit_row = pc.unit - request * unit_rows16;
  const int kv_head = unit_row / cp.row_tiles;
  const int row0 = (unit_row - kv_head * cp.row_tiles) * 16;
  const int rows = cp.group - row0 < 16 ? cp.group - row0 : 16;
  const int slot_rows = cp.group < 16 ? cp.group : 16;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 128) {
    const int row = i / (D / 4), col = 4 * (i % (D / 4));
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float pm, float pl, const float4& x) {
      const float next = fmaxf(m, pm);
      const float sub = next == -INFINITY ? 0.0f : next;
      const float f = ex2_approx(m - sub), w = ex2_approx(pm - sub);
      l = l * f + pl * w;
      acc.x = acc.x * f + x.x * w;
      acc.y = acc.y * f + x.y * w;
      acc.z = acc.z * f + x.z * w;
      acc.w = acc.w * f + x.w * w;
      m = next;
    };
    if (kPrefix) {
      const PrefixPieces& pp = cp.prefix;
      const int tile = request / pp.tile_batch;
      const int in = (request - tile * pp.tile_batch) * cp.group + row0 + row;
      const int tiles_a_unit = pp.unit_rows >> 7;
      const int qb = tile / tiles_a_unit;
      const int r = (tile - qb * tiles_a_unit) * 128 + in;
      const long long u = static_cast<long long>(kv_head) * pp.q_blocks + qb;
      const int c0 = cta_of_step(u * pp.steps, pp.total, pp.ctas);
      const int c1 = cta_of_step((u + 1) * pp.steps - 1, pp.total, pp.ctas);
      for (int c = c0; c <= c1; ++c) {
        const float* at = pp.slots + (c + u) * (static_cast<long long>(pp.unit_rows) * (D + 2));
        add(at[pp.unit_rows * D + r], at[pp.unit_rows * (D + 1) + r],
            *reinterpret_cast<const float4*>(at + static_cast<size_t>(r) * D + col));
      }
    }
    for (int k = 0; k < pc.count; ++k) {
      const int slot = k == 0 ? pc.first
                              : cp.pieces_only ? pc.cta + k + pc.unit : 2 * (pc.cta + k);
      const float* at = cp.slots + static_cast<size_t>(slot) * paged_slot_floats(slot_rows, D);
      add(at[slot_rows * D + row], at[slot_rows * (D + 1) + row],
          *reinterpret_cast<const float4*>(at + row * D + col));
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t* to = cp.out +
                   (static_cast<size_t>(request) * cp.kv_heads * cp.group + kv_head * cp.group +
                    row0 + row) * D + col;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<kBF16>(acc.x * inv, acc.y * inv),
                                               pack_pair<kBF16>(acc.z * inv, acc.w * inv));
  }
}

}  // namespace mfa
