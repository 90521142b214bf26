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
// Two or three CTAs per SM, each of four consumer warps and one producer warp, walk a common list
// of steps: a step is one 64-key tile of one unit, a unit one (request, k / v head, 16 query rows).
// The lengths are known to the GPU only, so every CTA sums them and takes an equal share of the
// steps. Tiles arrive by TMA, one box a page, in a ring of stages. In a tile each warp takes 16
// keys with a running maximum of its own; at the end of a unit the four warps' states meet in
// shared memory. What a CTA's share cuts off goes to a slot of the workspace as unnormalised 32-bit
// sums, which the combine kernel joins in CTA order.
//
// Measured on a B200 (64 requests of 100 to 16384 tokens, 8 k / v heads of 128, 4 rows each, bf16):
// 137 us, 6.3 TB/s of k and v, 96% of a copy's rate; DRAM reads equal the k and v bytes. Windows
// (100 requests, 4 heads of 64, up to 17 tiles a unit): 17.8 us, of which 4 are start-up
// (lengths, table, first copies) and a unit's merge takes as long as two tiles.
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
  const uint16_t* q;       // [batch, kv_heads * group, D], its strides in elements:
  long long q_request, q_head;
  int cols;                // columns of a row in memory: D, or 32 with D = 64 (see PagedConfig)
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
  // A prefix that all requests share, in the pages prefix_pages, as the first tiles of every
  // request (0: none, or one that the prefix kernel has; window is 0 with it).
  const int* prefix_pages;
  int prefix, prefix_tiles;
  float scale_log2;
  float* slots;            // of min(group, 16) rows each
  PagedPieces* pieces;     // [CTA], or [unit] if pieces_only
  unsigned long long timeout_ns;
  int* status;
};

// Rows of 32 columns run as D = 64: the boxes reach past them, where copies read zeros, which change
// no score, and what is computed there is not written. HBM sends the 32 columns only: 64 requests
// of 100 to 16384 tokens, 8 k / v heads, bf16 take 45.8 us at D = 32 (4.7 TB/s), 75.4 at D = 64 (5.7)
// and 137 at D = 128 (6.3).
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
  // CTAs of an SM, with 192 KB of stages together. (D = 64, two against three: 18.3 and 18.0 us at
  // 100 requests of window 1024, 69.5 and 68.1 at 100 of up to 17 thousand tokens, 27.9 and 26.0
  // with 16 rows; D = 128 has no registers for three.)
  static constexpr int kCtas = kD == 64 ? 3 : 2;
  static constexpr int kStages = 196608 / kCtas / (2 * kTileBytes);
  // a round of the merge: eight rows by 64 columns of each warp, or four rows by 128
  static constexpr int kMergeCols = 72;  // floats a row: float2s of four rows hit all banks once
  static constexpr int kMergeCols4 = 136;
  static constexpr int kMergeOff = kStages * 2 * kTileBytes;
  static constexpr int kStatsOff = kMergeOff + kWarps * 8 * kMergeCols * 4;  // [2][kWarps][kRows]
  static constexpr int kBarOff = kStatsOff + 2 * kWarps * kRows * 4;
  static constexpr int kBarFull = 0, kBarEmpty = kStages;
  static constexpr int kScanOff = kBarOff + 2 * kStages * 8;  // warp sums, start
  static constexpr int kAbortOff = kScanOff + 4 * (kWarps + 1 + 3 + kWarps + 1);
  static constexpr int kSmemBytes = kAbortOff + 4 + 1024;
  static_assert(kCtas * (kSmemBytes + 1024) <= 228 * 1024, "shared memory of an SM");
};

// Tiles of a request of n tokens: those of the prefix, those that hold sinks before the window,
// then the window's.
struct PagedSpan {
  int n, tiles, sinks, skip;
  __device__ void set(const PagedParams& p, int length) {
    const int most = p.columns << p.page_shift;  // < 2^31 (checked by the launcher)
    n = length < 0 ? 0 : length < most ? length : most;
    // a request that sees nothing has one tile, in which nothing is visible
    const int own = n > 0 ? ((n - 1) >> 6) + 1 : p.prefix_tiles == 0;
    const int w0 = p.window > 0 && n > p.window ? (n - p.window) >> 6 : 0;
    const int sb = (p.sinks >> 6) + ((p.sinks & 63) != 0);
    sinks = sb < w0 ? sb : w0;
    skip = w0 - sinks;
    tiles = p.prefix_tiles + own - skip;
  }
  // Tile t: whether it is of the prefix, its first key there or among the request's own, and the
  // first key behind the last of either.
  __device__ bool shared(const PagedParams& p, int t) const { return t < p.prefix_tiles; }
  __device__ int key0(const PagedParams& p, int t) const {
    const int own = t - p.prefix_tiles;
    return 64 * (own < 0 ? t : own < sinks ? own : own + skip);
  }
  __device__ int end(const PagedParams& p, int t) const { return shared(p, t) ? p.prefix : n; }
  __device__ bool visible(const PagedParams& p, int key, int end) const {
    return key < end && (p.window == 0 || key >= n - p.window || key < p.sinks);
  }
};

// CTA of step s when CTA c of `ctas` has the steps [c * total / ctas, (c + 1) * total / ctas).
__device__ __forceinline__ int cta_of_step(long long s, long long total, int ctas) {
  return static_cast<int>(((s + 1) * ctas - 1) / total);
}

// A unit's start and end (query, merge, output) cost about as much as two tiles of keys, so shares
// count two steps more than its tiles: 18.3 us against 20.7 with one and 18.4 with three at 100
// requests of 1 to 17 tiles (window 1024, D = 64); 137 to 138 us in all three at 64 requests of
// up to 256.
constexpr int kPagedUnitSteps = 2;

// A CTA's share of the steps, found by all its threads.
struct PagedShare {
  int total;    // steps of the whole call
  int ctas;     // CTAs that get a share
  int begin, end;
  int request;  // of step `begin`
  int length;   // its tokens
  int before;   // steps of the requests before it
  bool whole;   // CTA c has unit c instead, and nothing is cut
};

// The walk over a CTA's share, by segments (the tiles of one unit that it holds).
struct PagedCursor {
  PagedSpan span;
  int request, head, row0;  // k / v head and first query row (of the head's group) of the unit
  int t;                    // next tile of the unit
  int left;                 // steps left in the share
  int first;                // step of the unit's first tile
  int ahead;                // length of the next request, read early

  __device__ void read_ahead(const PagedParams& p) {
    ahead = p.lengths[request + 1 < p.batch ? request + 1 : request];
  }
  __device__ void init(const PagedParams& p, const PagedShare& sh) {
    if (sh.whole && static_cast<int>(blockIdx.x) < sh.ctas) {
      init_unit(p, static_cast<int>(blockIdx.x), 0, 1);
      return;
    }
    left = sh.end - sh.begin;
    request = sh.request;
    head = row0 = t = first = 0;
    if (left <= 0) return;
    span.set(p, sh.length);
    read_ahead(p);
    const int in = sh.begin - sh.before;
    const int unit = in / (span.tiles + kPagedUnitSteps);  // of the request
    t = in - unit * (span.tiles + kPagedUnitSteps);
    head = unit / p.row_tiles;
    row0 = 16 * (unit - head * p.row_tiles);
    first = sh.begin - t;
    if (t >= span.tiles) next_unit(p);
  }
  // CTA `rank` of the `size` that share one unit.
  __device__ void init_unit(const PagedParams& p, int unit, int rank, int size) {
    const int per_request = p.kv_heads * p.row_tiles;
    request = unit / per_request;
    const int in = unit - request * per_request;
    head = in / p.row_tiles;
    row0 = 16 * (in - head * p.row_tiles);
    ahead = p.lengths[request];
    span.set(p, ahead);
    first = 0;
    t = span.tiles * rank / size;
    left = span.tiles * (rank + 1) / size - t;
  }
  __device__ int segment() const { return span.tiles - t < left ? span.tiles - t : left; }
  // Past the unit's last tile (t >= tiles).
  __device__ void next_unit(const PagedParams& p) {
    const int rest = span.tiles + kPagedUnitSteps - t;
    left = left > rest ? left - rest : 0;
    if (left == 0) return;
    first += span.tiles + kPagedUnitSteps;
    t = 0;
    row0 += 16;
    if (row0 < p.group) return;
    row0 = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    ++request;
    span.set(p, ahead);
    read_ahead(p);
  }
  __device__ void advance(const PagedParams& p, int tiles) {
    left -= tiles;
    t += tiles;
    if (t == span.tiles && left > 0) next_unit(p);
  }
  // Query rows of the current unit.
  __device__ int rows(const PagedParams& p) const {
    const int r = p.group - row0;
    return r < 16 ? r : 16;
  }
  __device__ size_t query(const PagedParams& p) const {  // its first row in out
    return (static_cast<size_t>(request) * p.kv_heads + head) * p.group + row0;
  }
  __device__ int unit(const PagedParams& p) const {
    return (request * p.kv_heads + head) * p.row_tiles + (row0 >> 4);
  }
};

template <class Cfg>
__device__ __forceinline__ PagedShare paged_share(const PagedParams& p, int* scan) {
  // Each thread sums the steps of a run of requests; the block's exclusive sums tell the one
  // whose run holds the share's first step.
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + Cfg::kThreads - 1) / Cfg::kThreads;
  const int r0 = tid * per < p.batch ? tid * per : p.batch;
  const int r1 = r0 + per < p.batch ? r0 + per : p.batch;
  int mine = 0, most = 0;
  PagedSpan span;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    span.set(p, p.lengths[r]);
    mine += span.tiles + kPagedUnitSteps;
    most = max(most, span.tiles + kPagedUnitSteps);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  int* tops = scan + Cfg::kWarps + 4;
  if (lane == 31) {
    scan[warp] = upto;
    tops[warp] = most;
  }
  __syncthreads();
  int steps = 0, before = upto - mine;
#pragma unroll
  for (int w = 0; w <= Cfg::kWarps; ++w) {
    const int x = scan[w];
    if (w < warp) before += x;
    steps += x;
    most = max(most, tops[w]);
  }
  const int heads = p.kv_heads * p.row_tiles;
  PagedShare sh;
  sh.total = steps * heads;
  sh.ctas = static_cast<int>(gridDim.x) < sh.total ? static_cast<int>(gridDim.x) : sh.total;
  const int c = static_cast<int>(blockIdx.x);
  sh.begin = sh.end = 0;
  // A CTA for each unit, if there are enough and the longest is no more than a quarter over an
  // equal share: cutting nearly every unit in two costs more than that.
  sh.whole = p.batch * heads <= sh.ctas && 4LL * most * sh.ctas <= 5LL * sh.total;
  if (sh.whole) {
    sh.ctas = p.batch * heads;
    return sh;
  }
  if (c < sh.ctas) {
    sh.begin = static_cast<int>(static_cast<long long>(c) * sh.total / sh.ctas);
    sh.end = static_cast<int>(static_cast<long long>(c + 1) * sh.total / sh.ctas);
  }
  if (before * heads <= sh.begin && sh.begin < (before + mine) * heads) {
    int r = r0;
    if (per > 1) {  // with one request a thread, the span is that request's
      for (span.set(p, p.lengths[r]);
           (before + span.tiles + kPagedUnitSteps) * heads <= sh.begin;
           span.set(p, p.lengths[r])) {
        before += span.tiles + kPagedUnitSteps;
        ++r;
      }
    }
    scan[Cfg::kWarps + 1] = r;
    scan[Cfg::kWarps + 2] = before * heads;
    scan[Cfg::kWarps + 3] = span.n;
  }
  __syncthreads();
  sh.request = scan[Cfg::kWarps + 1];
  sh.before = scan[Cfg::kWarps + 2];
  sh.length = scan[Cfg::kWarps + 3];
  return sh;
}

// Producer warp: the tiles of the share, a box for every page that holds a visible key. Lane i
// looks up the page of box i of a batch of tiles (32 boxes at most, of one segment); the next
// batch's are on their way while this one's copies are issued.
template <class Cfg>
__device__ __forceinline__ void paged_load_role(const PagedParams& p, PagedCursor cur,
                                                uint32_t smem, uint32_t bars,
                                                const Watchdog& wd) {
  const int lane = threadIdx.x & 31;
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  const int box_shift = p.page_shift < 6 ? p.page_shift : 6;  // rows of a box
  const int tile_shift = 6 - box_shift;                       // boxes of a tile: 1, 2 or 4
  const uint32_t box_bytes = 128u << box_shift;
  struct Batch {
    int count;     // tiles
    int page;      // this lane's page, as the table has it
    bool visible;  // whether a key of this lane's box is seen (its page was looked up)
  };
  auto look_up = [&](const PagedCursor& at) -> Batch {
    Batch b;
    const int most = 32 >> tile_shift, seg = at.segment();
    b.count = seg < most ? seg : most;
    const int i = lane >> tile_shift, t = at.t + i;
    const int key0 = at.span.key0(p, t) + ((lane & ((1 << tile_shift) - 1)) << box_shift);
    b.visible = i < b.count && key0 < at.span.end(p, t) &&
                (p.window == 0 || key0 + (1 << box_shift) > at.span.n - p.window ||
                 key0 < p.sinks);
    b.page = 0;
    const int* table = at.span.shared(p, t)
                           ? p.prefix_pages
                           : p.block_table + static_cast<size_t>(at.request) * p.columns;
    if (b.visible) b.page = table[key0 >> p.page_shift];
    return b;
  };
  Batch batch{0, 0, false};
  if (cur.left > 0) batch = look_up(cur);
  int g = 0;
  bool ok = true;
  while (cur.left > 0 && ok) {
    PagedCursor next = cur;
    next.advance(p, batch.count);
    Batch later{0, 0, false};
    if (next.left > 0) later = look_up(next);
    const int head = cur.head;
    // a page outside the cache: a place outside the map, which reads as zero
    const bool bad = batch.visible && (batch.page < 0 || batch.page >= p.pages);
    if (bad) atomicCAS(p.status, 0, kStatusBadPage);
    const int page = bad ? p.pages : batch.page;
    const uint32_t have = __ballot_sync(0xffffffffu, batch.visible);
    for (int i = 0; i < batch.count; ++i) {
      const int st = g % Cfg::kStages;
      const uint32_t ph = static_cast<uint32_t>(g / Cfg::kStages) & 1u;
      if (!(ok = wait_warp(bar(Cfg::kBarEmpty + st), ph ^ 1u, wd, kSiteLoadKEmpty))) break;
      const uint32_t here = (have >> (i << tile_shift)) & ((1u << (1 << tile_shift)) - 1u);
      if (lane == 0)
        mbar_arrive_expect_tx(bar(Cfg::kBarFull + st),
                              2 * Cfg::kBoxes * box_bytes * __popc(here));
      __syncwarp();
      const int row0 = cur.span.key0(p, cur.t + i) & ((1 << p.page_shift) - 1);
      const uint32_t k_dst = smem + st * 2 * Cfg::kTileBytes, v_dst = k_dst + Cfg::kTileBytes;
      for (int j = 0; j < 1 << tile_shift; ++j) {
        const int pg = __shfl_sync(0xffffffffu, page, (i << tile_shift) + j);
        if (!((here >> j) & 1u) || lane != 0) continue;
#pragma unroll
        for (int x = 0; x < Cfg::kBoxes; ++x) {
          const uint32_t off = x * Cfg::kBoxBytes + j * box_bytes;
          tma_load_4d(k_dst + off, &p.tm_k, bar(Cfg::kBarFull + st), 64 * x, row0, head, pg);
          tma_load_4d(v_dst + off, &p.tm_v, bar(Cfg::kBarFull + st), 64 * x, row0, head, pg);
        }
      }
      ++g;
    }
    cur = next;
    batch = later;
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

// The 8x8 blocks of 16-bit values, as they stand and transposed.
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
// every 8 keys (scores) or 8 columns (out), the two at 2 q. With at most 8 rows the upper eight
// (g + 8) take part in the products only, as zeros, and are dropped.
// kCluster: the share is a part of one unit; its sums stay in shared memory, where the ring was.
template <class Cfg, bool kCluster>
__device__ __forceinline__ void paged_consume_role(const PagedParams& p, PagedCursor cur,
                                                   const PagedShare& sh, uint8_t* smem_ptr,
                                                   uint32_t bars, const Watchdog& wd) {
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

  // ldmatrix row addresses inside a tile: this lane's key row and the 16-byte chunk, which the
  // 128-byte swizzle moves to chunk ^ (row % 8)
  const int mat = lane >> 3, mrow = lane & 7;
  const uint32_t k_row = (warp * 16 + (mat >> 1) * 8 + mrow) * 128;
  const uint32_t v_row = (warp * 16 + (mat & 1) * 8 + mrow) * 128;
  auto chunk_off = [&](int chunk) -> uint32_t {
    return (chunk >> 3) * Cfg::kBoxBytes + (((chunk & 7) ^ mrow) << 4);
  };

  // Query fragments of a unit, straight from global memory; for every segment but the first they
  // are asked for when the one before has done its last scores, and arrive during its merge.
  uint32_t qf[kKSteps][4];
  auto read_query = [&](const PagedCursor& at) {
    const int rows = at.rows(p);
    const uint16_t* first = p.q + at.request * p.q_request + (at.head * p.group + at.row0) * p.q_head;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(first + (gq + 8 * r) * p.q_head) + q;
      const bool here = gq + 8 * r < rows;
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        const bool in = here && (D > 64 || 16 * kk < p.cols);
        qf[kk][r] = in ? src[8 * kk] : 0u;
        qf[kk][2 + r] = in ? src[8 * kk + 4] : 0u;
      }
    }
  };

  if (cur.left > 0) {
    read_query(cur);
    // The share's queries are a run of rows. Its first 128 lines are brought to L2: from HBM,
    // busy with keys, a unit's queries would take longer than the merge that hides them.
    const int heads = p.kv_heads * p.group;
    const int head = cur.head * p.group + cur.row0 + static_cast<int>(threadIdx.x) / (D / 64);
    const int request = cur.request + head / heads;
    if (request < p.batch)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.q + request * p.q_request +
                                                    head % heads * p.q_head +
                                                    64 * (threadIdx.x % (D / 64))));
  }
  int g = 0;
  bool ok = true, wrote = false, merged = false;
  while (cur.left > 0) {
    const int seg = cur.segment();
    const int rows = cur.rows(p);
    const bool upper = rows > 8;
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
      const int key0 = cur.span.key0(p, cur.t + i), end = cur.span.end(p, cur.t + i);
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};  // v rows 2 q, 2 q + 1 (+ 8 for the second)
      const bool edge = key0 + Cfg::kKeys > end ||
                        (p.window > 0 && key0 < cur.span.n - p.window &&
                         key0 + Cfg::kKeys > p.sinks);
      if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + warp * 16 + 8 * h + 2 * q;
          const bool a = cur.span.visible(p, key, end), b = cur.span.visible(p, key + 1, end);
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
                                      (upper && top[1] > m[1] + kRescaleThreshold))) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (r == 1 && !upper) break;
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
      // P: rows g, g + 8 by keys 2 q, then by keys 2 q + 8. Rounded to the type of v, as an operand of
      // the product with it; maxima, sums (of p before it is rounded) and outputs are 32-bit.
      uint32_t pf[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (r == 1 && !upper) break;
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

    // ---- the segment's end: the four warps' states to one. In a round every warp leaves its part
    // of some rows and columns in shared memory, and the 128 threads rescale, add and write
    // four columns of a row each.
    if (merged) named_bar_sync(1, 32 * Cfg::kWarps);  // the last segment's have been read
    PagedCursor next = cur;
    next.advance(p, seg);
    if (next.left > 0) read_query(next);
    const bool whole = cur.t == 0 && seg == cur.span.tiles;
    const bool to_slot = kCluster || p.pieces_only || !whole;
    const int unit = cur.unit(p);
    const int slot = p.pieces_only ? static_cast<int>(blockIdx.x) + unit
                                   : 2 * static_cast<int>(blockIdx.x) + (wrote ? 1 : 0);
    float* slot_at = kCluster
                         ? reinterpret_cast<float*>(smem_ptr)
                         : p.slots + static_cast<size_t>(slot) * paged_slot_floats(slot_rows, D);
    uint16_t* out_at = p.out + cur.query(p) * p.cols;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (q == 0) {
        stat_m[warp * Cfg::kRows + gq + 8 * r] = m[r];
        stat_l[warp * Cfg::kRows + gq + 8 * r] = l[r];
      }
    }
    // One thread's share of a round: four columns of a row, the warps' parts `part` floats apart.
    auto add_up = [&](int row, int col, const float* from, int part) {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w) top = fmaxf(top, stat_m[w * Cfg::kRows + row]);
      const float sub = top == -INFINITY ? 0.0f : top;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w) {
        const float f = ex2_approx(stat_m[w * Cfg::kRows + row] - sub);
        const float4 y = *reinterpret_cast<const float4*>(from + w * part);
        sum = fmaf(f, stat_l[w * Cfg::kRows + row], sum);
        acc.x = fmaf(f, y.x, acc.x);
        acc.y = fmaf(f, y.y, acc.y);
        acc.z = fmaf(f, y.z, acc.z);
        acc.w = fmaf(f, y.w, acc.w);
      }
      if (row >= rows || !ok) return;
      if (to_slot) {
        *reinterpret_cast<float4*>(slot_at + row * D + col) = acc;
        if (col == 0) {
          slot_at[slot_rows * D + row] = top;
          slot_at[slot_rows * (D + 1) + row] = sum;
        }
      } else if (D > 64 || col < p.cols) {
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2*>(out_at + row * p.cols + col) =
            make_uint2(pack_pair<Cfg::kBF16>(acc.x * inv, acc.y * inv),
                       pack_pair<Cfg::kBF16>(acc.z * inv, acc.w * inv));
      }
    };
    if (D == 128 && rows <= 4) {
      float* to = merge + (warp * 4 + gq) * Cfg::kMergeCols4 + 2 * q;
      if (gq < 4) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<float2*>(to + 8 * d) = make_float2(o[d][0], o[d][1]);
      }
      named_bar_sync(1, 32 * Cfg::kWarps);
      const int row = threadIdx.x >> 5, col = 4 * (threadIdx.x & 31);
      add_up(row, col, merge + row * Cfg::kMergeCols4 + col, 4 * Cfg::kMergeCols4);
    } else {
      const int row8 = threadIdx.x >> 4, col4 = 4 * (threadIdx.x & 15);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (r == 1 && !upper) break;
#pragma unroll
        for (int x = 0; x < Cfg::kBoxes; ++x) {
          if (r + x > 0) named_bar_sync(1, 32 * Cfg::kWarps);  // the round before has been read
#pragma unroll
          for (int d = 0; d < 8; ++d)
            *reinterpret_cast<float2*>(merge + (warp * 8 + gq) * Cfg::kMergeCols + 8 * d + 2 * q) =
                make_float2(o[8 * x + d][2 * r], o[8 * x + d][2 * r + 1]);
          named_bar_sync(1, 32 * Cfg::kWarps);
          add_up(8 * r + row8, 64 * x + col4, merge + row8 * Cfg::kMergeCols + col4,
                 8 * Cfg::kMergeCols);
        }
      }
    }
    if (!kCluster && threadIdx.x == 0 && to_slot && cur.t == 0) {
      // the unit starts here: its pieces run to the CTA of its last tile (said also when
      // unwinding: the combine kernel reads it in any case)
      const int last = sh.whole
                           ? static_cast<int>(blockIdx.x)
                           : cta_of_step(cur.first + cur.span.tiles - 1, sh.total, sh.ctas);
      PagedPieces out;
      out.count = last - static_cast<int>(blockIdx.x) + 1;
      out.first = slot;
      out.cta = static_cast<int>(blockIdx.x);
      out.unit = unit;
      p.pieces[p.pieces_only ? unit : static_cast<int>(blockIdx.x)] = out;
    }
    if (!whole) wrote = true;
    cur = next;
    merged = true;
  }
}

// Barriers of a CTA, by one thread, before any of them is used.
template <class Cfg>
__device__ __forceinline__ void paged_set_up(const PagedParams& p, uint32_t bars,
                                             volatile int* abort_flag) {
  tma_prefetch_desc(&p.tm_k);
  tma_prefetch_desc(&p.tm_v);
  *abort_flag = 0;
  for (int s = 0; s < Cfg::kStages; ++s) {
    mbar_init(bars + 8 * (Cfg::kBarFull + s), 1);
    mbar_init(bars + 8 * (Cfg::kBarEmpty + s), Cfg::kWarps);
  }
  mbar_init_fence();
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(PagedConfig<D, kBF16>::kThreads, PagedConfig<D, kBF16>::kCtas)
    mfa_paged_kernel(const __grid_constant__ PagedParams p) {
  using Cfg = PagedConfig<D, kBF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t bars = smem_addr(smem + Cfg::kBarOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kAbortOff);
  if (threadIdx.x == 0) {
    // the combine kernel may be scheduled; it waits for this grid before it reads
    grid_dependents_launch();
    paged_set_up<Cfg>(p, bars, abort_flag);
  }
  // Nothing above touches global memory. Behind a prefix kernel, whose results this one does not
  // read, it waits at its end instead (the combine kernel waits for this grid alone) and starts
  // on every SM that the prefix kernel has left. That rests on more than its own wait: the prefix
  // kernel's CTAs let it start only behind theirs, when the stream's earlier kernels have completed
  // and their writes are in global memory, and a grid that starts after that is taken to see
  // them. (64 requests behind 16001 tokens, 8 heads of 128: 45.8 us; 48.6 with the wait here, 47.9 with
  // a prefix kernel that is launched in plain stream order; 200 requests behind 3000: 63.4, 70.0
  // and 65.9.)
  if (!p.pieces_only) grid_dependency_wait();
  const PagedShare sh = paged_share<Cfg>(p, reinterpret_cast<int*>(smem + Cfg::kScanOff));
  // no piece to combine, unless a consumer below says so (the same thread writes that)
  if (threadIdx.x == 0 && !p.pieces_only) p.pieces[blockIdx.x].count = 0;
  const Watchdog wd{abort_flag, p.status, p.timeout_ns};
  PagedCursor cur;
  cur.init(p, sh);
  if (threadIdx.x < 32 * Cfg::kWarps)
    paged_consume_role<Cfg, false>(p, cur, sh, smem, bars, wd);
  else
    paged_load_role<Cfg>(p, cur, smem_addr(smem), bars, wd);
  if (p.pieces_only) grid_dependency_wait();
}

// Few units of few tiles: a cluster of CTAs (or one) a unit, which share its tiles and add their
// sums up in one another's shared memory. One launch, no scan over the requests, no workspace. The
// launcher takes it when all CTAs are resident at once and none has more than eight tiles; it
// measured (this against the two kernels, 8 k / v heads of 128, equal lengths) 4.6 against 7.0 us
// for 4 requests of 128 tokens (1 CTA a unit), 6.8 against 8.8 for 1000 and 11.5 against 12.9 for
// 4000 (8 CTAs), 5.7 against 7.5 for one request of 1000, 11.1 against 12.7 for 8000 but 17.3
// against 14.5 for 16000 (16 CTAs, 16 tiles each), and 9.9 against 13.9 for 32 of 512.
template <int D, bool kBF16>
__global__ void __launch_bounds__(PagedConfig<D, kBF16>::kThreads, PagedConfig<D, kBF16>::kCtas)
    mfa_paged_cluster_kernel(const __grid_constant__ PagedParams p) {
  using Cfg = PagedConfig<D, kBF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t bars = smem_addr(smem + Cfg::kBarOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kAbortOff);
  if (threadIdx.x == 0) {
    grid_dependents_launch();
    paged_set_up<Cfg>(p, bars, abort_flag);
  }
  __syncthreads();
  grid_dependency_wait();
  const int size = cluster_size(), rank = cluster_rank();
  const Watchdog wd{abort_flag, p.status, p.timeout_ns};
  PagedCursor cur;
  cur.init_unit(p, static_cast<int>(blockIdx.x) / size, rank, size);
  const int slot_rows = p.group < Cfg::kRows ? p.group : Cfg::kRows;
  float* sums = reinterpret_cast<float*>(smem);
  float* tops = sums + slot_rows * D;
  if (cur.left == 0) {  // no tile for this CTA: sums of nothing, which the others add as they are
    for (int i = threadIdx.x; i < slot_rows * (D / 4); i += Cfg::kThreads)
      reinterpret_cast<float4*>(sums)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (threadIdx.x < slot_rows) {
      tops[threadIdx.x] = -INFINITY;
      tops[slot_rows + threadIdx.x] = 0.0f;
    }
  } else if (threadIdx.x < 32 * Cfg::kWarps) {
    paged_consume_role<Cfg, true>(p, cur, PagedShare{}, smem, bars, wd);
  } else {
    paged_load_role<Cfg>(p, cur, smem_addr(smem), bars, wd);
  }
  __syncwarp();
  cluster_sync();
  // The CTAs take the unit's float4s in turn. (A CTA that is unwinding takes part: its sums are
  // not written, and the status word says so.)
  const int rows = cur.rows(p);
  const uint32_t base = smem_addr(sums), stats = smem_addr(tops);
  for (int i = rank + size * static_cast<int>(threadIdx.x); i < rows * (D / 4);
       i += size * Cfg::kThreads) {
    const int row = i / (D / 4), col = 4 * (i % (D / 4));
    if (D == 64 && col >= p.cols) continue;
    float m = -INFINITY;
    for (int c = 0; c < size; ++c) m = fmaxf(m, cluster_load(stats + 4 * row, c));
    const float sub = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < size; ++c) {
      const float w = ex2_approx(cluster_load(stats + 4 * row, c) - sub);
      const float pl = cluster_load(stats + 4 * (slot_rows + row), c);
      const float4 x = cluster_load4(base + 4 * (row * D + col), c);
      // (no weight is left out: of scores that are all NaN the maximum is -inf and the weight 0, of
      // an infinite one inf and NaN, and the sums, NaN in both, have to reach the output)
      l = fmaf(pl, w, l);
      acc.x = fmaf(x.x, w, acc.x);
      acc.y = fmaf(x.y, w, acc.y);
      acc.z = fmaf(x.z, w, acc.z);
      acc.w = fmaf(x.w, w, acc.w);
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint2*>(p.out + (cur.query(p) + row) * p.cols + col) =
        make_uint2(pack_pair<kBF16>(acc.x * inv, acc.y * inv),
                   pack_pair<kBF16>(acc.z * inv, acc.w * inv));
  }
  cluster_sync();  // nobody leaves while its sums may be read
}

// ---------------------------------------------------------------- combine
// What a prefix that all requests share adds: slots of the forward kernel's prefix variant.
struct PrefixPieces {
  const float* slots;   // [unit][split][unit_rows] x (D sums, then maxima, then sums of p)
  int splits;
  int q_blocks;         // units of a k / v head
  int unit_rows;        // rows of a unit, 128 a tile
  int tile_batch;       // requests of a 128-row tile
};

struct CombineParams {
  const PagedPieces* pieces;
  const float* slots;
  uint16_t* out;
  int kv_heads, group, row_tiles;
  int cols;  // as in PagedParams
  int pieces_only;
  PrefixPieces prefix;
};

// One CTA per entry of `pieces`; one float4 of a row a thread. The pieces are read eight at a time
// (one L2 round trip a batch) and folded in order.
template <int D, bool kBF16, bool kPrefix>
__global__ void __launch_bounds__(128) mfa_paged_combine_kernel(const CombineParams cp) {
  constexpr int kBatch = 8;
  grid_dependency_wait();
  const PagedPieces pc = cp.pieces[blockIdx.x];
  if (pc.count == 0) return;
  const int units_a_request = cp.kv_heads * cp.row_tiles;
  const int request = pc.unit / units_a_request, unit_row = pc.unit - request * units_a_request;
  const int kv_head = unit_row / cp.row_tiles;
  const int row0 = (unit_row - kv_head * cp.row_tiles) * 16;
  const int rows = cp.group - row0 < 16 ? cp.group - row0 : 16;
  const int slot_rows = cp.group < 16 ? cp.group : 16;
  // The prefix's pieces first: row `in_unit` (plus this row) of their slots.
  int prefix_count = 0, in_unit = 0;
  long long prefix_slot = 0;
  if (kPrefix) {
    const PrefixPieces& pp = cp.prefix;
    const int tile = request / pp.tile_batch, tiles_a_unit = pp.unit_rows >> 7;
    const int qb = tile / tiles_a_unit;
    in_unit = (tile - qb * tiles_a_unit) * 128 + (request - tile * pp.tile_batch) * cp.group + row0;
    const long long u = static_cast<long long>(kv_head) * pp.q_blocks + qb;
    prefix_count = pp.splits;
    prefix_slot = u * pp.splits;
  }
  const int count = prefix_count + pc.count;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 128) {
    const int row = i / (D / 4), col = 4 * (i % (D / 4));
    if (D == 64 && col >= cp.cols) continue;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < count; k0 += kBatch) {
      float pm[kBatch], pl[kBatch];
      float4 x[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int k = k0 + b;
        pm[b] = -INFINITY;
        pl[b] = 0.0f;
        x[b] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k >= count) continue;
        const float* at;
        int r, stride;
        if (kPrefix && k < prefix_count) {
          r = in_unit + row;
          stride = cp.prefix.unit_rows;
          at = cp.prefix.slots + (prefix_slot + k) * (static_cast<long long>(stride) * (D + 2));
        } else {
          const int piece = k - prefix_count;
          const int slot = piece == 0 ? pc.first
                                      : cp.pieces_only ? pc.cta + piece + pc.unit
                                                       : 2 * (pc.cta + piece);
          r = row;
          stride = slot_rows;
          at = cp.slots + static_cast<size_t>(slot) * paged_slot_floats(slot_rows, D);
        }
        pm[b] = at[stride * D + r];
        pl[b] = at[stride * (D + 1) + r];
        x[b] = *reinterpret_cast<const float4*>(at + static_cast<size_t>(r) * D + col);
      }
      float next = m;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) next = fmaxf(next, pm[b]);
      const float sub = next == -INFINITY ? 0.0f : next;
      const float f = ex2_approx(m - sub);
      l *= f;
      acc.x *= f;
      acc.y *= f;
      acc.z *= f;
      acc.w *= f;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const float w = ex2_approx(pm[b] - sub);
        l = fmaf(pl[b], w, l);
        acc.x = fmaf(x[b].x, w, acc.x);
        acc.y = fmaf(x[b].y, w, acc.y);
        acc.z = fmaf(x[b].z, w, acc.z);
        acc.w = fmaf(x[b].w, w, acc.w);
      }
      m = next;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t* to = cp.out +
                   ((static_cast<size_t>(request) * cp.kv_heads + kv_head) * cp.group + row0 + row) *
                       cp.cols + col;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<kBF16>(acc.x * inv, acc.y * inv),
                                               pack_pair<kBF16>(acc.z * inv, acc.w * inv));
  }
}

}  // namespace mfa
