// FlashAttention backward for sm_100a, fp16 or bf16: the last "next" item of the reference's README
// (backward pass, README.md:125). Not a translation: the reference has no backward. Two variants:
//   dense : D = 64, optional causal mask, as many k / v heads as query heads (mfa_bwd);
//   window: causal with a sliding window and sink tokens, k / v heads shared by groups of query
//           heads (mfa_bwd_window); D = 64, D = 32 as D = 64 with boxes that reach past the columns,
//           and D = 128.
//
// Given q, k, v, o, dO and the forward's row log-sum-exp L (natural log), with
// P = exp(scale * q k^T - L) and D_i = rowsum(dO ⊙ o) (mfa_bwd_prep_kernel):
//   dV = P^T dO,   dS = P ⊙ (dO v^T - D),   dQ = scale * dS k,   dK = scale * dS^T q.
// Passes of one persistent kernel, no atomics on sums (dQ gets its own pass, which recomputes S
// and dP, instead of accumulating across CTAs):
//   dQ pass  : a CTA keeps a 128-row block of q and dO resident and streams the k, v blocks;
//              S = q k^T and dP = dO v^T (tcgen05 SS MMAs into TMEM), dS in registers (fp16
//              or bf16 into TMEM), dQ += dS k (TS MMA; k read MN-major, no transpose).
//   dK/dV pass: a CTA keeps a 128-row block of k and v resident and streams the q, dO blocks
//              with their L and D slices; S^T = k q^T and dP^T = v dO^T, P^T and dS^T in TMEM,
//              dV += P^T dO and dK += dS^T q. At D = 128 a pass each for dK and dV (BwdPart); the
//              dV pass needs neither v nor dP.
// Dense units are dealt out by index (BwdCursor), the window's claimed from a counter, the longest
// of its dK/dV units in pieces whose 32-bit sums mfa_bwd_reduce_kernel adds (BwdWindowCursor).
// P and dS are operands of tensor-core products and therefore rounded to the type of q; everything
// else (S, dP, L, D, P before it is used, all sums) is held in 32 bits. The rounding of dS makes dQ and
// dK about 1.41 times as far off as their own, that of P dV.
// TMEM (columns): S or S^T [0,128), dP or dP^T [128,256) (not in the dV pass), the first operand
// [256,320): dS in the dQ pass, P^T in the dK/dV and dV passes, dS^T in the dK pass; dK/dV pass:
// dS^T [320,384), accumulators dV [384,448) and dK [448,512); the others: their one accumulator
// [320,384), at D = 128 [320,448).
// Warp roles as in the forward kernel (csrc/mfa_fwd_kernel.cuh): 16 softmax-side warps on
// 16x256b TMEM fragments (lane 4g + q: rows g and g + 8 of a 16-row slice, columns 2q, 2q + 1
// of every 8), two MMA warps (S and dP, accumulations; one elected lane issues), one TMA warp, one
// store thread (not at D = 128); every wait is bounded.
// The backward needs no row reductions (L and D come precomputed), so the 128 columns of a
// block are split between two warps per 16-row slice: warp w takes TMEM lane quadrant w % 4,
// slice half (w / 4) % 2 and column half w / 8, which doubles the warps that hide each other's
// latencies at the same TMEM footprint.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "mfa_common.cuh"
#include "mfa_exp2.cuh"
#include "mfa_ptx.cuh"

namespace mfa {

struct BwdParams {
  // {64, N, H, B} tensor maps, box {64, 128, 1, 1}, 128-byte swizzle (as the forward's)
  CUtensorMap tm_x, tm_y;    // resident: dQ pass q, dO; dK/dV pass k, v
  CUtensorMap tm_s0, tm_s1;  // streamed: dQ pass k, v; dK/dV pass q, dO
  CUtensorMap tm_o0, tm_o1;  // outputs: dQ pass dQ; dK/dV pass dK (o0), dV (o1)
  int n;                     // sequence length
  int heads;
  int bh;                    // batch * heads
  int blocks;                // 128-row blocks per head: ceil(N / 128)
  float scale;               // softmax scale (multiplies q.k; dQ and dK are scaled by it)
  float scale_log2;          // scale * log2(e)
  const float* lse2;         // [bh][blocks * 128]: L * log2(e), +inf past N
  const float* di;           // [bh][blocks * 128]: rowsum(dO ⊙ o), 0 past N
  unsigned long long timeout_ns;
  int* status;
  // CTAs [cta0, cta0 + ctas) of the launch run this pass
  int cta0;
  int ctas;
  int by_length;  // causal only: deal units out by length (below), else strided
  int reverse;    // CTA cta0 + c deals as CTA ctas - 1 - c (the second pass of a mixed launch)
  // Window variant only (see BwdWindowCursor)
  int window, sinks, sink_blocks;
  int group;         // query heads per k / v head
  int units;         // units of this pass, pieces counted
  int chunk_sink;    // dK/dV: steps of a piece, and pieces, of a sink block's unit ...
  int pieces_sink;
  int chunk_rest;    // ... and of any other block's
  int pieces_rest;
  int* claimed;      // units of this pass handed out so far
  float* partials;   // dK/dV: [slot][dK, dV][128][D] of the units in pieces
  // D = 128: the pass's gradient and its strides
  uint16_t* grad;
  long long grad_b, grad_h, grad_n;
};

template <class Cfg>
struct BwdCursor;
template <class Cfg>
struct BwdWindowCursor;

// What a pass over resident k and v computes. D = 64 does both at once; the two accumulators of
// D = 128 and the P^T and dS^T operands do not fit in TMEM together, so it takes a pass for each.
enum class BwdPart { kBoth, kDK, kDV };

template <bool kDKV_, bool kCausal_, bool kBF16_, bool kWindow_ = false, int kD_ = 64,
          BwdPart kPart_ = BwdPart::kBoth>
struct BwdConfig {
  static constexpr BwdPart kPart = kPart_;
  static constexpr bool kBoth = kDKV_ && kPart_ == BwdPart::kBoth;
  static constexpr bool kOnlyDV = kDKV_ && kPart_ == BwdPart::kDV;  // needs no dP, dS and v
  static_assert(kD_ == 64 || (kWindow_ && !kBoth), "D = 128: window variant, a pass each");
  // sliding window with sink tokens and grouped k / v heads, as the forward's window variant
  static constexpr bool kWindow = kWindow_;
  static_assert(!kWindow_ || kCausal_, "the window variant is causal");
  using Cursor = std::conditional_t<kWindow_, BwdWindowCursor<BwdConfig>, BwdCursor<BwdConfig>>;
  static constexpr bool kDKV = kDKV_;  // dK/dV pass (k, v resident) or dQ pass (q, dO resident)
  static constexpr bool kCausal = kCausal_;
  static constexpr bool kBF16 = kBF16_;
  static constexpr int kHeadDim = kD_;
  static constexpr int kRows = 128;  // resident rows per unit (M of every MMA)
  static constexpr int kCols = 128;  // streamed rows per step
  static constexpr int kTileBytes = kRows * kHeadDim * 2;
  static constexpr int kBoxes = kHeadDim / 64;       // 64-column boxes of a tile
  static constexpr int kBoxBytes = kRows * 64 * 2;
  // D = 64: two buffers for the resident tiles, three stages of a pair of streamed tiles.
  // D = 128, whose tiles are twice as large (seven fit): one buffer, and a ring for each streamed
  // tile of a step. The accumulation's operand (`late`: s0, in the dV pass s1) is held until
  // the step's end and has three stages; the other (`early`) is free after the S and dP
  // products and makes do with two (three in the dV pass, which has no second resident tile). With
  // two stages of both tiles together a step waited for its 64 KB from L2: 576 us where this took
  // 473 (16 heads x 8192, window 2048).
  static constexpr bool kSplit = kD_ == 128;
  static constexpr int STAGES = 3;
  static constexpr int kEarly = kOnlyDV ? 3 : 2;
  static constexpr int kVecSlots = kSplit ? 2 : STAGES;
  static constexpr int kResBuffers = kSplit ? 1 : 2;
  static constexpr int kResTiles = kOnlyDV ? 1 : 2;
  // buffer of a CTA's s-th unit, and the phase of its barriers
  __host__ __device__ static constexpr int res_buffer(int s) { return kResBuffers == 1 ? 0 : s & 1; }
  __host__ __device__ static constexpr uint32_t res_phase(int s) {
    return static_cast<uint32_t>(kResBuffers == 1 ? s : s >> 1) & 1u;
  }
  static constexpr int kSoftmaxWarps = 16;  // 16 rows x 64 columns each
  // Two MMA issuers: warp 16 the S and dP products (SS), warp 19 the accumulations (TS). One
  // thread issues a tcgen05.mma only every few tens of cycles, and a step has 24 products in
  // the dK/dV pass (16 in the dQ pass), most of them 128x64x16 (32 tensor-core cycles each).
  static constexpr int kMmaWarp = 16;
  static constexpr int kLoadWarp = 17;
  static constexpr int kStoreWarp = 18;  // TMA stores of finished units' gradients
  static constexpr int kAccWarp = 19;
  // As in the forward kernel: 640 threads (the two MMA warps, the load and the store warp fill
  // a fifth warpgroup) launch with 96 registers; setmaxnreg moves the control warpgroup to 64 and
  // the four softmax-side warpgroups to 104 (512 x 104 + 128 x 64 = 640 x 96; per SM
  // sub-partition 4 x 104 + 64 <= 512 registers per lane).
  static constexpr int kThreads = 32 * 20;
  static constexpr int kSoftmaxRegs = 104;
  static constexpr int kControlRegs = 64;

  // Shared memory (1024-aligned base). kSplit takes all of it: the slices and barriers lie in
  // front of the tiles, and the base is aligned by its declaration. Else slices and barriers lie
  // behind, with room for rounding the base up.
  static constexpr int kVecBytes = 2 * kCols * 4;  // L2 slice, D slice
  static constexpr int kHeaderBytes = kSplit ? 3 * 1024 : 0;
  static constexpr int kResOff = kHeaderBytes;  // [buffers][x, y]
  static constexpr int kStrOff = kResOff + kResBuffers * kResTiles * kTileBytes;
                                                // [STAGES][tile 0, tile 1]; kSplit: [STAGES] late
  static constexpr int kStageBytes = kSplit ? kTileBytes : 2 * kTileBytes;
  static constexpr int kEarlyOff = kStrOff + STAGES * kStageBytes;  // kSplit: [kEarly]
  static constexpr int kTilesEnd = kEarlyOff + (kSplit ? kEarly * kTileBytes : 0);
  static constexpr int kVecOff = kSplit ? 0 : kTilesEnd;  // [kVecSlots] (dK/dV pass)
  static constexpr int kBarOff = kSplit ? kVecSlots * kVecBytes
                                        : kVecOff + (kDKV ? kVecSlots * kVecBytes : 0);
  static constexpr int kBarResFull = 0;   // [2]
  static constexpr int kBarResEmpty = 2;  // [2]
  static constexpr int kBarStrFull = 4;   // [STAGES]
  static constexpr int kBarStrEmpty = kBarStrFull + STAGES;
  static constexpr int kBarSSFull = kBarStrEmpty + STAGES;  // S and dP computed
  static constexpr int kBarSSFree = kBarSSFull + 1;         // S and dP read by all 16 warps
  static constexpr int kBarOpFull = kBarSSFree + 1;         // fp16 operands written (16 warps)
  static constexpr int kBarAccDone = kBarOpFull + 1;        // TS MMAs of a step completed
  static constexpr int kBarStage = kBarAccDone + 1;         // output staging written (16 warps)
  static constexpr int kBarDrain = kBarStage + 1;  // [2]: one per MMA issuer
  // window variant: the ring of claimed units (index published / read by every other role)
  static constexpr int kClaims = 4;
  static constexpr int kBarClaimFull = kBarDrain + 2;  // [kClaims]
  static constexpr int kBarClaimEmpty = kBarClaimFull + (kWindow ? kClaims : 0);
  static constexpr int kBarEarlyFull = kBarClaimEmpty + (kWindow ? kClaims : 0);  // kSplit: [3]
  static constexpr int kBarEarlyEmpty = kBarEarlyFull + (kSplit ? 3 : 0);         // [3]
  static constexpr int kBarVecFull = kBarEarlyEmpty + (kSplit ? 3 : 0);           // [2]
  static constexpr int kBarVecEmpty = kBarVecFull + (kSplit ? 2 : 0);             // [2]
  static constexpr int kNumBars = kBarVecEmpty + (kSplit ? 2 : 0);
  // two MMA warps and, if outputs are staged, the store thread
  static constexpr int kClaimReaders = kSoftmaxWarps + (kSplit ? 2 : 3);
  static constexpr int kTmemSlotOff = kBarOff + kNumBars * 8;
  static constexpr int kAbortOff = kTmemSlotOff + 4;
  static constexpr int kSmemBytes =
      kSplit ? kTilesEnd : kAbortOff + 4 + (kWindow ? 4 * kClaims : 0) + 1024;
  static_assert(!kSplit || kAbortOff + 4 + 4 * kClaims <= kHeaderBytes, "header in front of the tiles");

  static constexpr int kTmemCols = 512;
  static constexpr int kColS = 0;
  static constexpr int kColDP = 128;
  static constexpr int kColOp0 = 256;  // dQ pass: dS; dK/dV pass: P^T
  static constexpr int kColOp1 = 320;  // dK/dV pass: dS^T
  static constexpr int kColAcc0 = kBoth ? 384 : 320;  // dQ pass: dQ; dK/dV pass: dV; the one alone
  static constexpr int kColAcc1 = 448;                // dK/dV pass: dK
  static constexpr int kPieceFloats = (kBoth ? 2 : 1) * kRows * kHeadDim;  // of BwdParams::partials
  static_assert(kColAcc0 + kHeadDim <= 512, "TMEM budget");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

// Window variant: where a CTA's roles find the units that its load thread has claimed.
struct BwdClaims {
  volatile int* ring;
  uint32_t bars;
  const Watchdog* wd;
};
enum class BwdRole { kLoad, kLane, kWarp };  // the load thread, one other thread, a whole warp

// Units are (batch * head, 128-row block) pairs, u = bh * blocks + block.
// dQ pass: unit = query block b, steps = key blocks [0, b + 1) with the causal mask, else all.
// dK/dV pass: unit = key block b, steps = query blocks [b, blocks) with the mask, else all.
// By default the pass's CTA c takes units c, c + ctas, ... (neighbouring CTAs on neighbouring
// blocks of a head, so the streamed blocks come from L2). With the mask and few units per CTA
// (by_length) unit lengths, which run from 1 to `blocks`, would leave CTAs unevenly loaded:
// the units are then taken in order of decreasing length (i = 0, 1, ...: block b = blocks - 1
// - i / bh for dQ, i / bh for dK/dV, head i % bh) and dealt out boustrophedon (wave k goes to
// CTAs 0..ctas-1 for even k, back from ctas-1 for odd k), which evens out the step counts.
template <class Cfg>
struct BwdCursor {
  int u;       // unit
  int j;       // streamed block of the current step
  int j0, j1;  // streamed blocks [j0, j1) of u
  int seg;     // units started by this CTA so far - 1

  __device__ void bounds(const BwdParams& p) {
    const int blk = u % p.blocks;
    if (Cfg::kDKV) {
      j0 = Cfg::kCausal ? blk : 0;
      j1 = p.blocks;
    } else {
      j0 = 0;
      j1 = Cfg::kCausal ? blk + 1 : p.blocks;
    }
    j = j0;
  }
  // Unit of this CTA's k-th assignment, or -1 past the end.
  __device__ static int unit_at(const BwdParams& p, int k) {
    // units <= 2^31 - 2^16 (checked by the launcher), k * ctas <= units: 32-bit arithmetic
    const int c0 = static_cast<int>(blockIdx.x) - p.cta0;
    const int c = p.reverse ? p.ctas - 1 - c0 : c0;
    const int units = p.bh * p.blocks;
    if (!Cfg::kCausal || !p.by_length) {
      const int u = k * p.ctas + c;
      return u < units ? u : -1;
    }
    const int i = k * p.ctas + ((k & 1) ? p.ctas - 1 - c : c);
    if (i >= units) return -1;
    const int wave = i / p.bh, head = i - wave * p.bh;
    const int blk = Cfg::kDKV ? wave : p.blocks - 1 - wave;
    return head * p.blocks + blk;
  }
  __device__ void init(const BwdParams& p, const BwdClaims&, BwdRole) {
    seg = 0;
    u = unit_at(p, 0);
    if (u >= 0) {
      bounds(p);
    } else {
      u = 0;
      j = j0 = j1 = 0;
    }
  }
  __device__ bool valid() const { return j < j1; }
  __device__ bool first_step() const { return j == j0; }
  __device__ void step(const BwdParams& p) {
    if (++j >= j1) {
      const int next = unit_at(p, seg + 1);
      if (next >= 0) {
        u = next;
        bounds(p);
        ++seg;
      }
    }
  }
  __device__ void next_unit(const BwdParams& p) {
    j = j1 - 1;
    step(p);
  }
  __device__ int row_block(const BwdParams& p) const { return u % p.blocks; }
  __device__ int head_row(const BwdParams& p) const { return u / p.blocks; }
  __device__ HeadBatch resident(const BwdParams& p) const {
    const int bh = u / p.blocks;
    return {bh % p.heads, bh / p.heads};
  }
  __device__ int block() const { return j; }
  __device__ size_t vec_row(const BwdParams& p) const { return static_cast<size_t>(u / p.blocks); }
  __device__ bool in_pieces() const { return false; }
  __device__ int slot() const { return 0; }
};

// Units of the window variant, with k / v heads shared by `group` query heads:
// dQ pass: unit = (query head, query block), steps = the key blocks that hold sinks before the
// window, then the window's blocks up to the diagonal.
// dK/dV pass: unit = (k / v head, key block), steps = for each of the group's query heads the
// query blocks from the diagonal to the last one that sees a key of the block (for a block
// with sinks, to the end of the sequence). The sum over the group stays in TMEM, so shared
// heads need no atomics. A unit of more steps than its chunk is cut into pieces of that many
// steps, whose sums go to `partials` for mfa_bwd_reduce_kernel: the units of sink blocks run
// over the whole sequence and would otherwise outlast all the others.
// Units differ in length, so each CTA claims its next one from a counter when it has issued
// the last loads of the current one; long units come first (sink blocks, then key blocks from
// the first; query blocks from the last). Which CTA takes a unit changes no result. The load
// thread claims, and passes the index to the other roles through a ring of kClaims entries.
// Measured at 16 query heads x 8192 over 4 k / v heads, window 2048, 16 sinks: 262 us, all CTAs done
// within 4%; a dK/dV step takes 2030 cycles and a dQ step 1770 (1950 on average without a window),
// a unit's start and end 1800, the change of passes 5400.
template <class Cfg>
struct BwdWindowCursor {
  const BwdClaims* c;
  BwdRole role;
  int seg;        // units started by this CTA so far - 1
  int blk, row;   // resident block, its batch * head row (k / v heads in the dK/dV pass)
  int j;          // streamed block, from...
  int j0, j1;     // ... [j0, j1); dQ: steps, the first `sinks` of them before the window
  int sinks, skip;
  int g;          // dK/dV: query head of the group
  int left;       // steps after this one; -1: no unit
  int steps;      // steps of the unit
  int piece;      // dK/dV: its slot in `partials`, or -1
  int ahead;      // load thread: the index claimed ahead

  // Steps of key block b in the dK/dV pass, for one query head.
  __device__ static int span(const BwdParams& p, int b) {
    if (b < p.sink_blocks) return p.blocks - b;
    const int last = b + ((126 + p.window) >> 7);  // block of query 128 b + 127 + window - 1
    return (last < p.blocks - 1 ? last : p.blocks - 1) - b + 1;
  }
  // The unit with index i; false if it is a piece past its unit's end.
  __device__ bool set(const BwdParams& p, int i) {
    piece = -1;
    if (Cfg::kDKV) {
      const int head_sinks = p.bh * p.pieces_sink;
      const int sink_units = p.sink_blocks * head_sinks;
      const bool sink = i < sink_units;
      const int pieces = sink ? p.pieces_sink : p.pieces_rest;
      const int per_block = p.bh * pieces;
      const int k = sink ? i : i - sink_units;
      const int part = k % per_block / p.bh;
      blk = k / per_block + (sink ? 0 : p.sink_blocks);
      row = k % p.bh;
      j0 = blk;
      j1 = blk + span(p, blk);
      const int chunk = sink ? p.chunk_sink : p.chunk_rest;
      const int total = (j1 - j0) * p.group;
      const int s0 = part * chunk;
      if (s0 >= total) return false;
      steps = total - s0 < chunk ? total - s0 : chunk;
      if (steps < total) piece = i;
      g = s0 / (j1 - j0);
      j = j0 + s0 % (j1 - j0);
      sinks = skip = 0;
    } else {
      blk = p.blocks - 1 - i / p.bh;
      row = i % p.bh;
      const int oldest = blk * Cfg::kRows - p.window + 1;
      const int w0 = oldest > 0 ? oldest >> 7 : 0;
      sinks = p.sink_blocks < w0 ? p.sink_blocks : w0;
      skip = w0 - sinks;
      j = j0 = g = 0;
      steps = j1 = blk + 1 - skip;
    }
    left = steps - 1;
    return true;
  }
  __device__ void claim(const BwdParams& p) {
    volatile int* ring = c->ring;
    const int slot = seg % Cfg::kClaims;
    const uint32_t phase = static_cast<uint32_t>(seg / Cfg::kClaims) & 1u;
    const uint32_t full = c->bars + 8u * static_cast<uint32_t>(Cfg::kBarClaimFull + slot);
    const uint32_t empty = c->bars + 8u * static_cast<uint32_t>(Cfg::kBarClaimEmpty + slot);
    left = -1;
    if (role == BwdRole::kLoad) {
      int i = ahead;
      while (i < p.units && !set(p, i)) i = atomicAdd(p.claimed, 1);
      const bool any = i < p.units;
      if (!any) left = -1;
      if (any) ahead = atomicAdd(p.claimed, 1);
      if (!wait_single(empty, phase ^ 1u, *c->wd, kSiteLoadQEmpty)) {
        left = -1;
        return;
      }
      ring[slot] = any ? i : -1;
      mbar_arrive(full);
      return;
    }
    const bool ok = role == BwdRole::kWarp ? wait_warp(full, phase, *c->wd, kSiteMmaQ)
                                           : wait_single(full, phase, *c->wd, kSiteMmaQ);
    if (!ok) return;
    const int i = ring[slot];
    if (role == BwdRole::kWarp) __syncwarp();
    if (role == BwdRole::kLane || (threadIdx.x & 31) == 0) mbar_arrive(empty);
    if (i >= 0) set(p, i);
  }
  __device__ void init(const BwdParams& p, const BwdClaims& claims, BwdRole r) {
    c = &claims;
    role = r;
    seg = 0;
    if (role == BwdRole::kLoad) ahead = atomicAdd(p.claimed, 1);
    claim(p);
  }
  __device__ bool valid() const { return left >= 0; }
  __device__ bool first_step() const { return left == steps - 1; }
  // The next step of this unit; false after the last one.
  __device__ bool advance() {
    if (left == 0) return false;
    --left;
    if (++j >= j1) {
      j = j0;
      ++g;
    }
    return true;
  }
  __device__ void next_unit(const BwdParams& p) {
    ++seg;
    claim(p);
  }
  __device__ void step(const BwdParams& p) {
    if (!advance()) next_unit(p);
  }
  __device__ int row_block(const BwdParams&) const { return blk; }
  __device__ int head_row(const BwdParams&) const { return row; }
  __device__ HeadBatch resident(const BwdParams& p) const {
    return {row % p.heads, row / p.heads};  // heads: of the resident tensors
  }
  __device__ int block() const { return Cfg::kDKV || j < sinks ? j : j + skip; }
  __device__ size_t vec_row(const BwdParams& p) const {  // query row of the L2 / D slices
    return static_cast<size_t>(row) * p.group + g;
  }
  __device__ bool in_pieces() const { return piece >= 0; }
  __device__ int slot() const { return piece; }
};

template <class Cfg>
__device__ __forceinline__ void bwd_load_role(const BwdParams& p, uint8_t* smem, uint32_t bars,
                                              const Watchdog& wd, const BwdClaims& claims) {
  constexpr int ST = Cfg::STAGES;
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  const uint32_t sbase = smem_addr(smem);
  tma_prefetch_desc(&p.tm_x);
  tma_prefetch_desc(&p.tm_y);
  tma_prefetch_desc(&p.tm_s0);
  tma_prefetch_desc(&p.tm_s1);
  const uint64_t keep = l2_policy_evict_last();  // streamed blocks are re-read by other units
  typename Cfg::Cursor cur;
  cur.init(p, claims, BwdRole::kLoad);
  int g = 0;
  int res_loaded = 0, str_issued = 0;
  [[maybe_unused]] int early_issued = 0, vec_issued = 0;
  HeadBatch res = {0, 0};              // of the resident tiles
  [[maybe_unused]] int str_h = 0;      // window variant: first head that the unit streams
  while (cur.valid()) {
    HeadBatch hb;  // of the streamed tiles; worked out before the waits
    if constexpr (Cfg::kWindow) {
      if (cur.first_step()) {
        res = cur.resident(p);
        str_h = Cfg::kDKV ? res.h * p.group : res.h / p.group;
      }
      hb = {str_h + (Cfg::kDKV ? cur.g : 0), res.b};
    } else {
      hb = res = cur.resident(p);
    }
    auto load_resident = [&]() -> bool {
      const int s = cur.seg, b = Cfg::res_buffer(s);
      if (!wait_single(bar(Cfg::kBarResEmpty + b), Cfg::res_phase(s) ^ 1u, wd, kSiteLoadQEmpty))
        return false;
      mbar_arrive_expect_tx(bar(Cfg::kBarResFull + b), Cfg::kResTiles * Cfg::kTileBytes);
      const int row = cur.row_block(p) * Cfg::kRows;
      const uint32_t dst = sbase + Cfg::kResOff + b * 2 * Cfg::kTileBytes;
#pragma unroll
      for (int x = 0; x < Cfg::kBoxes; ++x) {
        tma_load_4d(dst + x * Cfg::kBoxBytes, &p.tm_x, bar(Cfg::kBarResFull + b), 64 * x, row,
                    res.h, res.b);
        if (Cfg::kResTiles == 2)
          tma_load_4d(dst + Cfg::kTileBytes + x * Cfg::kBoxBytes, &p.tm_y,
                      bar(Cfg::kBarResFull + b), 64 * x, row, res.h, res.b);
      }
      res_loaded = s + 1;
      return true;
    };
    if (!Cfg::kSplit && cur.first_step()) {
      if (!load_resident()) break;
    }
    const int st = g % ST;
    const int row = cur.block() * Cfg::kCols;
    // L2 and D of the 128 streamed queries (padded arrays: 512-byte aligned slices)
    auto load_vec = [&](int slot, uint32_t full) {
      const size_t off = cur.vec_row(p) * p.blocks * Cfg::kCols + row;
      const uint32_t vdst = sbase + Cfg::kVecOff + slot * Cfg::kVecBytes;
      bulk_load(vdst, p.lse2 + off, Cfg::kCols * 4, full);
      bulk_load(vdst + Cfg::kCols * 4, p.di + off, Cfg::kCols * 4, full);
    };
    if constexpr (Cfg::kSplit) {
      auto load_tile = [&](uint32_t dst, const CUtensorMap* map, uint32_t full) {
        mbar_arrive_expect_tx(full, Cfg::kTileBytes);
#pragma unroll
        for (int x = 0; x < Cfg::kBoxes; ++x)
          tma_load_4d_hint(dst + x * Cfg::kBoxBytes, map, full, 64 * x, row, hb.h, hb.b, keep);
      };
      const int e = g % Cfg::kEarly;
      if (!wait_single(bar(Cfg::kBarEarlyEmpty + e),
                       (static_cast<uint32_t>(g / Cfg::kEarly) & 1u) ^ 1u, wd, kSiteLoadKEmpty))
        break;
      load_tile(sbase + Cfg::kEarlyOff + e * Cfg::kTileBytes, Cfg::kOnlyDV ? &p.tm_s0 : &p.tm_s1,
                bar(Cfg::kBarEarlyFull + e));
      early_issued = g + 1;
      if (!wait_single(bar(Cfg::kBarStrEmpty + st), (static_cast<uint32_t>(g / ST) & 1u) ^ 1u, wd,
                       kSiteLoadKEmpty))
        break;
      load_tile(sbase + Cfg::kStrOff + st * Cfg::kTileBytes, Cfg::kOnlyDV ? &p.tm_s1 : &p.tm_s0,
                bar(Cfg::kBarStrFull + st));
      str_issued = g + 1;
      // behind the streamed tiles, whose stages are free before the last unit's resident ones
      if (cur.first_step() && !load_resident()) break;
      if constexpr (Cfg::kDKV) {
        if (!wait_single(bar(Cfg::kBarVecEmpty + (g & 1)), (static_cast<uint32_t>(g >> 1) & 1u) ^ 1u,
                         wd, kSiteLoadKEmpty))
          break;
        mbar_arrive_expect_tx(bar(Cfg::kBarVecFull + (g & 1)), Cfg::kVecBytes);
        load_vec(g & 1, bar(Cfg::kBarVecFull + (g & 1)));
        vec_issued = g + 1;
      }
    } else {
      if (!wait_single(bar(Cfg::kBarStrEmpty + st), (static_cast<uint32_t>(g / ST) & 1u) ^ 1u, wd,
                       kSiteLoadKEmpty))
        break;
      mbar_arrive_expect_tx(bar(Cfg::kBarStrFull + st),
                            2 * Cfg::kTileBytes + (Cfg::kDKV ? Cfg::kVecBytes : 0));
      const uint32_t dst = sbase + Cfg::kStrOff + st * 2 * Cfg::kTileBytes;
      tma_load_4d_hint(dst, &p.tm_s0, bar(Cfg::kBarStrFull + st), 0, row, hb.h, hb.b, keep);
      tma_load_4d_hint(dst + Cfg::kTileBytes, &p.tm_s1, bar(Cfg::kBarStrFull + st), 0, row, hb.h,
                       hb.b, keep);
      if (Cfg::kDKV) load_vec(st, bar(Cfg::kBarStrFull + st));
      str_issued = g + 1;
    }
    ++g;
    cur.step(p);
  }
  if (*wd.abort) {
    // the last copies into each of a ring's `slots`, of `issued`
    auto drain = [&](int full, int slots, int issued) {
      for (int i = 0; i < slots; ++i) {
        int last = -1;
        for (int x = i; x < issued; x += slots) last = x;
        if (last >= 0) drain_wait(bar(full + i), static_cast<uint32_t>(last / slots) & 1u);
      }
    };
    drain(Cfg::kBarResFull, Cfg::kResBuffers, res_loaded);
    drain(Cfg::kBarStrFull, ST, str_issued);
    if constexpr (Cfg::kSplit) {
      drain(Cfg::kBarEarlyFull, Cfg::kEarly, early_issued);
      drain(Cfg::kBarVecFull, 2, vec_issued);
    }
  }
}

// kAcc false: the S and dP products of every step (warp kMmaWarp); kAcc true: the
// accumulations into dQ, or dV and dK (warp kAccWarp). Both read the streamed stage, whose
// empty barrier counts one commit from each.
template <class Cfg, bool kAcc>
__device__ __forceinline__ void bwd_mma_role(const BwdParams& p, uint8_t* smem, uint32_t bars,
                                             uint32_t tmem, const Watchdog& wd,
                                             const BwdClaims& claims) {
  constexpr int ST = Cfg::STAGES;
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  const uint32_t sbase = smem_addr(smem);
  constexpr uint32_t kIdescSS = idesc_f16_f32(128, 128, false, Cfg::kBF16);
  constexpr uint32_t kIdescTS = idesc_f16_f32(128, Cfg::kHeadDim, true, Cfg::kBF16);
  constexpr uint32_t kHi = smem_desc_hi(1024, kSwizzle128B);
  constexpr uint32_t kTile = Cfg::kTileBytes >> 4;
  const uint32_t res_lo = smem_desc_lo(sbase + Cfg::kResOff, 16);
  const uint32_t str_lo = smem_desc_lo(sbase + Cfg::kStrOff, 16);
  // MN-major (the streamed rows are the K of the accumulations): the leading offset goes from one
  // 64-column box to the next (unused at D = 64)
  const uint32_t str_mn_lo = smem_desc_lo(sbase + Cfg::kStrOff, Cfg::kBoxBytes);
  [[maybe_unused]] const uint32_t early_lo = smem_desc_lo(sbase + Cfg::kEarlyOff, 16);
  // descriptor offset (16-byte units) of the kk-th 16 columns of a K-major tile
  auto k_off = [](int kk) -> uint32_t {
    return static_cast<uint32_t>((kk >> 2) * (Cfg::kBoxBytes >> 4) + (kk & 3) * 2);
  };
  const bool leader = elect_one();
  bool issued_any = false;

  typename Cfg::Cursor cur;
  cur.init(p, claims, BwdRole::kWarp);
  int gs = 0, gp = 0;
  // S and dP of step gs once the softmax warps have read those of step gs - 1.
  auto issue_ss = [&]() -> bool {
    const int b = Cfg::res_buffer(cur.seg);
    if (cur.first_step()) {
      if (!wait_warp(bar(Cfg::kBarResFull + b), Cfg::res_phase(cur.seg), wd, kSiteMmaQ))
        return false;
    }
    const int st = gs % ST;
    [[maybe_unused]] const int e = gs % Cfg::kEarly;
    if constexpr (Cfg::kSplit) {
      if (!wait_warp(bar(Cfg::kBarEarlyFull + e), static_cast<uint32_t>(gs / Cfg::kEarly) & 1u, wd,
                     kSiteMmaK))
        return false;
    }
    if (!Cfg::kOnlyDV) {
      if (!wait_warp(bar(Cfg::kBarStrFull + st), static_cast<uint32_t>(gs / ST) & 1u, wd,
                     kSiteMmaK))
        return false;
    }
    if (gs > 0) {
      if (!wait_warp(bar(Cfg::kBarSSFree), static_cast<uint32_t>(gs - 1) & 1u, wd, kSiteMmaSFree))
        return false;
    }
    tc_fence_after();
    if (leader) {
      const uint32_t xd = res_lo + b * 2 * kTile, yd = xd + kTile;
      uint32_t s0 = str_lo + st * 2 * kTile, s1 = s0 + kTile;
      if constexpr (Cfg::kSplit) {
        s1 = early_lo + e * kTile;  // unused in the dV pass
        s0 = Cfg::kOnlyDV ? s1 : str_lo + st * kTile;
      }
#pragma unroll
      for (int kk = 0; kk < Cfg::kHeadDim / 16; ++kk)  // S = x s0^T
        mma_ss(tmem + Cfg::kColS, desc_join(xd + k_off(kk), kHi), desc_join(s0 + k_off(kk), kHi),
               kIdescSS, kk > 0 ? 1u : 0u);
      if constexpr (!Cfg::kOnlyDV) {
#pragma unroll
        for (int kk = 0; kk < Cfg::kHeadDim / 16; ++kk)  // dP = y s1^T
          mma_ss(tmem + Cfg::kColDP, desc_join(yd + k_off(kk), kHi), desc_join(s1 + k_off(kk), kHi),
                 kIdescSS, kk > 0 ? 1u : 0u);
      }
      mma_commit(bar(Cfg::kBarSSFull));
      if constexpr (Cfg::kSplit) {
        mma_commit(bar(Cfg::kBarEarlyEmpty + e));
        if (cur.left == 0) mma_commit(bar(Cfg::kBarResEmpty));  // the unit's last products
      }
      if constexpr (!Cfg::kOnlyDV) mma_commit(bar(Cfg::kBarStrEmpty + st));
    }
    __syncwarp();
    issued_any = true;
    ++gs;
    cur.step(p);
    return true;
  };

  if (!kAcc) {
    while (cur.valid())
      if (!issue_ss()) goto unwind;
  }
  while (kAcc && cur.valid()) {
    {
      const int st = gp % ST;
      // the stage's tiles are this thread's operands too
      if (!wait_warp(bar(Cfg::kBarStrFull + st), static_cast<uint32_t>(gp / ST) & 1u, wd,
                     kSiteMmaK))
        goto unwind;
      if (!wait_warp(bar(Cfg::kBarOpFull), static_cast<uint32_t>(gp) & 1u, wd, kSiteMmaPFull))
        goto unwind;
      tc_fence_after();
      if (leader) {
        const bool fresh = cur.first_step();
        const uint32_t s0 = str_mn_lo + st * (Cfg::kStageBytes >> 4);  // kSplit: the late tile
        [[maybe_unused]] const uint32_t s1 = s0 + kTile;
        if (Cfg::kBoth) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // dV += P^T dO
            mma_ts(tmem + Cfg::kColAcc0, tmem + Cfg::kColOp0 + 8 * kk,
                   desc_join(s1 + 128 * kk, kHi), kIdescTS, (!fresh || kk > 0) ? 1u : 0u);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // dK += dS^T q
            mma_ts(tmem + Cfg::kColAcc1, tmem + Cfg::kColOp1 + 8 * kk,
                   desc_join(s0 + 128 * kk, kHi), kIdescTS, (!fresh || kk > 0) ? 1u : 0u);
        } else {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // dQ += dS k; dK += dS^T q or dV += P^T dO alone
            mma_ts(tmem + Cfg::kColAcc0, tmem + Cfg::kColOp0 + 8 * kk,
                   desc_join(s0 + 128 * kk, kHi), kIdescTS, (!fresh || kk > 0) ? 1u : 0u);
        }
        mma_commit(bar(Cfg::kBarAccDone));
        mma_commit(bar(Cfg::kBarStrEmpty + st));
        if constexpr (Cfg::kSplit && Cfg::kDKV) mma_commit(bar(Cfg::kBarVecEmpty + (gp & 1)));
      }
      __syncwarp();
      issued_any = true;
      ++gp;
      cur.step(p);
    }
  }
  // Every commit of this pass has arrived before the role returns (the barriers may be
  // initialised again for a second pass).
  if (issued_any) {
    if (leader) mma_commit(bar(Cfg::kBarDrain + (kAcc ? 1 : 0)));
    __syncwarp();
    // on failure the CTA unwinds
    wait_warp(bar(Cfg::kBarDrain + (kAcc ? 1 : 0)), 0, wd, kSiteMmaDrain);
  }
  return;

unwind:
  if (issued_any) {
    if (leader) mma_commit(bar(Cfg::kBarDrain + (kAcc ? 1 : 0)));
    __syncwarp();
    drain_wait(bar(Cfg::kBarDrain + (kAcc ? 1 : 0)), 0);
  }
}

// One step of a softmax-side warp on its 16 rows: P = 2^(S * scale * log2 e - L2), and
// dS = P ⊙ (dP - D). dQ pass: rows are queries, L2 and D are per row; dK/dV pass: rows are
// keys, columns queries, L2 and D come per column from the streamed slices in shared memory.
template <class Cfg>
__device__ __forceinline__ bool bwd_step(const BwdParams& p, uint8_t* smem, uint32_t bars,
                                         uint32_t tS, uint32_t tDP, uint32_t tOp0, uint32_t tOp1,
                                         int lane, int half, int g, int blk, int j, int row0,
                                         const float (&lrow)[2], const float (&drow)[2],
                                         const Watchdog& wd) {
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  auto f = [](uint32_t u) { return __uint_as_float(u); };
  if (!wait_warp(bar(Cfg::kBarSSFull), static_cast<uint32_t>(g) & 1u, wd, kSiteSoftSFull))
    return false;
  tc_fence_after();
  // [4i + e]: row g + 8 (e / 2), column 64 * half + 8i + 2q + e % 2 (tS, tDP already point at
  // this warp's column half)
  uint32_t sr[32];
  [[maybe_unused]] uint32_t dp[32];
  if constexpr (Cfg::kOnlyDV)
    tmem_ld_16x256b_sync(tS, sr);
  else
    tmem_ld2_16x256b_sync(tS, sr, tDP, dp);
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar(Cfg::kBarSSFree));

  const int q2 = 2 * (lane & 3) + 64 * half;  // first of this thread's columns in a block
  const int gq = lane >> 2;
  if constexpr (Cfg::kWindow) {
    // This thread's 16 columns of a row are c0 + 8 i + e; see window_bits. (Keys past N are past
    // every query; queries past N have L2 = +inf, so their P is 0.)
    const int res0 = row0 + gq, str0 = j * Cfg::kCols + q2;  // first resident row, streamed column
    if constexpr (!Cfg::kDKV) {
      // resident queries, streamed keys: as in the forward kernel
      const int key0 = j * Cfg::kCols;
      if (key0 + Cfg::kCols - 1 > row0 ||
          (key0 <= row0 + 15 - p.window && key0 + Cfg::kCols > p.sinks)) {
        const uint32_t sink_bits = window_bits(p.sinks - 1 - str0);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int t = res0 + 8 * r - str0;
          const uint32_t seen = window_bits(t) & (~window_bits(t - p.window) | sink_bits);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (!((seen >> k) & 1u)) sr[4 * (k >> 1) + 2 * r + (k & 1)] = __float_as_uint(-INFINITY);
        }
      }
    } else {
      // resident keys, streamed queries: those from the key on, up to window - 1 after it (for a
      // sink, all)
      if (j == blk || ((j + 1) * Cfg::kCols > row0 + p.window && row0 + 16 > p.sinks)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int t = res0 + 8 * r - str0;
          uint32_t seen = ~window_bits(t - 1);
          if (res0 + 8 * r >= p.sinks) seen &= window_bits(t + p.window - 1);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (!((seen >> k) & 1u)) sr[4 * (k >> 1) + 2 * r + (k & 1)] = __float_as_uint(-INFINITY);
        }
      }
    }
  } else {
    if (!Cfg::kDKV) {
      // keys past N (last key block) and, with the mask, keys after the query row
      if (j == p.blocks - 1) {
        const int valid = p.n - j * Cfg::kCols;
        if (valid < Cfg::kCols) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (8 * i + q2 + (e & 1) >= valid) sr[4 * i + e] = __float_as_uint(-INFINITY);
        }
      }
      if (Cfg::kCausal) {
        const int t0 = row0 + gq - j * Cfg::kCols;  // column k masked when k > t0 (+8 for e >= 2)
        if (j * Cfg::kCols + Cfg::kCols - 1 > row0) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (8 * i + q2 + (e & 1) > t0 + 8 * (e >> 1)) sr[4 * i + e] = __float_as_uint(-INFINITY);
        }
      }
    } else if (Cfg::kCausal && j == blk) {
      // diagonal block: queries (columns) before the key row score -inf
      const int t0 = row0 + gq - j * Cfg::kCols;  // column k masked when k < t0 (+8 for e >= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (8 * i + q2 + (e & 1) < t0 + 8 * (e >> 1)) sr[4 * i + e] = __float_as_uint(-INFINITY);
    }
  }

  const uint64_t c2 = f2_splat(p.scale_log2);
  [[maybe_unused]] uint32_t pk[16], dk[16];  // [2i + r]: row g + 8r, columns 8i + q2, 8i + q2 + 1 (16x128b)
  const int st = g % Cfg::kVecSlots;
  const float* vec = reinterpret_cast<const float*>(smem + Cfg::kVecOff + st * Cfg::kVecBytes);
  if (Cfg::kDKV) {
    // the L2 / D slices came by bulk copy: observe their completion before reading them (the
    // stage cannot be refilled before this step's OpFull)
    if (!wait_warp(bar((Cfg::kSplit ? Cfg::kBarVecFull : Cfg::kBarStrFull) + st),
                   static_cast<uint32_t>(g / Cfg::kVecSlots) & 1u, wd, kSiteSoftStage))
      return false;
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int i = k >> 1, r = k & 1;
    uint64_t nl, d2;
    if (Cfg::kDKV) {
      const float2 lv = *reinterpret_cast<const float2*>(vec + 8 * i + q2);
      const float2 dv = *reinterpret_cast<const float2*>(vec + Cfg::kCols + 8 * i + q2);
      nl = f2_pack(-lv.x, -lv.y);
      d2 = f2_pack(dv.x, dv.y);
    } else {
      nl = f2_splat(-lrow[r]);
      d2 = f2_splat(drow[r]);
    }
    const uint64_t x = f2_fma(f2_pack(f(sr[2 * k]), f(sr[2 * k + 1])), c2, nl);
    float x0, x1;
    f2_unpack(x, x0, x1);
    const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
    if constexpr (!Cfg::kOnlyDV) {
      const uint64_t t = f2_add(f2_pack(f(dp[2 * k]), f(dp[2 * k + 1])), f2_neg(d2));
      const uint64_t ds = f2_mul(f2_pack(e0, e1), t);
      float ds0, ds1;
      f2_unpack(ds, ds0, ds1);
      dk[k] = pack_pair<Cfg::kBF16>(ds0, ds1);
    }
    pk[k] = pack_pair<Cfg::kBF16>(e0, e1);
  }
  // The operand columns are free once the previous step's TS MMAs have completed.
  if (g > 0) {
    if (!wait_warp(bar(Cfg::kBarAccDone), static_cast<uint32_t>(g - 1) & 1u, wd, kSiteSoftODone))
      return false;
    tc_fence_after();
  }
  if constexpr (Cfg::kBoth) {
    tmem_st_16x128b_x8(tOp0, pk);
    tmem_st_16x128b_x8(tOp1, dk);
  } else if constexpr (Cfg::kOnlyDV) {
    tmem_st_16x128b_x8(tOp0, pk);
  } else {
    tmem_st_16x128b_x8(tOp0, dk);
  }
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar(Cfg::kBarOpFull));
  return true;
}

template <class Cfg>
__device__ __forceinline__ void bwd_softmax_role(const BwdParams& p, uint8_t* smem, uint32_t bars,
                                                 uint32_t tmem, const Watchdog& wd,
                                                 const BwdClaims& claims) {
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int slice = (warp & 3) * 32 + ((warp >> 2) & 1) * 16;
  const int half = warp >> 3;  // columns [64 half, 64 half + 64) of a block
  const int gq = lane >> 2;
  const int q = lane & 3;
  const uint32_t lb = static_cast<uint32_t>(slice) << 16;
  const uint32_t tS = tmem + lb + Cfg::kColS + 64 * half;
  const uint32_t tDP = tmem + lb + Cfg::kColDP + 64 * half;
  // P / dS operands: fp16 / bf16 pairs, 32 columns per half
  const uint32_t tOp0 = tmem + lb + Cfg::kColOp0 + 32 * half;
  const uint32_t tOp1 = tmem + lb + Cfg::kColOp1 + 32 * half;
  int g = 0;
  typename Cfg::Cursor cur;
  cur.init(p, claims, BwdRole::kWarp);
  while (cur.valid()) {
    const int blk = cur.row_block(p);
    const int bh = cur.head_row(p);
    const int row0 = blk * Cfg::kRows + slice;  // first resident row of this warp
    float lrow[2] = {0.f, 0.f}, drow[2] = {0.f, 0.f};
    if (!Cfg::kDKV) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const size_t idx = static_cast<size_t>(bh) * p.blocks * Cfg::kRows + row0 + gq + 8 * r;
        lrow[r] = p.lse2[idx];
        drow[r] = p.di[idx];
      }
    }
    const int b = Cfg::res_buffer(cur.seg);
    if constexpr (Cfg::kWindow) {
      do {
        if (!bwd_step<Cfg>(p, smem, bars, tS, tDP, tOp0, tOp1, lane, half, g, blk, cur.block(),
                           row0, lrow, drow, wd))
          return;
        ++g;
      } while (cur.advance());
    } else {
      const int j0 = cur.j0, j1 = cur.j1;
      for (int j = j0; j < j1; ++j, ++g) {
        if (!bwd_step<Cfg>(p, smem, bars, tS, tDP, tOp0, tOp1, lane, half, g, blk, j, row0, lrow,
                           drow, wd))
          return;
      }
    }
    // ---- unit epilogue. A unit in pieces: 32-bit sums to its slot of `partials`. Else the scaled
    // accumulators, rounded, go to the staging tiles and the store thread's TMA (D = 64), or
    // straight to global memory (D = 128).
    if (!wait_warp(bar(Cfg::kBarAccDone), static_cast<uint32_t>(g - 1) & 1u, wd, kSiteSoftOFinal))
      return;
    tc_fence_after();
    [[maybe_unused]] uint8_t* res = smem + Cfg::kResOff + b * 2 * Cfg::kTileBytes;
    // This warp's 32 of the accumulator's columns: 16-byte chunks 4 * half .. 4 * half + 3 of each of
    // its rows in the 128B-swizzled staging tile.
    auto stage_acc = [&](uint32_t col, float mul, uint8_t* dst_tile) {
      uint32_t a[16];
      tmem_ld_16x256b_sync(tmem + lb + col + 32 * half, a);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = slice + gq + 8 * r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = pack_pair<Cfg::kBF16>(__uint_as_float(a[4 * i + 2 * r]) * mul,
                                                   __uint_as_float(a[4 * i + 2 * r + 1]) * mul);
          const uint32_t dst =
              smem_addr(dst_tile + row * 128 + (((4 * half + i) ^ (row & 7)) << 4) + 4 * q);
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(w) : "memory");
        }
      }
    };
    // kSplit: straight to global memory, 16 bytes a thread after a transposition inside each
    // quad (64 bytes a row). The resident tiles are then free after the last products that read
    // them, and the next unit's are loaded while this one ends. (Staged: 473 us where this takes
    // 449, at 16 heads x 8192, window 2048; 244 and 223 at 4 x 16 x 2048, window 512.)
    [[maybe_unused]] auto write_acc = [&](uint32_t col, float mul) {
      const HeadBatch hb = cur.resident(p);
      uint16_t* at = p.grad + hb.b * p.grad_b + hb.h * p.grad_h + (row0 + gq) * p.grad_n + 8 * q;
#pragma unroll
      for (int sub = 0; sub < Cfg::kBoxes; ++sub) {
        const int c0 = Cfg::kHeadDim / 2 * half + 32 * sub;
        uint32_t a[16];
        tmem_ld_16x256b_sync(tmem + lb + col + c0, a);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t w[4];  // columns c0 + 8 i + 2 q, + 1
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack_pair<Cfg::kBF16>(__uint_as_float(a[4 * i + 2 * r]) * mul,
                                         __uint_as_float(a[4 * i + 2 * r + 1]) * mul);
#pragma unroll
          for (int bit = 1; bit <= 2; bit <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i & bit) continue;
              const uint32_t got =
                  __shfl_xor_sync(0xffffffffu, (q & bit) ? w[i] : w[i + bit], bit);
              if (q & bit)
                w[i] = got;
              else
                w[i + bit] = got;
            }
          }
          if (row0 + gq + 8 * r < p.n)
            *reinterpret_cast<uint4*>(at + 8 * r * p.grad_n + c0) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    };
    if (Cfg::kDKV && cur.in_pieces()) {
      // a piece's sums, unscaled, for the reduce kernel
      float* part = p.partials + static_cast<size_t>(cur.slot()) * Cfg::kPieceFloats;
      auto keep_acc = [&](uint32_t col, float* dst) {
#pragma unroll
        for (int sub = 0; sub < Cfg::kBoxes; ++sub) {
          const int c0 = Cfg::kHeadDim / 2 * half + 32 * sub;
          uint32_t a[16];
          tmem_ld_16x256b_sync(tmem + lb + col + c0, a);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float* at = dst + (slice + gq + 8 * r) * Cfg::kHeadDim + c0 + 2 * q;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float2*>(at + 8 * i) =
                  make_float2(__uint_as_float(a[4 * i + 2 * r]),
                              __uint_as_float(a[4 * i + 2 * r + 1]));
          }
        }
      };
      if constexpr (Cfg::kBoth) {
        keep_acc(Cfg::kColAcc1, part);
        keep_acc(Cfg::kColAcc0, part + Cfg::kRows * Cfg::kHeadDim);
      } else {
        keep_acc(Cfg::kColAcc0, part);
      }
    } else if constexpr (Cfg::kBoth) {
      stage_acc(Cfg::kColAcc1, p.scale, res);                    // dK over the k tile
      stage_acc(Cfg::kColAcc0, 1.0f, res + Cfg::kTileBytes);     // dV over the v tile
    } else if constexpr (Cfg::kSplit) {
      write_acc(Cfg::kColAcc0, Cfg::kOnlyDV ? 1.0f : p.scale);
    } else {
      stage_acc(Cfg::kColAcc0, p.scale, res);                    // dQ over the q tile
    }
    tc_fence_before();
    if constexpr (!Cfg::kSplit) {
      fence_proxy_async_smem();
      __syncwarp();
      // staging rows written: the store warp takes the unit from here (bwd_store_role)
      if (lane == 0) mbar_arrive(bar(Cfg::kBarStage));
    }
    cur.next_unit(p);
  }
}

// One thread of the store warp: once the 16 softmax-side warps have staged a unit's gradients
// in its resident buffers, store them with TMA and free the buffers for the load warp when
// the stores have read them; the softmax-side warps go straight on to the next unit.
template <class Cfg>
__device__ __forceinline__ void bwd_store_role(const BwdParams& p, uint8_t* smem, uint32_t bars,
                                               const Watchdog& wd, const BwdClaims& claims) {
  auto bar = [&](int idx) { return bars + 8u * static_cast<uint32_t>(idx); };
  typename Cfg::Cursor cur;
  cur.init(p, claims, BwdRole::kLane);
  int stores = 0;
  while (cur.valid()) {
    const int b = Cfg::res_buffer(cur.seg);
    if (!wait_single(bar(Cfg::kBarStage), static_cast<uint32_t>(stores) & 1u, wd, kSiteSoftStage))
      break;
    uint8_t* res = smem + Cfg::kResOff + b * 2 * Cfg::kTileBytes;
    if (!cur.in_pieces()) {
      const int r0 = cur.row_block(p) * Cfg::kRows;
      const HeadBatch hb = cur.resident(p);
      tma_store_4d(&p.tm_o0, smem_addr(res), 0, r0, hb.h, hb.b);
      if (Cfg::kBoth) tma_store_4d(&p.tm_o1, smem_addr(res + Cfg::kTileBytes), 0, r0, hb.h, hb.b);
      tma_store_commit();
      tma_store_wait_read();
    }
    mbar_arrive(bar(Cfg::kBarResEmpty + b));
    ++stores;
    cur.next_unit(p);
  }
  // unwinding or done: shared memory must outlive every store's read of it
  tma_store_wait_read();
}

// The barriers of a CTA, initialised by one thread (the indices are those of all its passes).
template <class Cfg>
__device__ __forceinline__ void bwd_init_bars(uint32_t bars) {
  for (int b = 0; b < 2; ++b) {
    mbar_init(bars + 8 * (Cfg::kBarResFull + b), 1);
    mbar_init(bars + 8 * (Cfg::kBarResEmpty + b), 1);
  }
  for (int s = 0; s < Cfg::STAGES; ++s) {
    mbar_init(bars + 8 * (Cfg::kBarStrFull + s), 1);
    // both MMA issuers read the stage (the dV pass's late tile: the accumulation alone)
    mbar_init(bars + 8 * (Cfg::kBarStrEmpty + s), Cfg::kOnlyDV ? 1 : 2);
  }
  if constexpr (Cfg::kSplit) {
    for (int s = 0; s < 3; ++s) {
      mbar_init(bars + 8 * (Cfg::kBarEarlyFull + s), 1);
      mbar_init(bars + 8 * (Cfg::kBarEarlyEmpty + s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bars + 8 * (Cfg::kBarVecFull + s), 1);
      mbar_init(bars + 8 * (Cfg::kBarVecEmpty + s), 1);
    }
  }
  mbar_init(bars + 8 * Cfg::kBarSSFull, 1);
  mbar_init(bars + 8 * Cfg::kBarSSFree, Cfg::kSoftmaxWarps);
  mbar_init(bars + 8 * Cfg::kBarOpFull, Cfg::kSoftmaxWarps);
  mbar_init(bars + 8 * Cfg::kBarAccDone, 1);
  mbar_init(bars + 8 * Cfg::kBarStage, Cfg::kSoftmaxWarps);
  mbar_init(bars + 8 * Cfg::kBarDrain, 1);
  mbar_init(bars + 8 * (Cfg::kBarDrain + 1), 1);
  if constexpr (Cfg::kWindow) {
    for (int i = 0; i < Cfg::kClaims; ++i) {
      mbar_init(bars + 8 * (Cfg::kBarClaimFull + i), 1);
      mbar_init(bars + 8 * (Cfg::kBarClaimEmpty + i), Cfg::kClaimReaders);
    }
  }
  mbar_init_fence();
}

// One CTA: the units of pass CA (params pa), then, with kPasses > 1, those of pass CB (params pb),
// then, with 3, those of CC (pc). Between the passes every role has finished (the MMA warps drain
// their commits, the store thread waits for its stores' shared-memory reads), the CTA meets on
// named barrier 2 and the barriers start afresh; TMEM stays allocated. The barriers live past all
// passes' shared-memory layouts. Each role's calls stay inside its setmaxnreg branch, which is what
// lets the register allocator give the softmax-side warps their 104 registers.
template <class CA, class CB, class CC, int kPasses>
__device__ __forceinline__ void bwd_cta(const BwdParams& pa, const BwdParams& pb,
                                        const BwdParams& pc) {
  static_assert(CA::kNumBars == CB::kNumBars && CA::kThreads == CB::kThreads &&
                    CA::kTmemCols == CB::kTmemCols && CA::kNumBars == CC::kNumBars &&
                    CA::kThreads == CC::kThreads && CA::kTmemCols == CC::kTmemCols,
                "passes of one CTA share barriers, threads and TMEM");
  constexpr int kBarOff2 = CA::kBarOff > CB::kBarOff ? CA::kBarOff : CB::kBarOff;
  constexpr int kBarOff = kBarOff2 > CC::kBarOff ? kBarOff2 : CC::kBarOff;
  constexpr int kTmemSlotOff = kBarOff + CA::kNumBars * 8;
  constexpr int kAbortOff = kTmemSlotOff + 4;
  constexpr int kRingBytes = CA::kWindow ? 4 * CA::kClaims : 0;
  constexpr int kSmem2 = CA::kSmemBytes > CB::kSmemBytes ? CA::kSmemBytes : CB::kSmemBytes;
  static_assert(kAbortOff + 4 + kRingBytes + 1024 <=
                    (kSmem2 > CC::kSmemBytes ? kSmem2 : CC::kSmemBytes),
                "barriers inside the launch's shared memory");
  static_assert(CA::kSplit == CB::kSplit && CA::kSplit == CC::kSplit &&
                    (!CA::kSplit || (CA::kBarOff == CB::kBarOff && CA::kBarOff == CC::kBarOff)),
                "passes of one CTA share the header");
  uint8_t* smem;
  if constexpr (CA::kSplit) {
    extern __shared__ __align__(1024) uint8_t smem_aligned[];
    smem = smem_aligned;
  } else {
    extern __shared__ uint8_t smem_raw[];
    smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                      ~static_cast<uintptr_t>(1023));
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t bars = smem_addr(smem + kBarOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kTmemSlotOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kAbortOff);
  volatile int* ring = reinterpret_cast<volatile int*>(smem + kAbortOff + 4);
  if (CA::kWindow && threadIdx.x == 0) grid_dependents_launch();  // the reduce kernel, which waits
  // Between the passes: true if the next pass runs (the same verdict in every thread:
  // nothing writes the flag between the two barriers).
  auto next_pass = [&](auto config) -> bool {
    __syncwarp();
    tc_fence_before();
    named_bar_sync(2, CA::kThreads);
    tc_fence_after();
    const bool go = *abort_flag == 0;
    if (go && warp == CA::kLoadWarp && lane == 0) {
      for (int i = 0; i < CA::kNumBars; ++i) mbar_inval(bars + 8 * i);
      bwd_init_bars<decltype(config)>(bars);
    }
    named_bar_sync(2, CA::kThreads);
    return go;
  };
  // As in the forward kernel: the load thread initialises the barriers and goes straight on
  // to its first copies; the other warps wait on named barrier 1 for the barriers and warp
  // 0's TMEM allocation (the load warp only arrives there).
  uint32_t tmem = 0;
  if (warp == CA::kLoadWarp) {
    if (lane == 0) {
      *abort_flag = 0;
      bwd_init_bars<CA>(bars);
    }
    __syncwarp();
    named_bar_arrive(1, CA::kThreads);
    setmaxnreg_dec<CA::kControlRegs>();
    if constexpr (CA::kWindow) grid_dependency_wait();
    const Watchdog wd{abort_flag, pa.status, pa.timeout_ns};
    const BwdClaims claims{ring, bars, &wd};
    if (lane == 0) bwd_load_role<CA>(pa, smem, bars, wd, claims);
    if constexpr (kPasses > 1) {
      const bool go = next_pass(CB{});
      if (go && lane == 0) bwd_load_role<CB>(pb, smem, bars, wd, claims);
      if constexpr (kPasses > 2) {
        if (go && next_pass(CC{}) && lane == 0) bwd_load_role<CC>(pc, smem, bars, wd, claims);
      }
    }
  } else {
    if (warp == 0) {
      tmem_alloc(smem_addr(tmem_slot), CA::kTmemCols);
      tmem_relinquish();
    }
    tc_fence_before();
    named_bar_sync(1, CA::kThreads);
    tc_fence_after();
    tmem = *tmem_slot;
    // window variant: a programmatic dependent of the row pass, as the forward kernel is of the
    // stream's previous kernel
    if constexpr (CA::kWindow) grid_dependency_wait();
    const Watchdog wd{abort_flag, pa.status, pa.timeout_ns};
    const BwdClaims claims{ring, bars, &wd};
    if (warp < CA::kSoftmaxWarps) {
      setmaxnreg_inc<CA::kSoftmaxRegs>();
      bwd_softmax_role<CA>(pa, smem, bars, tmem, wd, claims);
      if constexpr (kPasses > 1) {
        if (next_pass(CB{})) {
          bwd_softmax_role<CB>(pb, smem, bars, tmem, wd, claims);
          if constexpr (kPasses > 2) {
            if (next_pass(CC{})) bwd_softmax_role<CC>(pc, smem, bars, tmem, wd, claims);
          }
        }
      }
    } else {
      setmaxnreg_dec<CA::kControlRegs>();
      if (warp == CA::kMmaWarp) {
        bwd_mma_role<CA, false>(pa, smem, bars, tmem, wd, claims);
      } else if (warp == CA::kAccWarp) {
        bwd_mma_role<CA, true>(pa, smem, bars, tmem, wd, claims);
      } else if (warp == CA::kStoreWarp) {
        if (!CA::kSplit && lane == 0) bwd_store_role<CA>(pa, smem, bars, wd, claims);
      }
      if constexpr (kPasses > 1) {
        if (next_pass(CB{})) {
          if (warp == CB::kMmaWarp) {
            bwd_mma_role<CB, false>(pb, smem, bars, tmem, wd, claims);
          } else if (warp == CB::kAccWarp) {
            bwd_mma_role<CB, true>(pb, smem, bars, tmem, wd, claims);
          } else if (warp == CB::kStoreWarp) {
            if (!CB::kSplit && lane == 0) bwd_store_role<CB>(pb, smem, bars, wd, claims);
          }
          if constexpr (kPasses > 2) {
            if (next_pass(CC{})) {
              if (warp == CC::kMmaWarp) {
                bwd_mma_role<CC, false>(pc, smem, bars, tmem, wd, claims);
              } else if (warp == CC::kAccWarp) {
                bwd_mma_role<CC, true>(pc, smem, bars, tmem, wd, claims);
              } else if (warp == CC::kStoreWarp) {
                if (!CC::kSplit && lane == 0) bwd_store_role<CC>(pc, smem, bars, wd, claims);
              }
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, CA::kTmemCols);
}

// Both passes in one launch, at the same time on separate SMs: CTAs [0, pkv.cta0) run the dQ
// pass, the rest the dK/dV pass. Used when each pass has fewer units than about two per SM.
template <bool kCausal, bool kBF16>
__global__ void __launch_bounds__(BwdConfig<true, kCausal, kBF16>::kThreads, 1)
    mfa_bwd_kernel(const __grid_constant__ BwdParams pq, const __grid_constant__ BwdParams pkv) {
  using CQ = BwdConfig<false, kCausal, kBF16>;
  using CK = BwdConfig<true, kCausal, kBF16>;
  if (static_cast<int>(blockIdx.x) < pkv.cta0)
    bwd_cta<CQ, CQ, CQ, 1>(pq, pq, pq);
  else
    bwd_cta<CK, CK, CK, 1>(pkv, pkv, pkv);
}

// Both passes in one launch, every CTA on both: its dK/dV units first, then its dQ units,
// dealt from the other end of the grid (pq.reverse), so that the CTAs with one dK/dV unit
// more than the others have none of the extra dQ units. Used when a pass has a few units
// per SM: 512 units per pass on 148 SMs take 4 dK/dV + 3 dQ units on the slowest CTA, where
// separate SMs per pass take 7 dK/dV units (a dK/dV step costs more than a dQ step).
template <bool kCausal, bool kBF16>
__global__ void __launch_bounds__(BwdConfig<true, kCausal, kBF16>::kThreads, 1)
    mfa_bwd_mixed_kernel(const __grid_constant__ BwdParams pq,
                         const __grid_constant__ BwdParams pkv) {
  using CQ = BwdConfig<false, kCausal, kBF16>;
  bwd_cta<BwdConfig<true, kCausal, kBF16>, CQ, CQ, 2>(pkv, pq, pq);
}

// Window variant: every CTA on both passes, dK/dV units first (they are the longer ones), each
// unit claimed from the pass's counter.
template <bool kBF16>
__global__ void __launch_bounds__(BwdConfig<true, true, kBF16, true>::kThreads, 1)
    mfa_bwd_window_kernel(const __grid_constant__ BwdParams pq,
                          const __grid_constant__ BwdParams pkv) {
  using CQ = BwdConfig<false, true, kBF16, true>;
  bwd_cta<BwdConfig<true, true, kBF16, true>, CQ, CQ, 2>(pkv, pq, pq);
}

// D = 128: dK, dV and dQ in a pass each (the dV pass without dP): eight products a step where five
// would do, but S, dP, both operands and both accumulators of dK and dV are 640 columns of TMEM.
// Measured at 16 query heads x 8192 over 4 k / v heads, window 2048, 16 sinks, bf16: 449 us, 1079
// TFLOP/s over the eight products (674 over five); D = 64 278 us (545 over five).
template <bool kBF16>
using BwdDK128 = BwdConfig<true, true, kBF16, true, 128, BwdPart::kDK>;
template <bool kBF16>
using BwdDV128 = BwdConfig<true, true, kBF16, true, 128, BwdPart::kDV>;
template <bool kBF16>
using BwdDQ128 = BwdConfig<false, true, kBF16, true, 128>;

template <bool kBF16>
__global__ void __launch_bounds__(BwdDQ128<kBF16>::kThreads, 1)
    mfa_bwd_window128_kernel(const __grid_constant__ BwdParams pq,
                             const __grid_constant__ BwdParams pk,
                             const __grid_constant__ BwdParams pv) {
  bwd_cta<BwdDK128<kBF16>, BwdDV128<kBF16>, BwdDQ128<kBF16>, 3>(pk, pv, pq);
}

// dK and dV of the blocks whose units ran in pieces: the sum of the pieces in order, dK scaled. The
// pieces of slot i are at dk_sums and dv_sums + i * slot_floats. One CTA per 1024 / D rows of a
// (block, k / v head row) pair that may have pieces, sink blocks first; D / 4 threads a row, four
// columns each, of the tensors' `cols`. The pieces are read four at a time (an L2 round trip each).
// (16 heads x 8192, 16 sinks, D = 64: 4 blocks of 4 pieces, 3 us behind the passes; one CTA a block
// took 9.)
template <bool kBF16, int kD>
__global__ void __launch_bounds__(256)
    mfa_bwd_reduce_kernel(const BwdParams p, const float* dk_sums, const float* dv_sums,
                          long long slot_floats, int cols, uint16_t* dk, uint16_t* dv,
                          long long stride_b, long long stride_h, long long stride_n) {
  constexpr int kRows = 1024 / kD, kCtas = 128 / kRows;
  grid_dependency_wait();
  const int pair = static_cast<int>(blockIdx.x) / kCtas;
  const int blk = pair / p.bh, row = pair % p.bh;
  const bool sink = blk < p.sink_blocks;
  const int span = BwdWindowCursor<BwdConfig<true, true, kBF16, true>>::span(p, blk);
  const int chunk = sink ? p.chunk_sink : p.chunk_rest;
  const int count = (span * p.group + chunk - 1) / chunk;
  if (count < 2) return;
  // unit index of the pair's piece 0; its pieces are p.bh apart
  const long long first =
      sink ? static_cast<long long>(blk) * p.bh * p.pieces_sink + row
           : static_cast<long long>(p.sink_blocks) * p.bh * p.pieces_sink +
                 static_cast<long long>(blk - p.sink_blocks) * p.bh * p.pieces_rest + row;
  const long long base =
      static_cast<long long>(row / p.heads) * stride_b + (row % p.heads) * stride_h;
  const int col = 4 * (threadIdx.x % (kD / 4));
  const int r = static_cast<int>(blockIdx.x) % kCtas * kRows + threadIdx.x / (kD / 4);
  if (blk * 128 + r < p.n && col < cols) {
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const long long at = (first + static_cast<long long>(i) * p.bh) * slot_floats + r * kD + col;
      const float4 a = *reinterpret_cast<const float4*>(dk_sums + at);
      const float4 b = *reinterpret_cast<const float4*>(dv_sums + at);
      k.x += a.x, k.y += a.y, k.z += a.z, k.w += a.w;
      v.x += b.x, v.y += b.y, v.z += b.z, v.w += b.w;
    }
    const long long off = base + static_cast<long long>(blk * 128 + r) * stride_n + col;
    *reinterpret_cast<uint2*>(dk + off) =
        make_uint2(pack_pair<kBF16>(k.x * p.scale, k.y * p.scale),
                   pack_pair<kBF16>(k.z * p.scale, k.w * p.scale));
    *reinterpret_cast<uint2*>(dv + off) =
        make_uint2(pack_pair<kBF16>(v.x, v.y), pack_pair<kBF16>(v.z, v.w));
  }
}

// One pass per launch (many units per SM), all CTAs on it; a kernel of its own, which measured
// 2-5% faster than the two-pass kernel above run with all CTAs on one pass.
template <bool kDKV, bool kCausal, bool kBF16>
__global__ void __launch_bounds__(BwdConfig<kDKV, kCausal, kBF16>::kThreads, 1)
    mfa_bwd_pass_kernel(const __grid_constant__ BwdParams p) {
  using C = BwdConfig<kDKV, kCausal, kBF16>;
  bwd_cta<C, C, C, 1>(p, p, p);
}

// Dynamic shared memory of the two-pass launch.
template <bool kCausal, bool kBF16>
constexpr int bwd_smem_bytes() {
  return BwdConfig<false, kCausal, kBF16>::kSmemBytes > BwdConfig<true, kCausal, kBF16>::kSmemBytes
             ? BwdConfig<false, kCausal, kBF16>::kSmemBytes
             : BwdConfig<true, kCausal, kBF16>::kSmemBytes;
}

// D_i = rowsum(dO ⊙ o) and L2_i = L_i * log2(e) for every row, into [bh][blocks * 128] arrays
// padded past N with D = 0, L2 = +inf (so that padded queries get P = 0 in the dK/dV pass).
// D / 8 threads per row (16 bytes each), grid-stride. `rest` is what the rounding of o left, of the
// first rest_rows (0: none) rows of every head: dP - D is a difference, in which the rounding of o
// weighs most where few keys are visible. (Errors of dq over those of rounding it alone, normal
// inputs, D = 64, without the rest and with it: 2.2 and 1.48 in rows that see two to four keys, 1.61 and
// 1.46 up to 16, 1.49 and 1.45 up to 64, 1.45 and 1.44 beyond, at any length. The rounding of dS alone
// makes 1.41, that of P for o most of what is left.)
template <bool kBF16, bool kWindow = false, int kD = 64>
__global__ void __launch_bounds__(256) mfa_bwd_prep_kernel(const void* o, const void* dout,
                                                           const float* lse, float* lse2,
                                                           float* di, int bh, int n, int heads,
                                                           long long stride_b, long long stride_h,
                                                           long long stride_n, int blocks,
                                                           int* counters = nullptr,
                                                           const void* rest = nullptr,
                                                           int rest_rows = 0,
                                                           long long rest_b = 0,
                                                           long long rest_h = 0,
                                                           long long rest_n = 0) {
  if constexpr (kWindow) {
    // a programmatic dependent, as is the kernel after it; the passes' unit counters start at 0
    if (threadIdx.x == 0) grid_dependents_launch();
    grid_dependency_wait();
    if (blockIdx.x == 0 && threadIdx.x < 3) counters[threadIdx.x] = 0;
  }
  constexpr int kLanes = kD / 8, kRows = 32 / kLanes;  // threads of a row, rows of a warp
  const long long rows = static_cast<long long>(bh) * blocks * 128;  // a multiple of kRows
  const int sub = threadIdx.x & (kLanes - 1);
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  // kRows rows per warp and iteration; the trip count is the same for the whole warp
  for (long long w = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
       w * kRows < rows; w += warps) {
    const long long r = w * kRows + (threadIdx.x & 31) / kLanes;
    const int h = static_cast<int>(r / (static_cast<long long>(blocks) * 128));
    const int row = static_cast<int>(r - static_cast<long long>(h) * blocks * 128);
    float acc = 0.0f;
    if (row < n) {
      const long long off = static_cast<long long>(h / heads) * stride_b +
                            static_cast<long long>(h % heads) * stride_h +
                            static_cast<long long>(row) * stride_n + 8 * sub;
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(o) + off);
      const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(dout) + off);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
      uint4 c = make_uint4(0u, 0u, 0u, 0u);
      if (kWindow && row < rest_rows)
        c = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(rest) +
                                            h / heads * rest_b + h % heads * rest_h +
                                            row * rest_n + 8 * sub);
      [[maybe_unused]] const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a0, a1, b0, b1;
        unpack_pair<kBF16>(aw[e], a0, a1);
        unpack_pair<kBF16>(bw[e], b0, b1);
        if constexpr (kWindow) {
          float c0, c1;
          unpack_pair<kBF16>(cw[e], c0, c1);
          a0 += c0;
          a1 += c1;
        }
        acc = fmaf(a0, b0, fmaf(a1, b1, acc));
      }
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (sub == 0) {
      di[r] = row < n ? acc : 0.0f;
      lse2[r] = row < n ? lse[static_cast<long long>(h) * n + row] * 1.4426950408889634f
                        : INFINITY;
    }
  }
}

}  // namespace mfa
