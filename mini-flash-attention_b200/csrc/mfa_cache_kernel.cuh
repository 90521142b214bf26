// Extending a paged key / value cache: pages and slots for new tokens, and the copy of their k and v.
#pragma once

#include <cstdint>

#include "mfa_ptx.cuh"
#include "mfa_schedule.cuh"

namespace mfa {

// Request r has cached[r] tokens, in the first ceil(cached / page_size) pages of its table row,
// and gets added[r] new ones. With F(r) = the pages that it needs beyond those,
//   table[r][have + i] = free_pages[sum of F over the requests before r + i],   i < F(r)
//   slots[sum of added over the requests before r + i] = page * page_size + row
// of the token at position cached[r] + i, and -1 behind the last token. A token whose page would
// lie past the row's last column or the last free page gets the slot -1 (and such a page -1).
struct ExtendParams {
  int* table;  // [batch, columns]
  const int* cached;
  const int* added;
  const int* free_pages;
  int batch, columns, free_count, page_size;
  int* slots;
  int capacity;
  int* starts;  // [batch + 1]: each request's first token in slots
  int* used;    // pages taken from free_pages
};

constexpr int kExtendThreads = 256;

// Every CTA scans all requests, kExtendThreads at a time (each chunk's sums in shared memory), and
// fills its share of the chunk's pages and tokens, whose requests it finds by bisection: no second
// launch for the sums, and the work is even however uneven the requests are. Entries of the table
// are read in the columns below ceil(cached / page_size) and written from there on. B200: 3.7 us for
// 256 requests of one token, 4.7 us for 33 requests of 46 thousand; latencies bound it (lengths,
// bisection, table or list).
__global__ void __launch_bounds__(kExtendThreads) mfa_extend_kernel(const ExtendParams p) {
  constexpr int kN = kExtendThreads;
  __shared__ long long token0[kN + 1];  // first token, first free page of the chunk's requests
  __shared__ long long page0[kN + 1];
  __shared__ long long warp_tokens[kN / 32], warp_pages[kN / 32];
  __shared__ int length[kN];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long at = static_cast<long long>(blockIdx.x) * kN + tid;
  const long long step = static_cast<long long>(gridDim.x) * kN;
  const int page_size = p.page_size;
  if (tid == 0) grid_dependents_launch();  // the copy may be set up, and waits
  grid_dependency_wait();
  long long tokens = 0, pages = 0;  // of the chunks before
  auto saturate = [](long long x) { return static_cast<int>(x < 0x7fffffff ? x : 0x7fffffff); };
  auto columns_of = [&](long long n) {  // pages of n tokens, as many as a row has
    const long long c = (n + page_size - 1) / page_size;
    return c < p.columns ? static_cast<int>(c) : p.columns;
  };
  for (int r0 = 0; r0 < p.batch; r0 += kN) {
    const int r = r0 + tid;
    int c = 0, a = 0;
    if (r < p.batch) {
      c = p.cached[r] > 0 ? p.cached[r] : 0;
      a = p.added[r] > 0 ? p.added[r] : 0;
    }
    const long long fresh = columns_of(static_cast<long long>(c) + a) - columns_of(c);
    long long t = a, f = fresh;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, t, o);
      const long long y = __shfl_up_sync(0xffffffffu, f, o);
      if (lane >= o) {
        t += x;
        f += y;
      }
    }
    __syncthreads();  // the chunk before is done with
    if (lane == 31) {
      warp_tokens[warp] = t;
      warp_pages[warp] = f;
    }
    length[tid] = c;
    __syncthreads();
    long long before_t = tokens, before_f = pages;
#pragma unroll
    for (int w = 0; w < kN / 32; ++w) {
      if (w < warp) {
        before_t += warp_tokens[w];
        before_f += warp_pages[w];
      }
    }
    token0[tid] = before_t + t - a;
    page0[tid] = before_f + f - fresh;
    if (tid == kN - 1) {
      token0[kN] = before_t + t;
      page0[kN] = before_f + f;
    }
    __syncthreads();
    if (blockIdx.x == 0 && r < p.batch) p.starts[r + 1] = saturate(token0[tid + 1]);
    // the last request whose first index is not after i: the one that owns it
    auto owner = [&](const long long* first, long long i) {
      int lo = 0;
#pragma unroll
      for (int s = kN / 2; s > 0; s >>= 1)
        if (first[lo + s] <= i) lo += s;
      return lo;
    };
    for (long long i = page0[0] + at; i < page0[kN]; i += step) {
      const int o = owner(page0, i);
      const int column = columns_of(length[o]) + static_cast<int>(i - page0[o]);
      p.table[static_cast<size_t>(r0 + o) * p.columns + column] =
          i < p.free_count ? p.free_pages[i] : -1;
    }
    const long long end = token0[kN] < p.capacity ? token0[kN] : p.capacity;
    for (long long i = token0[0] + at; i < end; i += step) {
      const int o = owner(token0, i);
      const long long pos = length[o] + (i - token0[o]);
      const long long column = pos / page_size;
      const int have = columns_of(length[o]);
      int page = -1;
      if (column < have) {
        page = p.table[static_cast<size_t>(r0 + o) * p.columns + column];
      } else if (column < p.columns) {
        const long long from = page0[o] + (column - have);
        if (from < p.free_count) page = p.free_pages[from];
      }
      const long long slot = static_cast<long long>(page) * page_size + (pos - column * page_size);
      p.slots[i] = page < 0 || slot > 0x7fffffff ? -1 : static_cast<int>(slot);
    }
    tokens = token0[kN];
    pages = page0[kN];
  }
  for (long long i = tokens + at; i < p.capacity; i += step) p.slots[i] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[0] = 0;
    p.used[0] = saturate(pages);
  }
}

// Token t's k and v rows go to slot slots[t] of the caches ([pages, kv_heads, page_size, d]); a slot
// outside them is skipped.
struct AppendParams {
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* k_cache;
  uint16_t* v_cache;
  const int* slots;
  long long k_token, k_head, v_token, v_head;  // strides in elements
  int tokens, kv_heads, d;
  int page_size;
  long long slot_count;
  int tokens_a_block;
  Div31 by_chunks, by_heads, by_page;  // d / 8, kv_heads, page_size
};

// A copy, bound by HBM: 16 bytes of k and of v a thread and item, neighbouring threads along a row,
// four items' loads in flight at a time. B200: 46 thousand tokens of 8 heads of 64, 184 MB in and out,
// 31.8 us (5.8 TB/s; 33.7 with one item after the other); 256 tokens 2.1 us.
__global__ void __launch_bounds__(256) mfa_append_kernel(const AppendParams p) {
  constexpr int kBatch = 4;
  if (threadIdx.x == 0) grid_dependents_launch();
  grid_dependency_wait();
  const int chunks = p.d / 8;
  const int t0 = static_cast<int>(blockIdx.x) * p.tokens_a_block;
  const int count = p.tokens - t0 < p.tokens_a_block ? p.tokens - t0 : p.tokens_a_block;
  const int items = count * p.kv_heads * chunks;
  for (int i0 = threadIdx.x; i0 < items; i0 += 256 * kBatch) {
    uint4 x[kBatch], y[kBatch];
    long long to[kBatch];
    int slot[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + 256 * b;
      slot[b] = i < items ? p.slots[t0 + static_cast<int>(p.by_heads(p.by_chunks(i)))] : -1;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + 256 * b;
      to[b] = -1;
      if (slot[b] < 0 || slot[b] >= p.slot_count) continue;
      const int row = static_cast<int>(p.by_chunks(i));
      const int in = static_cast<int>(p.by_heads(row));
      const int c = 8 * (i - row * chunks), h = row - in * p.kv_heads;
      const long long t = t0 + in;
      const int page = static_cast<int>(p.by_page(slot[b]));
      x[b] = *reinterpret_cast<const uint4*>(p.k + t * p.k_token + h * p.k_head + c);
      y[b] = *reinterpret_cast<const uint4*>(p.v + t * p.v_token + h * p.v_head + c);
      to[b] = ((static_cast<long long>(page) * p.kv_heads + h) * p.page_size + slot[b] -
               page * p.page_size) * p.d + c;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (to[b] < 0) continue;
      *reinterpret_cast<uint4*>(p.k_cache + to[b]) = x[b];
      *reinterpret_cast<uint4*>(p.v_cache + to[b]) = y[b];
    }
  }
}

}  // namespace mfa
