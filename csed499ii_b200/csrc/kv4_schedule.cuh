// Block tables and slots of a serving step, from the requests' lengths.
//
// Everything a step has to know follows from three prefix sums over the
// requests: of their new tokens (which row belongs to whom), of the pages
// that ended requests give back, and of the pages that growing requests need.
// Every CTA makes the three sums of all requests itself (a few KB that sit in
// L2) and then fills its share of the rows and of the tables, so nothing is
// handed from CTA to CTA and one launch does it all.  Pages that are given
// back and handed out in the same step are looked up where they lie (in the
// ended request's table row): no CTA reads what another writes.
//
// Latency bounds it: loads, two scans of the block, a search for a row's request
// and a page's entry one after another.  A step of 8 requests takes 3.6 us on the
// GPU (a launch alone about 2.2), 500 requests with 9000 rows 6.2 us: 14 us with a
// CTA for 2048 rows, 64-bit divisions and twelve barriers instead of three.  Where
// the lengths or the count are updated in place one CTA does it all: 4.7 us, 23.5,
// and 60 for 64 prompts with 65536 rows that take 4.1 otherwise.
#pragma once

#include <stdint.h>

#include "device_primitives.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kScheduleThreads = 512;
constexpr int kMaxBatch = 8192;  // requests of a step: 20 bytes of shared memory each

struct ScheduleParams {
  const int* new_lens;   // tokens of this step; negative: the request has ended
  const int* lens;       // tokens in the cache
  int* tables;           // [batch][table_stride], `width` entries used
  int64_t table_stride;
  int width;
  int batch;
  int* free_pages;       // a stack: entries [0, *free_count) are free, the last is its top
  int capacity;
  const int* free_count;
  int rows;
  int page_size;
  int* lens_out;
  int* free_count_out;
  int* starts;           // [batch + 1]
  int* slots;            // [rows]
  int* positions;        // [rows]
  int* fate;             // [batch]
};

enum : int { kFateOk = 0, kFateNoPages = 1, kFateTable = 2, kFateRows = 3 };

// Inclusive prefix sums of `x` over the block, in thread order, and its sums.
// `warp_sums` is another buffer than the last call's.
template <int N>
__device__ __forceinline__ void block_scan(int64_t (&x)[N], int64_t (&total)[N],
                                           int64_t (*warp_sums)[kScheduleThreads / 32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x[n], s);
      if (lane >= s) x[n] += y;
    }
    if (lane == 31) warp_sums[n][warp] = x[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    total[n] = 0;
#pragma unroll
    for (int w = 0; w < kScheduleThreads / 32; ++w) {
      if (w == warp) x[n] += total[n];
      total[n] += warp_sums[n][w];
    }
  }
}

// Pages of `tokens` tokens.
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page) {
  const uint32_t n = tokens / page;
  return n + (n * page != tokens);
}

// First index whose (ascending) entry is above `x`; n if there is none.
__device__ __forceinline__ int upper_bound(const int* a, int n, int x) {
  int lo = 0;
  while (n > 0) {
    const int half = n >> 1;
    if (a[lo + half] <= x) {
      lo += half + 1;
      n -= half + 1;
    } else {
      n = half;
    }
  }
  return lo;
}

__device__ __forceinline__ int clamp_int(int64_t x) {
  return x > 0x7fffffff ? 0x7fffffff : static_cast<int>(x);
}

__global__ void __launch_bounds__(kScheduleThreads)
    kv4_schedule_kernel(const __grid_constant__ ScheduleParams p) {
  extern __shared__ int schedule_smem[];
  __shared__ int64_t warp_sums[2][2][kScheduleThreads / 32];
  __shared__ int granted;
  int* ends = schedule_smem;       // new tokens up to and with the request
  int* backs = ends + p.batch;     // pages given back up to and with it
  int* needs = backs + p.batch;    // pages needed by the requests before it
  int* grants = needs + p.batch;   // pages it gets, or -1 - fate where it is refused
  int* lens = grants + p.batch;    // tokens in the cache (lens_out may be the same array as lens)
  grid_dependency_wait();
  grid_dependency_launch();
  const int count = min(max(*p.free_count, 0), p.capacity);
  const uint32_t page = p.page_size;
  if (threadIdx.x == 0) granted = 0;

  int64_t end0 = 0, back0 = 0;
  int turn = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kScheduleThreads) {
    const int b = b0 + threadIdx.x;
    int64_t x[2] = {0, 0}, all[2];
    if (b < p.batch) {
      const int asked = p.new_lens[b];
      const int len = lens[b] = max(p.lens[b], 0);
      x[0] = max(asked, 0);
      if (asked < 0) x[1] = min(pages_of(len, page), static_cast<uint32_t>(p.width));
      grants[b] = asked;
    }
    block_scan(x, all, warp_sums[turn ^= 1]);
    if (b < p.batch) {
      ends[b] = clamp_int(end0 + x[0]);
      backs[b] = clamp_int(back0 + x[1]);
      if (blockIdx.x == 0) p.starts[b + 1] = ends[b];
    }
    end0 += all[0];
    back0 += all[1];
  }
  const int64_t full = count + back0;  // free pages once the ended requests' are back

  // A request that comes too late for its pages leaves those after it none: the
  // sum of all needs before it only grows, and what is granted is the largest
  // that the pages reach.
  int64_t need0 = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kScheduleThreads) {
    const int b = b0 + threadIdx.x;
    int64_t need = 0;
    int fate = kFateOk, asked = 0, len = 0;
    if (b < p.batch) {
      asked = grants[b];
      len = lens[b];
      if (asked > 0) {
        const uint32_t wanted = pages_of(static_cast<uint32_t>(len) + asked, page);
        if (ends[b] > p.rows) {
          fate = kFateRows;
        } else if (wanted > static_cast<uint32_t>(p.width)) {
          fate = kFateTable;
        } else {
          need = wanted - pages_of(len, page);
        }
      }
    }
    int64_t x[1] = {need}, all[1];
    block_scan(x, all, warp_sums[turn ^= 1]);
    const int64_t upto = need0 + x[0];
    need0 += all[0];
    if (need > 0 && upto > full) fate = kFateNoPages;
    if (b < p.batch) {
      needs[b] = clamp_int(upto - need);
      grants[b] = fate == kFateOk ? static_cast<int>(need) : -1 - fate;
      if (blockIdx.x == 0) {
        p.fate[b] = fate;
        p.lens_out[b] = asked < 0 ? 0 : fate == kFateOk ? clamp_int(static_cast<int64_t>(len) + asked) : len;
      }
    }
    const int most = __reduce_max_sync(0xffffffffu, upto <= full ? clamp_int(upto) : 0);
    if (blockIdx.x == 0 && (threadIdx.x & 31) == 0) atomicMax(&granted, most);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.starts[0] = 0;
    *p.free_count_out = clamp_int(full - granted);
  }

  // entry `i` of the stack with the given-back pages on it, in request and table order
  auto stack = [&](int64_t i) -> int {
    if (i < count) return p.free_pages[i];
    const int j = static_cast<int>(i - count);
    const int b = upper_bound(backs, p.batch, j);
    return p.tables[p.table_stride * b + (j - (b ? backs[b - 1] : 0))];
  };

  const int threads = gridDim.x * kScheduleThreads;
  const int thread = blockIdx.x * kScheduleThreads + threadIdx.x;
  for (int r = thread; r < p.rows; r += threads) {
    const int b = upper_bound(ends, p.batch, r);
    int slot = -1;
    uint32_t position = 0;
    if (b < p.batch) {
      const int len = lens[b];
      position = static_cast<uint32_t>(len) + (r - (b ? ends[b - 1] : 0));
      if (grants[b] >= 0) {
        const int entry = position / page, used = pages_of(len, page);
        const int id = entry < used ? p.tables[p.table_stride * b + entry]
                                    : stack(full - 1 - needs[b] - (entry - used));
        slot = id * page + position - entry * page;
      }
    }
    p.slots[r] = slot;
    p.positions[r] = clamp_int(position);
  }
  const int lane = threadIdx.x & 31;
  for (int b = thread >> 5; b < p.batch; b += threads >> 5) {
    const int back = backs[b] - (b ? backs[b - 1] : 0);
    for (int i = lane; i < back; i += 32) {
      const int64_t at = static_cast<int64_t>(count) + backs[b] - back + i;
      if (at < p.capacity) p.free_pages[at] = p.tables[p.table_stride * b + i];
    }
    if (grants[b] <= 0) continue;
    const int used = pages_of(lens[b], page);
    for (int i = lane; i < grants[b]; i += 32)
      p.tables[p.table_stride * b + used + i] = stack(full - 1 - needs[b] - i);
  }
}

}  // namespace kv4
}  // namespace sm100
