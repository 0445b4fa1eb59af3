// Attention over the 4-bit cache.
//
//   out[r, h] = sum_j softmax_j(scale q[r, h] . k[j, h / G]) v[j, h / G]
//
// over the keys j that row r's request holds, up to the row's own position
// and, with a window, no further back than that.
#pragma once

#include <math_constants.h>

#include "kv4_format.cuh"

namespace sm100 {
namespace kv4 {

struct AttentionParams {
  Cache cache;
  const uint8_t* q;      // element (row, head, c) at q_row * row + q_head * head + c
  int64_t q_row, q_head;
  uint8_t* out;          // [rows][q_heads][D]
  const int* tables;     // [batch][table_stride], `width` entries used
  int64_t table_stride;
  int width;
  const int* lens;       // tokens of each request in the cache, the step's own among them
  const int* starts;     // [batch + 1] first row of each request; null: row b is request b's
  int batch;
  int rows;
  int q_heads;
  int group;             // query heads per key/value head
  int window;            // 0: none
  float scale;
  int most;              // requests with at most this many query rows a group are left alone
};

// First index whose (ascending) entry is above `x`; n if there is none.
__device__ __forceinline__ int first_above(const int* a, int n, int x) {
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

// One CTA of four warps per row and query head; the warps take the tiles in
// turn and join their running maxima and sums at the end.
template <class T, int D>
__global__ void __launch_bounds__(128) kv4_attention_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int kPer = D / 32;
  __shared__ float qs[D];
  __shared__ float part[4][D + 2];
  const int row = blockIdx.x, qh = blockIdx.y, head = qh / p.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b = row, first = row, end = row + 1;
  if (p.starts) {
    b = first_above(p.starts + 1, p.batch, row);
    first = b < p.batch ? p.starts[b] : row;
    end = b < p.batch ? p.starts[b + 1] : row;
  }
  if (b >= p.batch || static_cast<int64_t>(end - first) * p.group <= p.most) return;
  const int64_t room = static_cast<int64_t>(p.width) * p.cache.page_size;
  const int len = b < p.batch ? static_cast<int>(min(static_cast<int64_t>(p.lens[b]), room)) : 0;
  const int position = len - (end - row);  // of this row
  const int to = min(position + 1, len);
  const int from = p.window ? max(0, position - p.window + 1) : 0;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + p.q_row * row + p.q_head * qh;
  for (int c = threadIdx.x; c < D; c += 128) qs[c] = T::up(q[c]).x;
  __syncthreads();
  float m = -CUDART_INF_F, l = 0.f, o[kPer] = {};
  const int token = lane & 15, half = lane >> 4;
  for (int t = from / kTile + warp; t * kTile < to; t += 4) {
    const int page = p.tables[p.table_stride * b + t * kTile / p.cache.page_size];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.cache.pages)) continue;
    const uint8_t* tile =
        p.cache.page_tiles<D>(page, head) + t * kTile % p.cache.page_size / kTile * tile_bytes(D);
    const float2 kp = T::up(*reinterpret_cast<const uint32_t*>(tile + off_k_pair(D, token)));
    float s = 0.f;
    for (int c = half * D / 2; c < (half + 1) * D / 2; ++c) {
      const uint32_t code = (tile[off_k(D, token) + c / 2] >> (c % 2 * 4)) & 15u;
      s += qs[c] * fmaf(static_cast<float>(code), kp.x, kp.y);
    }
    s += __shfl_xor_sync(0xffffffffu, s, 16);
    s *= p.scale;
    const int j = t * kTile + token;
    const bool seen = j >= from && j < to;
    float top = seen ? s : -CUDART_INF_F;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float m2 = fmaxf(m, top);
    const float base = m2 == -CUDART_INF_F ? 0.f : m2;
    const float keep = expf(m - base);
    const float w = seen ? expf(s - base) : 0.f;
    l = l * keep;
    m = m2;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] *= keep;
    for (int i = 0; i < kTile; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const int ji = t * kTile + i;
      if (ji < from || ji >= to) continue;  // whatever lies there
      l += wi;
      const float2 vp = T::up(*reinterpret_cast<const uint32_t*>(tile + off_v_pair(D, i)));
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int c = lane * kPer + x;
        const uint32_t code =
            (tile[off_v(D, i, c / (D / 8)) + c % (D / 8) / 2] >> (c % 2 * 4)) & 15u;
        o[x] += wi * fmaf(static_cast<float>(code), vp.x, vp.y);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < kPer; ++x) part[warp][lane * kPer + x] = o[x];
  if (lane == 0) part[warp][D] = m, part[warp][D + 1] = l;
  __syncthreads();
  float top = -CUDART_INF_F;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][D]);
  if (top == -CUDART_INF_F) top = 0.f;
  float sum = 0.f;
  for (int w = 0; w < 4; ++w) sum += part[w][D + 1] * expf(part[w][D] - top);
  const float over = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (static_cast<int64_t>(row) * p.q_heads + qh) * D;
  for (int c = threadIdx.x; c < D; c += 128) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += part[w][c] * expf(part[w][D] - top);
    out[c] = static_cast<uint16_t>(T::down(x * over, 0.f));
  }
}

}  // namespace kv4
}  // namespace sm100
