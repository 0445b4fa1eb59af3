// Writing keys and values into the 4-bit cache, and reading them back.
// The layout and the rounding are those of kv4_format.cuh.
//
// Both are bound by memory.  A group of D/8 lanes owns one row (one token, one
// head, keys or values): each lane holds 8 channels, 16 bytes, so a warp reads
// 512 contiguous bytes an instruction; the row's range is a shuffle reduction,
// and every lane's 8 codes are one 32-bit word of the tile.
#pragma once

#include <math_constants.h>

#include "kv4_format.cuh"

namespace sm100 {
namespace kv4 {

struct AppendParams {
  Cache cache;
  const uint8_t* k;      // element (token, head, c) at k_row * token + k_head * head + c
  const uint8_t* v;
  int64_t k_row, k_head, v_row, v_head;  // in elements
  const int* slots;      // page * page_size + place, or out of range: the row is skipped
  int tokens;
  int aligned;           // 1: every row of k and v starts on a 16-byte boundary
};

struct ReadParams {
  Cache cache;
  uint8_t* k;            // [tokens][heads][D]
  uint8_t* v;
  const int* slots;      // out of range: zeros
  int tokens;
};

// 8 channels as 4 words of two.
__device__ __forceinline__ uint4 load_8(const uint8_t* p, bool aligned) {
  if (aligned) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  uint4 x;
  x.x = e[0] | static_cast<uint32_t>(e[1]) << 16;
  x.y = e[2] | static_cast<uint32_t>(e[3]) << 16;
  x.z = e[4] | static_cast<uint32_t>(e[5]) << 16;
  x.w = e[6] | static_cast<uint32_t>(e[7]) << 16;
  return x;
}

template <class T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kLanes = D / 8;  // of a row
  const int lane = threadIdx.x & 31;
  const int sub = lane % kLanes;
  const int64_t rows = 2ll * p.tokens * p.cache.heads;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  // a warp's rows are adjacent; rows past the end repeat the last one without storing it
  const bool live = row < rows;
  const int64_t r = live ? row : rows - 1;
  const bool is_v = r & 1;
  const int token = static_cast<int>((r >> 1) / p.cache.heads);
  const int head = static_cast<int>((r >> 1) - static_cast<int64_t>(token) * p.cache.heads);
  const uint8_t* src = is_v ? p.v + 2 * (p.v_row * token + p.v_head * head)
                            : p.k + 2 * (p.k_row * token + p.k_head * head);
  const int slot = p.slots[token];
  const uint4 raw = load_8(src + 16 * sub, p.aligned);
  float x[8];
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::up(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
  float lo = x[0], hi = x[0];
  bool odd = false;  // an infinity or a NaN
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    odd |= !(fabsf(x[i]) <= 3.402823466e38f);
  }
#pragma unroll
  for (int s = kLanes / 2; s > 0; s >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
  }
  const uint32_t group = ((kLanes == 32 ? 0u : (1u << kLanes)) - 1u) << (lane - sub);
  odd = (__ballot_sync(0xffffffffu, odd) & group) != 0;
  const uint32_t pair_of_scale = T::down(__fdiv_rn(__fsub_rn(hi, lo), 15.f), lo);
  const float scale = T::up(pair_of_scale).x;
  odd |= !(scale <= 3.402823466e38f);
  uint32_t codes = 0;
  if (!odd && scale > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = rintf(__fdiv_rn(__fsub_rn(x[i], lo), scale));
      codes |= static_cast<uint32_t>(fminf(c, 15.f)) << (4 * i);  // c >= 0: lo is the least x
    }
  }
  const uint32_t pair = odd ? T::down(CUDART_NAN_F, CUDART_NAN_F) : pair_of_scale;
  if (!live || static_cast<uint32_t>(slot) >= static_cast<uint32_t>(p.cache.pages) * p.cache.page_size)
    return;
  const int page = slot / p.cache.page_size, place = slot - page * p.cache.page_size;
  uint8_t* tile = p.cache.page_tiles<D>(page, head) + (place / kTile) * tile_bytes(D);
  const int at = place % kTile;
  const int off = is_v ? off_v(D, at, sub * 8 / kLanes) + (D == 128 ? (sub & 1) * 4 : 0)
                       : off_k(D, at) + 4 * sub;
  *reinterpret_cast<uint32_t*>(tile + off) = codes;
  if (sub == 0)
    *reinterpret_cast<uint32_t*>(tile + (is_v ? off_v_pair(D, at) : off_k_pair(D, at))) = pair;
}

template <class T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kLanes = D / 8;
  const int sub = threadIdx.x % kLanes;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  if (row >= 2ll * p.tokens * p.cache.heads) return;
  const bool is_v = row & 1;
  const int64_t r = row >> 1;
  const int token = static_cast<int>(r / p.cache.heads);
  const int head = static_cast<int>(r - static_cast<int64_t>(token) * p.cache.heads);
  const int slot = p.slots[token];
  uint4 out = make_uint4(0, 0, 0, 0);
  if (static_cast<uint32_t>(slot) < static_cast<uint32_t>(p.cache.pages) * p.cache.page_size) {
    const int page = slot / p.cache.page_size, place = slot - page * p.cache.page_size;
    const uint8_t* tile = p.cache.page_tiles<D>(page, head) + (place / kTile) * tile_bytes(D);
    const int at = place % kTile;
    const int off = is_v ? off_v(D, at, sub * 8 / kLanes) + (D == 128 ? (sub & 1) * 4 : 0)
                         : off_k(D, at) + 4 * sub;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(tile + off);
    const float2 so = T::up(*reinterpret_cast<const uint32_t*>(
        tile + (is_v ? off_v_pair(D, at) : off_k_pair(D, at))));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = static_cast<float>((codes >> (8 * i)) & 15u);
      const float b = static_cast<float>((codes >> (8 * i + 4)) & 15u);
      w[i] = T::down(fmaf(a, so.x, so.y), fmaf(b, so.x, so.y));
    }
    out = make_uint4(w[0], w[1], w[2], w[3]);
  }
  *reinterpret_cast<uint4*>((is_v ? p.v : p.k) + 2 * D * r + 16 * sub) = out;
}

}  // namespace kv4
}  // namespace sm100
