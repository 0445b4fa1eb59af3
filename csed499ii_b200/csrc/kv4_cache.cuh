// Writing keys and values into the 4-bit cache, and reading them back.
// The layout and the rounding are those of kv4_format.cuh.
//
// Both are bound by memory: 4 D bytes of a token and head one way and D + 8 the
// other.  A group of D/8 lanes owns one token and head, its key and its value
// row: each lane holds 8 channels of both, so a warp has 1 KB of loads under
// way; the rows' ranges are shuffle reductions, and a lane's 8 codes of a row
// are one 32-bit word of the tile.
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
  if (aligned) return __ldg(reinterpret_cast<const uint4*>(p));
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  uint4 x;
  x.x = e[0] | static_cast<uint32_t>(e[1]) << 16;
  x.y = e[2] | static_cast<uint32_t>(e[3]) << 16;
  x.z = e[4] | static_cast<uint32_t>(e[5]) << 16;
  x.w = e[6] | static_cast<uint32_t>(e[7]) << 16;
  return x;
}

// The codes of this lane's 8 channels of a row of D/8 lanes, and the row's pair.
template <class T, int D>
__device__ __forceinline__ void quantise(const uint4& raw, uint32_t& codes, uint32_t& pair) {
  constexpr int kLanes = D / 8;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::up(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
  float lo = x[0], hi = x[0], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    sum = fmaf(x[i], 0.f, sum);  // 0, or a NaN for an infinity or a NaN
  }
#pragma unroll
  for (int s = kLanes / 2; s > 0; s >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
  }
  const int lane = threadIdx.x & 31;
  const uint32_t group = ((1u << kLanes) - 1u) << (lane / kLanes * kLanes);
  bool odd = (__ballot_sync(0xffffffffu, !(sum == 0.f)) & group) != 0;
  pair = T::down(__fdiv_rn(__fsub_rn(hi, lo), 15.f), lo);
  const float scale = T::up(pair).x;
  odd |= !(scale <= 3.402823466e38f);
  codes = 0;
  if (odd) {
    pair = T::down(CUDART_NAN_F, CUDART_NAN_F);
  } else if (scale > 0.f) {
    // The quotient rounded to binary32 decides a code.  Times the reciprocal it
    // is within 2^-21 of 15; where that leaves the nearest integer open, and
    // where the reciprocal is not a normal number, it is divided.
    const float inv = __fdividef(1.f, scale);
    bool near = !(inv < 1e37f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = __fmul_rn(__fsub_rn(x[i], lo), inv);
      const float c = rintf(q);
      near |= fabsf(fabsf(q - c) - 0.5f) < 1e-4f;
      codes |= static_cast<uint32_t>(fminf(c, 15.f)) << (4 * i);  // c >= 0: lo is the least x
    }
    if (near) {
      codes = 0;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const float2 f = T::up(i < 4 ? i < 2 ? raw.x : raw.y : i < 6 ? raw.z : raw.w);
        const float c = rintf(__fdiv_rn(__fsub_rn(i & 1 ? f.y : f.x, lo), scale));
        codes |= static_cast<uint32_t>(fminf(c, 15.f)) << (4 * i);
      }
    }
  }
}

// Where a lane's codes and a row's pair of a slot lie.
template <int D>
struct Place {
  uint8_t* tile;
  int k, v, at;

  __device__ __forceinline__ Place(const Cache& cache, int slot, int head, int sub) {
    const int page = slot / cache.page_size, place = slot - page * cache.page_size;
    tile = cache.page_tiles<D>(page, head) + (place / kTile) * tile_bytes(D);
    at = place % kTile;
    k = off_k(D, at) + 4 * sub;
    v = off_v(D, at, sub * 64 / D) + (D == 128 ? (sub & 1) * 4 : 0);
  }
};

template <class T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kLanes = D / 8;  // of a row
  grid_dependency_launch();
  const int sub = threadIdx.x % kLanes;
  const uint32_t rows = static_cast<uint32_t>(p.tokens) * p.cache.heads;
  const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  // a warp's rows are adjacent; rows past the end repeat the last one without storing it
  const uint32_t r = min(row, rows - 1);
  const int token = r / p.cache.heads, head = r - token * p.cache.heads;
  grid_dependency_wait();
  const uint4 k = load_8(p.k + 2 * (p.k_row * token + p.k_head * head) + 16 * sub, p.aligned);
  const uint4 v = load_8(p.v + 2 * (p.v_row * token + p.v_head * head) + 16 * sub, p.aligned);
  const int slot = p.slots[token];
  uint32_t k_codes, k_pair, v_codes, v_pair;
  quantise<T, D>(k, k_codes, k_pair);
  quantise<T, D>(v, v_codes, v_pair);
  if (row >= rows || static_cast<uint32_t>(slot) >= static_cast<uint32_t>(p.cache.pages) * p.cache.page_size)
    return;
  const Place<D> to(p.cache, slot, head, sub);
  *reinterpret_cast<uint32_t*>(to.tile + to.k) = k_codes;
  *reinterpret_cast<uint32_t*>(to.tile + to.v) = v_codes;
  if (sub < 2)
    *reinterpret_cast<uint32_t*>(to.tile + (sub ? off_v_pair(D, to.at) : off_k_pair(D, to.at))) =
        sub ? v_pair : k_pair;
}

// What 8 codes stand for, in the model's type.
template <class T>
__device__ __forceinline__ uint4 values_of(uint32_t codes, uint32_t pair) {
  const float2 so = T::up(pair);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = T::down(fmaf(static_cast<float>((codes >> (8 * i)) & 15u), so.x, so.y),
                   fmaf(static_cast<float>((codes >> (8 * i + 4)) & 15u), so.x, so.y));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kLanes = D / 8;
  grid_dependency_launch();
  const int sub = threadIdx.x % kLanes;
  const uint32_t rows = static_cast<uint32_t>(p.tokens) * p.cache.heads;
  const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int token = row / p.cache.heads, head = row - token * p.cache.heads;
  grid_dependency_wait();
  if (row >= rows) return;
  const int slot = p.slots[token];
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (static_cast<uint32_t>(slot) < static_cast<uint32_t>(p.cache.pages) * p.cache.page_size) {
    const Place<D> at(p.cache, slot, head, sub);
    const uint32_t k_codes = *reinterpret_cast<const uint32_t*>(at.tile + at.k);
    const uint32_t v_codes = *reinterpret_cast<const uint32_t*>(at.tile + at.v);
    const uint32_t k_pair = *reinterpret_cast<const uint32_t*>(at.tile + off_k_pair(D, at.at));
    const uint32_t v_pair = *reinterpret_cast<const uint32_t*>(at.tile + off_v_pair(D, at.at));
    k = values_of<T>(k_codes, k_pair);
    v = values_of<T>(v_codes, v_pair);
  }
  const int64_t to = 2ll * D * row + 16 * sub;
  __stcs(reinterpret_cast<uint4*>(p.k + to), k);
  __stcs(reinterpret_cast<uint4*>(p.v + to), v);
}

}  // namespace kv4
}  // namespace sm100
