// The 4-bit paged key/value cache: its layout, and the numbers in it.
//
// A page holds `page_size` tokens (a multiple of 16) of one layer; per page
// and key/value head it is a row of tiles of 16 tokens.  With D channels a
// head, a tile is 16*D + 128 bytes (2176 at D = 128, 1152 at D = 64: both
// multiples of 128, so a tile is one aligned bulk copy):
//
//   [0, 8D)           key codes: 16 rows of D/2 bytes, channel 2i in the low
//                     half of byte i
//   [8D, 16D)         value codes, [2][8][8][D/16] bytes: half of the tile,
//                     eighth of the row, token in the half, byte
//   [16D, 16D + 64)   16 pairs (scale, offset) of the keys, 16-bit each
//   [16D + 64, +64)   16 pairs of the values
//
// Both orders are operand orders of mma.m16n8k16: a lane (g = lane / 4,
// t = lane % 4) finds the key codes of token g (and g + 8) in D/8 adjacent
// bytes, lane after lane, and the value codes of tokens 2t and 2t + 1 (of
// either half) for channels [D/8 g, D/8 (g + 1)) in D/8 adjacent bytes, lane
// after lane.
//
// The row x[0..D) of one token and head, in binary32 rounded to nearest even:
//   offset = min x,  scale = (max x - min x) / 15 rounded to the model's type,
//   code = rint((x - offset) / scale) kept in 0..15 (0 where scale is 0).
// offset is one of the row's own values, so it is exact in the model's type.
// A row with an infinity or a NaN, or whose range overflows, gets a NaN scale:
// all of it stands for NaN, as its attention would be in any precision.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "device_primitives.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kTile = 16;  // tokens of a tile

__host__ __device__ constexpr int tile_bytes(int dim) { return 16 * dim + 128; }

// Byte offsets inside a tile.
__host__ __device__ constexpr int off_k(int dim, int token) { return token * (dim / 2); }
__host__ __device__ constexpr int off_v(int dim, int token, int piece) {
  return 8 * dim + (token >> 3) * (4 * dim) + piece * (dim / 2) + (token & 7) * (dim / 16);
}
__host__ __device__ constexpr int off_k_pair(int dim, int token) { return 16 * dim + 4 * token; }
__host__ __device__ constexpr int off_v_pair(int dim, int token) { return 16 * dim + 64 + 4 * token; }

// The cache tensor: [pages][heads][page_size / 16] tiles.
struct Cache {
  uint8_t* tiles;
  int pages;
  int heads;
  int page_size;

  // First tile of (page, head); 64-bit, since a cache passes 4 GB.
  template <int D>
  __device__ __forceinline__ uint8_t* page_tiles(int page, int head) const {
    return tiles + (static_cast<int64_t>(page) * heads + head) * (page_size / kTile) *
                       static_cast<int64_t>(tile_bytes(D));
  }
  // Tile `nth` of (page, head); a page alone can pass 2 GB.
  template <int D>
  __device__ __forceinline__ uint8_t* tile(int page, int head, int nth) const {
    return page_tiles<D>(page, head) + static_cast<int64_t>(nth) * tile_bytes(D);
  }
};

// Two floats in one register pair, for the two-wide instructions.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The two 16-bit types of a model.
struct Half {
  static constexpr bool kBf16 = false;
  // of two pairs; NaN where either is
  static __device__ __forceinline__ uint32_t least(uint32_t x, uint32_t y) {
    const half2 h = __hmin2_nan(*reinterpret_cast<const half2*>(&x), *reinterpret_cast<const half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {
    const half2 h = __hmax2_nan(*reinterpret_cast<const half2*>(&x), *reinterpret_cast<const half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 up(uint32_t x) {
    return __half22float2(*reinterpret_cast<const half2*>(&x));
  }
  static __device__ __forceinline__ uint32_t down(float lo, float hi) {
    const half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

struct Bf16 {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ uint32_t least(uint32_t x, uint32_t y) {
    const __nv_bfloat162 h =
        __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {
    const __nv_bfloat162 h =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 up(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t down(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

}  // namespace kv4
}  // namespace sm100
