// Writing keys and values into the 4-bit cache, and reading them back.
// The layout and the rounding are those of kv4_format.cuh.
//
// Both are bound by memory: 4 D bytes of a token and head one way and D + 8 the
// other.  Eight lanes own one token and head, its key and its value row: a lane
// holds D/64 pieces of 8 channels of both, 64 channels apart; the rows' ranges
// are shuffle reductions, and the 8 codes of a piece are one 32-bit word of the
// tile.  8192 tokens of 8 heads of 128, one call after another: written in 13.0 us
// (42.5 MB, 3.3 TB/s; 62% of issue slots are taken, the integer and the float pipe two
// fifths of the time each), read in 9.1 us (4.7 TB/s of 6.55 measured for a copy).
// With a lane for 8 channels of a row the row's own numbers cost twice as much, a
// third and a sixth more time.
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

// 8 channels as 4 words of two.  Not through the read-only path: this kernel has
// begun while the one before it may still write them, and loads of that path need
// not stay behind the wait.
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

constexpr int kCacheThreads = 128, kRowLanes = 8;

// The codes of this lane's pieces of a row, and the row's pair.
//
// The quotient rounded to binary32 decides a code.  It comes from the rounded
// reciprocal y of the scale, by Markstein's theorem (IBM J. Res. Dev. 34, 1990):
// q = d y, r = d - q scale (exact), and q + r y rounded is d / scale rounded.
// Scales that bring r near the ends of binary32, or so small in their type that
// quotients can pass 15.5, are divided one by one.  Two channels an instruction, and the codes are put
// together as sums of binary32 integers: one by one, with minima and maxima in
// binary32, the instructions bound the kernel (8192 tokens of 8 heads of 128
// took 25 us).
template <class T, int N>
__device__ __forceinline__ void quantise(const uint4 (&raw)[N], uint32_t (&codes)[N], uint32_t& pair) {
  // the least channel, and the largest negated, which is the least then too
  uint32_t ends;
  {
    uint32_t lo = T::least(T::least(raw[0].x, raw[0].y), T::least(raw[0].z, raw[0].w));
    uint32_t hi = T::most(T::most(raw[0].x, raw[0].y), T::most(raw[0].z, raw[0].w));
#pragma unroll
    for (int n = 1; n < N; ++n) {
      lo = T::least(lo, T::least(T::least(raw[n].x, raw[n].y), T::least(raw[n].z, raw[n].w)));
      hi = T::most(hi, T::most(T::most(raw[n].x, raw[n].y), T::most(raw[n].z, raw[n].w)));
    }
    hi ^= 0x80008000u;
    ends = T::least(prmt_b32(lo, hi, 0x5410), prmt_b32(lo, hi, 0x7632));
  }
#pragma unroll
  for (int s = kRowLanes / 2; s > 0; s >>= 1) ends = T::least(ends, __shfl_xor_sync(0xffffffffu, ends, s));
  const float lo = T::up(ends).x, hi = -T::up(ends).y;
  pair = T::down(__fdiv_rn(__fsub_rn(hi, lo), 15.f), lo);
  const float scale = T::up(pair).x;
#pragma unroll
  for (int n = 0; n < N; ++n) codes[n] = 0;
  if (!(scale <= 3.402823466e38f)) {  // an infinity or a NaN in the row, or a range past the type
    pair = T::down(CUDART_NAN_F, CUDART_NAN_F);
  } else if (scale > 0.f) {
    const float y = __frcp_rn(scale);
    constexpr float kInt = 12582912.f;  // 1.5 * 2^23: what is added to it is rounded to an integer
    const F2 lo2 = pack2(-lo, -lo), y2 = pack2(y, y), scale2 = pack2(-scale, -scale), one = pack2(1.f, 1.f);
    const F2 zero = pack2(-0.f, -0.f), to_int = pack2(kInt, kInt), from_int = pack2(-kInt, -kInt);
    const F2 k256 = pack2(256.f, 256.f), k2_23 = pack2(8388608.f, 0.f);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t w[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
      F2 c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = T::up(w[i]);
        const F2 d = fma2(one, pack2(x.x, x.y), lo2), q = fma2(d, y2, zero);
        c[i] = fma2(one, fma2(one, fma2(fma2(q, scale2, d), y2, q), to_int), from_int);
      }
      const float2 a = unpack2(fma2(c[1], k256, fma2(one, c[0], k2_23)));
      const float2 b = unpack2(fma2(c[3], k256, fma2(one, c[2], k2_23)));
      codes[n] = prmt_b32(__float_as_uint(fmaf(a.y, 16.f, a.x)), __float_as_uint(fmaf(b.y, 16.f, b.x)), 0x5410);
    }
    if (!(scale > (T::kBf16 ? 0x1p-80f : 0x1p-19f) && scale < 0x1p80f)) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        codes[n] = 0;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const float2 f = T::up(i < 4 ? i < 2 ? raw[n].x : raw[n].y : i < 6 ? raw[n].z : raw[n].w);
          const float q = rintf(__fdiv_rn(__fsub_rn(i & 1 ? f.y : f.x, lo), scale));
          codes[n] |= static_cast<uint32_t>(fminf(q, 15.f)) << (4 * i);  // q >= 0: lo is the least
        }
      }
    }
  }
}

// Where the codes and the pairs of a slot lie.
template <int D>
struct Place {
  uint8_t* tile;
  int at;

  __device__ __forceinline__ Place(const Cache& cache, int slot, int head) {
    const int page = slot / cache.page_size, place = slot - page * cache.page_size;
    tile = cache.tile<D>(page, head, place / kTile);
    at = place % kTile;
  }
  // of channels [8 o, 8 o + 8)
  __device__ __forceinline__ uint32_t* k(int o) const {
    return reinterpret_cast<uint32_t*>(tile + off_k(D, at) + 4 * o);
  }
  __device__ __forceinline__ uint32_t* v(int o) const {
    return reinterpret_cast<uint32_t*>(tile + off_v(D, at, o * 64 / D) + (D == 128 ? (o & 1) * 4 : 0));
  }
  __device__ __forceinline__ uint32_t* pair(bool v) const {
    return reinterpret_cast<uint32_t*>(tile + (v ? off_v_pair(D, at) : off_k_pair(D, at)));
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kCacheThreads) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int N = D / 64;
  const int sub = threadIdx.x % kRowLanes;
  const uint32_t rows = static_cast<uint32_t>(p.tokens) * p.cache.heads;
  const uint32_t row = blockIdx.x * (kCacheThreads / kRowLanes) + threadIdx.x / kRowLanes;
  // a warp's rows are adjacent; rows past the end repeat the last one without storing it
  const uint32_t r = min(row, rows - 1);
  const int token = r / p.cache.heads, head = r - token * p.cache.heads;
  const uint8_t* k_from = p.k + 2 * (p.k_row * token + p.k_head * head) + 16 * sub;
  const uint8_t* v_from = p.v + 2 * (p.v_row * token + p.v_head * head) + 16 * sub;
  grid_dependency_wait();
  grid_dependency_launch();
  uint4 k[N], v[N];
#pragma unroll
  for (int n = 0; n < N; ++n) k[n] = load_8(k_from + 128 * n, p.aligned), v[n] = load_8(v_from + 128 * n, p.aligned);
  const int slot = p.slots[token];
  uint32_t k_codes[N], k_pair, v_codes[N], v_pair;
  quantise<T>(k, k_codes, k_pair);
  quantise<T>(v, v_codes, v_pair);
  if (row >= rows || static_cast<uint32_t>(slot) >= static_cast<uint32_t>(p.cache.pages) * p.cache.page_size)
    return;
  const Place<D> to(p.cache, slot, head);
#pragma unroll
  for (int n = 0; n < N; ++n) *to.k(sub + 8 * n) = k_codes[n], *to.v(sub + 8 * n) = v_codes[n];
  if (sub < 2) *to.pair(sub) = sub ? v_pair : k_pair;
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
__global__ void __launch_bounds__(kCacheThreads) kv4_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int N = D / 64;
  const int sub = threadIdx.x % kRowLanes;
  const uint32_t rows = static_cast<uint32_t>(p.tokens) * p.cache.heads;
  const uint32_t row = blockIdx.x * (kCacheThreads / kRowLanes) + threadIdx.x / kRowLanes;
  const int token = row / p.cache.heads, head = row - token * p.cache.heads;
  grid_dependency_wait();
  grid_dependency_launch();
  if (row >= rows) return;
  const int slot = p.slots[token];
  uint4 k[N], v[N];
#pragma unroll
  for (int n = 0; n < N; ++n) k[n] = v[n] = make_uint4(0, 0, 0, 0);
  if (static_cast<uint32_t>(slot) < static_cast<uint32_t>(p.cache.pages) * p.cache.page_size) {
    const Place<D> at(p.cache, slot, head);
    uint32_t k_codes[N], v_codes[N];
#pragma unroll
    for (int n = 0; n < N; ++n) k_codes[n] = *at.k(sub + 8 * n), v_codes[n] = *at.v(sub + 8 * n);
    const uint32_t k_pair = *at.pair(false), v_pair = *at.pair(true);
#pragma unroll
    for (int n = 0; n < N; ++n) k[n] = values_of<T>(k_codes[n], k_pair), v[n] = values_of<T>(v_codes[n], v_pair);
  }
  const int64_t to = 2ll * D * row + 16 * sub;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    __stcs(reinterpret_cast<uint4*>(p.k + to + 128 * n), k[n]);
    __stcs(reinterpret_cast<uint4*>(p.v + to + 128 * n), v[n]);
  }
}

}  // namespace kv4
}  // namespace sm100
