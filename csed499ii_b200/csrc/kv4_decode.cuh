// Attention over the 4-bit cache for requests with few query rows (single
// tokens, a few speculated ones).
//
// The bytes of the cache bound it: D + 8 bytes per token and key/value head,
// against 4 * D * rows operations.  So the cache is read once, in its tiles of
// 16 tokens, and the codes go to the tensor cores as they are:
//
//   scores  S[t, r] = s_t (c_t . q_r) + o_t sum(q_r)      (keys' scale, offset)
//   result  O[d, r] = sum_t (p_tr s_t) c_td + sum_t p_tr o_t        (values')
//
// Codes 0..15 are exact in 16 bits and scale and offset stay in 32 bits
// outside the products, so nothing is dequantised and nothing is rounded but
// the weights w = p s (to half, whatever the model's type).  The exponential
// gives w itself, its argument is the score plus log2 s, and the running
// maximum is that of these arguments: a half then holds the weights that
// matter whatever sizes the values have, and p is w / s in 32 bits.  The
// rounding errors would be multiplied by codes that are all positive; the exact
// correction 8 (w - rounded w) in the offset term makes them act as if centred
// on 8, which is what rounding a weight of a dequantised value costs.
//
// mma.m16n8k16 takes 16 tokens (scores) or 16 channels (result) as its rows
// and 8 query rows as its columns; the 8 query heads of a group fill it.  Codes
// become 16-bit operands with one AND per two of them: an integer c < 16 in
// the low bits of a half is the subnormal c * 2^-24, and c << 4 is c * 2^-20,
// both exact in the product; for bf16 queries the codes are OR-ed into the
// mantissa of 128 (128 + c) and the offset term takes the 128 back.
//
// Work is dealt in tiles: all tiles of all (request, head) pairs in a row, cut
// into equal runs, one per warp, whatever the lengths are.  A warp streams its
// run through its own ring of bulk copies, over the borders of pairs; what it
// has of a pair that other warps share is joined in the CTA through shared
// memory, and between CTAs through the workspace by whichever finishes last,
// in CTA order, so results do not depend on timing.
#pragma once

#include <math_constants.h>

#include "kv4_format.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kDecodeBatch = 1024;  // requests of a launch: 8 bytes of shared memory each

struct DecodeParams {
  Cache cache;
  const uint8_t* q;      // element (row, head, c) at q_row * row + q_head * head + c
  int64_t q_row, q_head;
  int q_aligned;         // 1: every row of q starts on a 16-byte boundary
  uint8_t* out;          // [rows][q_heads][D]
  const int* tables;     // [batch][table_stride], `width` entries used
  int64_t table_stride;
  int width;
  const int* lens;       // tokens of each request in the cache, the step's own among them
  const int* starts;     // [batch + 1] first row of each request; null: row b is request b's
  int row0;              // row of request 0 where starts is null
  int batch;
  int rows;              // of q
  int pad;               // 1: rows past the last request are set to zero
  int q_heads;
  int group;             // query heads per key/value head
  int window;            // 0: none
  int most;              // requests with more query rows a group than this are left alone
  float scale;
  int* counters;         // [grid], zero between launches
  float* partials;       // [grid][2] parts
  int* status;
};

template <int D, int NT>
struct DecodeCfg {
  static constexpr int kWarps = 8;
  static constexpr int kDepth = 4;             // tiles in a warp's ring
  static constexpr int kRows = 8 * NT;         // query rows of an item
  static constexpr int kPart = kRows * (D + 2);  // floats: results, maxima, sums
  static constexpr int kRing = kWarps * kDepth * tile_bytes(D);
  static constexpr int kOffParts = kRing;
  static constexpr int kOffPre = kOffParts + kWarps * kPart * 4;
  static constexpr int kOffMisc = kOffPre + kDecodeBatch * 8;
  static constexpr int kSmem = kOffMisc + 2048;
  static constexpr int kCtas = kSmem <= 113 * 1024 ? 2 : 1;  // of an SM
  // a warp's last part takes the place of its ring
  static_assert(kPart * 4 <= kDepth * tile_bytes(D), "part does not fit the ring");
};

// What a launch knows about one request.
struct Span {
  int first, n, len;    // query rows, tokens
  int tile0, tiles;     // that any of its rows sees
  int chunks;           // of query rows
};

template <int ROWS>
__device__ __forceinline__ Span span_of(const DecodeParams& p, int b) {
  Span s;
  s.first = p.starts ? min(max(p.starts[b], 0), p.rows) : p.row0 + b;
  s.n = p.starts ? min(p.starts[b + 1], p.rows) - s.first : 1;
  const int64_t room = static_cast<int64_t>(p.width) * p.cache.page_size;
  s.len = static_cast<int>(min(static_cast<int64_t>(p.lens[b]), room));
  const int64_t rows = static_cast<int64_t>(s.n) * p.group;
  const bool mine = s.n > 0 && rows <= p.most;
  s.chunks = mine ? static_cast<int>((rows + ROWS - 1) / ROWS) : 0;
  const int from = p.window && s.len - s.n >= p.window ? s.len - s.n - p.window + 1 : 0;
  s.tile0 = from / kTile;
  s.tiles = mine && s.len > 0 ? (s.len + kTile - 1) / kTile - s.tile0 : 0;
  return s;
}

// One place in the row of all tiles.
struct Walk {
  Span s;
  int b, head, chunk, tile;  // tile of the request
};

template <int ROWS>
__device__ __forceinline__ Walk walk_to(const DecodeParams& p, const int64_t* pre, int64_t at) {
  int lo = 0, n = p.batch - 1;  // the first request whose end is past `at`
  while (n > 0) {
    const int half = n >> 1;
    if (pre[lo + half] <= at) {
      lo += half + 1;
      n -= half + 1;
    } else {
      n = half;
    }
  }
  Walk w;
  w.b = lo;
  w.s = span_of<ROWS>(p, lo);
  const int64_t off = at - (lo ? pre[lo - 1] : 0);
  const int tiles = max(w.s.tiles, 1);
  const int item = static_cast<int>(off / tiles);
  w.tile = w.s.tile0 + static_cast<int>(off - static_cast<int64_t>(item) * tiles);
  w.head = item / max(w.s.chunks, 1);
  w.chunk = item - w.head * max(w.s.chunks, 1);
  return w;
}

// To the next tile; true where that begins another item.
template <int ROWS>
__device__ __forceinline__ bool walk_on(const DecodeParams& p, Walk& w) {
  if (++w.tile < w.s.tile0 + w.s.tiles) return false;
  if (++w.chunk == w.s.chunks) {
    w.chunk = 0;
    if (++w.head == p.cache.heads) {
      w.head = 0;
      do {
        if (++w.b >= p.batch) return true;  // the end of all work
        w.s = span_of<ROWS>(p, w.b);
      } while (w.s.tiles == 0);
    }
  }
  w.tile = w.s.tile0;
  return true;
}

__device__ __forceinline__ int page_of(const DecodeParams& p, const Walk& w) {
  return w.b < p.batch ? p.tables[p.table_stride * w.b + w.tile / (p.cache.page_size / kTile)] : -1;
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// The 8x8 matrix of 16-bit values spread over the warp, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Codes 2i of the word as key operands: nibbles j and j + 4 of `w`, j = 2i.
template <bool BF16>
__device__ __forceinline__ uint32_t key_even(uint32_t w) {
  return BF16 ? lop3<kLutAndOr>(w, 0x000f000fu, 0x43004300u) : w & 0x000f000fu;
}
// ... and the odd nibbles: 16 times too large in the half form.
template <bool BF16>
__device__ __forceinline__ uint32_t key_odd(uint32_t w) {
  return BF16 ? lop3<kLutAndOr>(w >> 4, 0x000f000fu, 0x43004300u) : w & 0x00f000f0u;
}

// log2 e: scores are kept as exponents of two.
constexpr float kLog2e = 1.4426950408889634f;

// What the weights need to know of a row of values: its scale's logarithm and
// reciprocal, and its value at code 8 over the scale.  A row without a scale
// has all codes 0, so any scale tells the same values; a small one rounds its
// weights where nothing shows.
struct ValueRow {
  float log_s, inv_s, at_8;
};
__device__ __forceinline__ ValueRow value_row(float2 pair) {
  const float s = pair.x > 0x1p-60f ? pair.x : fmaxf(fabsf(pair.y) * 0x1p-10f, 0x1p-60f);
  ValueRow r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r.log_s) : "f"(s));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv_s) : "f"(s));
  r.at_8 = fmaf(pair.y, r.inv_s, 8.f);
  return r;
}

// A part of an item, or all of it: results (already divided by the sum), the
// running maximum of the scores (times log2 e) and the sum of the weights.
struct Segment {
  long long begin, end;  // the item's place in the row of all tiles; begin < 0: none
  int b, head, chunk;
};

constexpr float kLowest = -3.0e38f;

template <class T, int D, int NT>
__global__ void __launch_bounds__(256, DecodeCfg<D, NT>::kCtas)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D, NT>;
  constexpr int kRows = Cfg::kRows, kPart = Cfg::kPart, kDepth = Cfg::kDepth, kBytes = tile_bytes(D);
  constexpr int kWords = D / 32;  // code words of a lane in a row of keys
  constexpr bool kBf = T::kBf16;
  extern __shared__ __align__(128) uint8_t smem[];
  int64_t* pre = reinterpret_cast<int64_t*>(smem + Cfg::kOffPre);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffMisc);            // [warps][depth]
  int* there = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 256);               // [warps][depth]
  Segment* segments = reinterpret_cast<Segment*>(smem + Cfg::kOffMisc + 384);    // [warps][2]
  int64_t* sums = reinterpret_cast<int64_t*>(smem + Cfg::kOffMisc + 1024);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kOffMisc + 1152);
  volatile int* drain_flag = abort_flag + 2;
  int* last_flag = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 1156);
  static_assert(sizeof(Segment) * 16 <= 640, "segments");

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_addr(smem) + warp * kDepth * kBytes;
  const uint32_t bar0 = smem_addr(bars + warp * kDepth);

  if (lane < kDepth) mbar_init(bar0 + 8 * lane, 1);
  if (lane == 0) segments[2 * warp].begin = segments[2 * warp + 1].begin = -1;
  if (threadIdx.x == 0) *abort_flag = *drain_flag = 0;
  fence_mbar_init();

  // --- the row of all tiles: where each request's end is -------------------
  int64_t total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 256) {
    const int b = b0 + threadIdx.x;
    int64_t x = 0;
    if (b < p.batch) {
      const Span s = span_of<kRows>(p, b);
      x = static_cast<int64_t>(p.cache.heads) * s.chunks * s.tiles;
    }
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, i);
      if (lane >= i) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i == warp) x += all;
      all += sums[i];
    }
    if (b < p.batch) pre[b] = total + x;
    total += all;
    __syncthreads();
  }

  // --- rows that see nothing ------------------------------------------------
  {
    const int64_t row_bytes = 2ll * p.q_heads * D;
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (pre[b] != (b ? pre[b - 1] : 0)) continue;
      const Span s = span_of<kRows>(p, b);
      if (s.chunks == 0) continue;
      for (int64_t i = 16 * threadIdx.x; i < s.n * row_bytes; i += 16 * 256)
        *reinterpret_cast<uint4*>(p.out + s.first * row_bytes + i) = make_uint4(0, 0, 0, 0);
    }
    const int end = !p.starts || !p.pad ? p.rows : p.batch ? max(p.starts[p.batch], 0) : 0;
    for (int row = min(end, p.rows) + blockIdx.x; row < p.rows; row += gridDim.x)
      for (int64_t i = 16 * threadIdx.x; i < row_bytes; i += 16 * 256)
        *reinterpret_cast<uint4*>(p.out + row * row_bytes + i) = make_uint4(0, 0, 0, 0);
  }

  const int64_t warps = static_cast<int64_t>(gridDim.x) * Cfg::kWarps;
  const int64_t quota = max((total + warps - 1) / warps, static_cast<int64_t>(2));
  const int64_t cta_begin = quota * Cfg::kWarps * blockIdx.x;
  if (cta_begin >= total) return;
  const int64_t begin = min(cta_begin + quota * warp, total);
  const int64_t end = min(begin + quota, total);
  const int count = static_cast<int>(end - begin);

  // --- this warp's run ------------------------------------------------------
  if (count > 0) {
    Walk in = walk_to<kRows>(p, pre, begin), at = in;
    int page = page_of(p, in);
    int issued = 0;
    const uint64_t policy = policy_evict_first();
    // starts the copy of the next tile of the run; its page was looked up a tile ago
    auto issue = [&]() {
      const int slot = issued % kDepth;
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.pages);
      if (lane == 0) {
        there[warp * kDepth + slot] = ok;
        if (ok) {
          const uint8_t* src = p.cache.page_tiles<D>(page, in.head) +
                               in.tile % (p.cache.page_size / kTile) * kBytes;
          mbar_arrive_expect_tx(bar0 + 8 * slot, kBytes);
          bulk_g2s(ring + slot * kBytes, src, kBytes, bar0 + 8 * slot, policy);
        } else {
          mbar_arrive(bar0 + 8 * slot);
        }
      }
      if (++issued < count) {
        walk_on<kRows>(p, in);
        page = page_of(p, in);
      }
    };
    for (int i = 0; i < kDepth && issued < count; ++i) issue();

    uint32_t qe[NT][kWords][2], qo[NT][kWords][2];  // queries: even and odd nibbles' channels
    float sumq[NT][2];
    int place[NT][2];                               // positions of this lane's two rows
    float acc[NT][D / 16][4];
    float top[NT][2], l[NT][2], a1[NT][2], a2[NT][2];
    const float c2 = p.scale * kLog2e;
    const float c1 = kBf ? c2 : c2 * 16777216.f;
    bool fresh = true;
    int64_t item_begin = 0, item_end = 0;

    for (int i = 0; i < count; ++i) {
      if (fresh) {
        fresh = false;
        item_begin = begin + i - (at.tile - at.s.tile0);
        item_end = item_begin + at.s.tiles;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = at.chunk * kRows + nt * 8 + g;
          const int token = r / p.group, h = at.head * p.group + r % p.group;
          float sum = 0.f;
          const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) +
                                p.q_row * (at.s.first + token) + p.q_head * h + t * (D / 4);
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (token < at.s.n) {
              if (p.q_aligned) {
                x = *reinterpret_cast<const uint4*>(src + 8 * w);
              } else {
                uint32_t y[4];
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  y[z] = src[8 * w + 2 * z] | static_cast<uint32_t>(src[8 * w + 2 * z + 1]) << 16;
                x = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
            qe[nt][w][0] = prmt_b32(x.x, x.z, 0x5410);
            qe[nt][w][1] = prmt_b32(x.y, x.w, 0x5410);
            qo[nt][w][0] = prmt_b32(x.x, x.z, 0x7632);
            qo[nt][w][1] = prmt_b32(x.y, x.w, 0x7632);
            const float2 f0 = T::up(x.x), f1 = T::up(x.y), f2 = T::up(x.z), f3 = T::up(x.w);
            sum += ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            sumq[nt][c] = __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
            place[nt][c] = at.s.len - at.s.n + (at.chunk * kRows + nt * 8 + 2 * t + c) / p.group;
            top[nt][c] = kLowest;
            l[nt][c] = a1[nt][c] = a2[nt][c] = 0.f;
          }
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[nt][x][c] = 0.f;
        }
      }

      const int slot = i % kDepth;
      const uint32_t tile = ring + slot * kBytes;
      if (!mbar_wait_bounded(bar0 + 8 * slot, (i / kDepth) & 1, abort_flag)) {
        if (lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
        // the copies still in flight land before the CTA's memory is handed on
        for (int j = i; j < issued; ++j)
          mbar_wait_bounded(bar0 + 8 * (j % kDepth), (j / kDepth) & 1, drain_flag);
        break;
      }
      if (there[warp * kDepth + slot]) {
        // scores
        uint32_t k0[kWords], k1[kWords];
        if constexpr (D == 128) {
          const uint4 x = lds128(tile + 16 * lane), y = lds128(tile + 512 + 16 * lane);
          k0[0] = x.x, k0[1] = x.y, k0[2] = x.z, k0[3] = x.w;
          k1[0] = y.x, k1[1] = y.y, k1[2] = y.z, k1[3] = y.w;
        } else {
          const uint2 x = lds64(tile + 8 * lane), y = lds64(tile + 256 + 8 * lane);
          k0[0] = x.x, k0[1] = x.y;
          k1[0] = y.x, k1[1] = y.y;
        }
        const float2 kp0 = T::up(lds32(tile + off_k_pair(D, g))), kp1 = T::up(lds32(tile + off_k_pair(D, g + 8)));
        const ValueRow v0 = value_row(T::up(lds32(tile + off_v_pair(D, g))));
        const ValueRow v1 = value_row(T::up(lds32(tile + off_v_pair(D, g + 8))));
        float x[NT][4];  // arguments of the weights
        {
          float e[NT][4] = {}, o[NT][4] = {};
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const uint32_t h0 = k0[w] >> 8, h1 = k1[w] >> 8;
            const uint32_t ea0 = key_even<kBf>(k0[w]), ea1 = key_even<kBf>(k1[w]);
            const uint32_t ea2 = key_even<kBf>(h0), ea3 = key_even<kBf>(h1);
            const uint32_t oa0 = key_odd<kBf>(k0[w]), oa1 = key_odd<kBf>(k1[w]);
            const uint32_t oa2 = key_odd<kBf>(h0), oa3 = key_odd<kBf>(h1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<kBf>(e[nt], ea0, ea1, ea2, ea3, qe[nt][w][0], qe[nt][w][1]);
              mma_16816<kBf>(o[nt], oa0, oa1, oa2, oa3, qo[nt][w][0], qo[nt][w][1]);
            }
          }
          const float s0 = kp0.x * c1, s1 = kp1.x * c1;
          const float z0 = (kBf ? fmaf(kp0.x, -128.f, kp0.y) : kp0.y) * c2;
          const float z1 = (kBf ? fmaf(kp1.x, -128.f, kp1.y) : kp1.y) * c2;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float dot = fmaf(o[nt][c], kBf ? 1.f : 0.0625f, e[nt][c]);
              x[nt][c] = fmaf(c < 2 ? s0 : s1, dot,
                              fmaf(c < 2 ? z0 : z1, sumq[nt][c & 1], c < 2 ? v0.log_s : v1.log_s));
            }
        }
        // what of the tile each row sees; most tiles are seen whole
        const int j0 = at.tile * kTile;
        const bool whole = j0 + kTile <= at.s.len - at.s.n + 1 &&
                           (p.window == 0 || at.s.len - j0 <= p.window);
        bool seen[NT][4];
        if (!whole) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int j = j0 + g + (c < 2 ? 0 : 8);
              seen[nt][c] = j <= place[nt][c & 1] && j < at.s.len &&
                            (p.window == 0 || place[nt][c & 1] - j < p.window);
              if (!seen[nt][c]) x[nt][c] = -CUDART_INF_F;
            }
        }
        // The maximum moves only where an argument passes it by more than 8 (a
        // factor of 256, harmless in the sums), so most tiles need no exchange.
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) moves |= x[nt][c] > top[nt][c & 1] + 8.f;
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float m = fmaxf(top[nt][c], fmaxf(x[nt][c], x[nt][c + 2]));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              f[c] = exp2_approx(top[nt][c] - m);
              top[nt][c] = m;
              l[nt][c] *= f[c];
              a1[nt][c] *= f[c];
              a2[nt][c] *= f[c];
            }
#pragma unroll
            for (int y = 0; y < D / 16; ++y) {
              acc[nt][y][0] *= f[0];
              acc[nt][y][1] *= f[1];
              acc[nt][y][2] *= f[0];
              acc[nt][y][3] *= f[1];
            }
          }
        }
        // weights, and their sums
        uint32_t wb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            w[c] = exp2_approx(x[nt][c] - top[nt][c & 1]);
            // where nothing is seen, scale and offset may be anything
            const bool none = !whole && !seen[nt][c];
            l[nt][c & 1] = fmaf(w[c], none ? 0.f : c < 2 ? v0.inv_s : v1.inv_s, l[nt][c & 1]);
            a1[nt][c & 1] = fmaf(w[c], none ? 0.f : c < 2 ? v0.at_8 : v1.at_8, a1[nt][c & 1]);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t y = Half::down(w[2 * c], w[2 * c + 1]);
            const float2 back = Half::up(y);
            a2[nt][0] += back.x;
            a2[nt][1] += back.y;
            wb[nt][c] = transpose_8x8(y);
          }
        }
        // result
        constexpr int kOctets = D / 64;
        uint32_t va[kOctets], vb[kOctets], vc[kOctets], vd[kOctets];  // tokens 2t, 2t+1, 2t+8, 2t+9
        if constexpr (D == 128) {
          const uint4 y = lds128(tile + 8 * D + 16 * lane), z = lds128(tile + 12 * D + 16 * lane);
          va[0] = y.x, va[1] = y.y, vb[0] = y.z, vb[1] = y.w;
          vc[0] = z.x, vc[1] = z.y, vd[0] = z.z, vd[1] = z.w;
        } else {
          const uint2 y = lds64(tile + 8 * D + 8 * lane), z = lds64(tile + 12 * D + 8 * lane);
          va[0] = y.x, vb[0] = y.y;
          vc[0] = z.x, vd[0] = z.y;
        }
#pragma unroll
        for (int o = 0; o < kOctets; ++o)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t y = prmt_b32(va[o], vb[o], sel), z = prmt_b32(vc[o], vd[o], sel);
            const uint32_t y8 = y >> 8, z8 = z >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<false>(acc[nt][4 * o + 2 * half], y & 0x000f000fu, y & 0x00f000f0u,
                               z & 0x000f000fu, z & 0x00f000f0u, wb[nt][0], wb[nt][1]);
              mma_16816<false>(acc[nt][4 * o + 2 * half + 1], y8 & 0x000f000fu, y8 & 0x00f000f0u,
                               z8 & 0x000f000fu, z8 & 0x00f000f0u, wb[nt][0], wb[nt][1]);
            }
          }
      }
      __syncwarp();  // the slot is read
      if (issued < count) issue();

      // --- the end of an item, or of the run --------------------------------
      const Walk here = at;
      const bool ends = walk_on<kRows>(p, at);
      if (!ends && i + 1 < count) continue;
      fresh = true;
      const bool all = item_begin >= begin && item_end <= end;
      const bool is_head = !all && ends && item_begin < begin && i + 1 < count;
      float* part = is_head ? reinterpret_cast<float*>(smem + Cfg::kOffParts) + warp * kPart
                            : reinterpret_cast<float*>(smem + warp * kDepth * kBytes);
      if (!all && lane == 0)
        segments[2 * warp + (is_head ? 0 : 1)] = {item_begin, item_end, here.b, here.head, here.chunk};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) {
            l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], s);
            a1[nt][c] += __shfl_xor_sync(0xffffffffu, a1[nt][c], s);
            a2[nt][c] += __shfl_xor_sync(0xffffffffu, a2[nt][c], s);
          }
          const float over = l[nt][c] == 0.f ? 0.f : 1.f / l[nt][c];
          // this lane has channels [D/8 g, D/8 (g + 1)) of the row
          float y[D / 8];
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            y[2 * x] = (fmaf(acc[nt][x][c], 16777216.f, -8.f * a2[nt][c]) + a1[nt][c]) * over;
            y[2 * x + 1] = (fmaf(acc[nt][x][c + 2], 1048576.f, -8.f * a2[nt][c]) + a1[nt][c]) * over;
          }
          const int r = nt * 8 + 2 * t + c, row = here.chunk * kRows + r;
          if (row >= here.s.n * p.group) continue;
          if (all) {
            uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(here.s.first + row / p.group) * p.q_heads +
                                         here.head * p.group + row % p.group) * D + D / 8 * g);
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              *reinterpret_cast<uint4*>(dst + 16 * x) =
                  make_uint4(T::down(y[8 * x], y[8 * x + 1]), T::down(y[8 * x + 2], y[8 * x + 3]),
                             T::down(y[8 * x + 4], y[8 * x + 5]), T::down(y[8 * x + 6], y[8 * x + 7]));
          } else {
#pragma unroll
            for (int x = 0; x < D / 32; ++x)
              *reinterpret_cast<float4*>(part + r * D + D / 8 * g + 4 * x) =
                  make_float4(y[4 * x], y[4 * x + 1], y[4 * x + 2], y[4 * x + 3]);
            if (g == 0) part[kRows * D + r] = top[nt][c], part[kRows * D + kRows + r] = l[nt][c];
          }
        }
    }
  }
  __syncthreads();
  if (*abort_flag) return;

  // --- parts of this CTA's warps, joined -------------------------------------
  const int64_t cta_quota = quota * Cfg::kWarps;
  const int64_t cta_end = min(cta_begin + cta_quota, total);
  auto part_of = [&](int s) -> const float* {
    return s & 1 ? reinterpret_cast<const float*>(smem + (s >> 1) * kDepth * kBytes)
                 : reinterpret_cast<const float*>(smem + Cfg::kOffParts) + (s >> 1) * kPart;
  };
  for (int s0 = 0; s0 < 2 * Cfg::kWarps;) {
    const Segment seg = segments[s0];
    if (seg.begin < 0) {
      ++s0;
      continue;
    }
    int s1 = s0 + 1;
    while (s1 < 2 * Cfg::kWarps && (segments[s1].begin < 0 || segments[s1].begin == seg.begin)) ++s1;
    const Span sp = span_of<kRows>(p, seg.b);
    const int rows = min(kRows, sp.n * p.group - seg.chunk * kRows);
    const bool all = seg.begin >= cta_begin && seg.end <= cta_end;
    const int c0 = static_cast<int>(seg.begin / cta_quota), c1 = static_cast<int>((seg.end - 1) / cta_quota);
    float* to = p.partials + (2ll * blockIdx.x + (seg.begin < cta_begin ? 0 : 1)) * kPart;
    auto store = [&](int i, float lo, float hi) {
      const int row = seg.chunk * kRows + i / (D / 2);
      *reinterpret_cast<uint32_t*>(
          p.out + 2 * ((static_cast<int64_t>(sp.first + row / p.group) * p.q_heads + seg.head * p.group +
                        row % p.group) * D + 2 * (i % (D / 2)))) = T::down(lo, hi);
    };
    for (int i = threadIdx.x; i < rows * (D / 2); i += 256) {
      const int r = i / (D / 2);
      float m = kLowest;
      for (int s = s0; s < s1; ++s)
        if (segments[s].begin >= 0) m = fmaxf(m, part_of(s)[kRows * D + r]);
      float sum = 0.f, x = 0.f, y = 0.f;
      for (int s = s0; s < s1; ++s) {
        if (segments[s].begin < 0) continue;
        const float* part = part_of(s);
        const float w = part[kRows * D + kRows + r] * exp2_approx(part[kRows * D + r] - m);
        const float2 v = *reinterpret_cast<const float2*>(part + 2 * i);
        sum += w;
        x = fmaf(w, v.x, x);
        y = fmaf(w, v.y, y);
      }
      const float over = sum == 0.f ? 0.f : 1.f / sum;
      if (all) {
        store(i, x * over, y * over);
      } else {
        *reinterpret_cast<float2*>(to + 2 * i) = make_float2(x * over, y * over);
        if (i % (D / 2) == 0) to[kRows * D + r] = m, to[kRows * D + kRows + r] = sum;
      }
    }
    if (!all) {
      // the last CTA to bring its part joins them, in CTA order
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) *last_flag = atomicAdd(p.counters + c0, 1) == c1 - c0;
      __syncthreads();
      if (*last_flag) {
        __threadfence();
        auto from = [&](int c) -> const float* {
          return p.partials + (2ll * c + (c == c0 ? 1 : 0)) * kPart;
        };
        for (int i = threadIdx.x; i < rows * (D / 2); i += 256) {
          const int r = i / (D / 2);
          float m = kLowest;
          for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(from(c) + kRows * D + r));
          float sum = 0.f, x = 0.f, y = 0.f;
          for (int c = c0; c <= c1; ++c) {
            const float w = __ldcg(from(c) + kRows * D + kRows + r) * exp2_approx(__ldcg(from(c) + kRows * D + r) - m);
            const float2 v = __ldcg(reinterpret_cast<const float2*>(from(c) + 2 * i));
            sum += w;
            x = fmaf(w, v.x, x);
            y = fmaf(w, v.y, y);
          }
          const float over = sum == 0.f ? 0.f : 1.f / sum;
          store(i, x * over, y * over);
        }
        if (threadIdx.x == 0) p.counters[c0] = 0;
      }
      __syncthreads();
    }
    s0 = s1;
  }
}

}  // namespace kv4
}  // namespace sm100
