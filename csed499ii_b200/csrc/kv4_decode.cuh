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

constexpr int kDecodeBatch = 1024;  // requests of a launch: 4 bytes of shared memory each
constexpr int kLeast = 16;          // tiles of a CTA: fewer are not worth sharing an item

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
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kDepth = 4;             // tiles in a warp's ring
  static constexpr int kRows = 8 * NT;         // query rows of an item
  static constexpr int kPart = kRows * (D + 2);  // floats: results, maxima, sums
  static constexpr int kRing = kWarps * kDepth * tile_bytes(D);
  static constexpr int kOffParts = kRing;
  static constexpr int kOffPre = kOffParts + kWarps * kPart * 4;
  static constexpr int kOffMisc = kOffPre + kDecodeBatch * 4;
  static constexpr int kMisc = 1424 + 64 * kRows;
  static constexpr int kSmem = kOffMisc + kMisc;
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

// One item (a request, a key/value head, kRows of its query rows) and a tile.
struct Walk {
  Span s;
  int b, head, chunk, tile;  // tile of the request
};

template <int ROWS>
__device__ __forceinline__ Walk walk_to(const DecodeParams& p, const int* pre, int at) {
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
  const int off = at - (lo ? pre[lo - 1] : 0);
  const int tiles = max(w.s.tiles, 1);
  const int item = off / tiles;
  w.tile = w.s.tile0 + off - item * tiles;
  w.head = item / max(w.s.chunks, 1);
  w.chunk = item - w.head * max(w.s.chunks, 1);
  return w;
}

// To the first tile of the next item; only called while there is one.
template <int ROWS>
__device__ __forceinline__ void next_item(const DecodeParams& p, Walk& w) {
  if (++w.chunk == w.s.chunks) {
    w.chunk = 0;
    if (++w.head == p.cache.heads) {
      w.head = 0;
      do {
        w.s = span_of<ROWS>(p, ++w.b);
      } while (w.s.tiles == 0 && w.b + 1 < p.batch);
    }
  }
  w.tile = w.s.tile0;
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

__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
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
  int begin, end;  // the item's place in the row of all tiles; begin < 0: none
  int b, head, chunk;
};

constexpr float kLowest = -3.0e38f;

template <class T, int D, int NT>
__global__ void __launch_bounds__(DecodeCfg<D, NT>::kThreads, DecodeCfg<D, NT>::kCtas)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D, NT>;
  constexpr int kRows = Cfg::kRows, kPart = Cfg::kPart, kDepth = Cfg::kDepth, kBytes = tile_bytes(D);
  constexpr int kWords = D / 32;  // code words of a lane in a row of keys
  constexpr bool kBf = T::kBf16;
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre = reinterpret_cast<int*>(smem + Cfg::kOffPre);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffMisc);            // [warps][depth]
  int* there = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 512);               // [warps][depth]
  Segment* segments = reinterpret_cast<Segment*>(smem + Cfg::kOffMisc + 640);    // [warps][2]
  int* sums = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 1280);               // [warps]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kOffMisc + 1408);
  volatile int* drain_flag = abort_flag + 1;
  int* last_flag = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 1416);
  float* join_w = reinterpret_cast<float*>(smem + Cfg::kOffMisc + 1424);         // [2 warps][rows]
  static_assert(sizeof(Segment) * 16 <= 640 && 1424 + 4 * 16 * kRows <= Cfg::kMisc, "shared memory");

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  if (lane < kDepth) mbar_init(smem_addr(bars + kDepth * warp + lane), 1);
  if (lane == 0) segments[2 * warp].begin = segments[2 * warp + 1].begin = -1;
  if (threadIdx.x == 0) *abort_flag = *drain_flag = 0;
  fence_mbar_init();

  // --- the row of all tiles: where each request's end is -------------------
  int total = 0;  // the host keeps it below 2^31
  for (int b0 = 0; b0 < p.batch; b0 += Cfg::kThreads) {
    const int b = b0 + threadIdx.x;
    int x = 0;
    if (b < p.batch) {
      const Span s = span_of<kRows>(p, b);
      x = p.cache.heads * s.chunks * s.tiles;
    }
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, i);
      if (lane >= i) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < Cfg::kWarps; ++i) {
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
      for (int64_t i = 16 * threadIdx.x; i < s.n * row_bytes; i += 16 * Cfg::kThreads)
        *reinterpret_cast<uint4*>(p.out + s.first * row_bytes + i) = make_uint4(0, 0, 0, 0);
    }
    const int end = !p.starts || !p.pad ? p.rows : p.batch ? max(p.starts[p.batch], 0) : 0;
    for (int row = min(end, p.rows) + blockIdx.x; row < p.rows; row += gridDim.x)
      for (int64_t i = 16 * threadIdx.x; i < row_bytes; i += 16 * Cfg::kThreads)
        *reinterpret_cast<uint4*>(p.out + row * row_bytes + i) = make_uint4(0, 0, 0, 0);
  }

  const int quota = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), kLeast);  // of a CTA
  if (static_cast<int64_t>(quota) * blockIdx.x >= total) return;
  const int cta_begin = quota * blockIdx.x;
  const int cta_end = min(cta_begin + quota, total);
  const int share = (cta_end - cta_begin + Cfg::kWarps - 1) / Cfg::kWarps;
  const int begin = min(cta_begin + share * warp, cta_end);
  const int count = min(begin + share, cta_end) - begin;

  // --- this warp's run ------------------------------------------------------
  if (count > 0) {
    const uint32_t ring = smem_addr(smem) + warp * kDepth * kBytes;
    const uint32_t full = smem_addr(bars + kDepth * warp);
    Walk at = walk_to<kRows>(p, pre, begin);

    // The copies run ahead of the work: `in` is the item of the next one, and
    // a page's number is looked up a page early.
    Walk in = at;
    const int per_page = p.cache.page_size / kTile;
    const uint64_t policy = policy_evict_first();
    int issued = 0, entry, nth, page, next;  // nth tile of the page
    auto start = [&]() {
      entry = in.tile / per_page;
      nth = in.tile - entry * per_page;
      const int* table = p.tables + p.table_stride * in.b;
      page = table[entry];
      next = entry + 1 < p.width ? table[entry + 1] : -1;
    };
    auto issue = [&]() {
      const int slot = issued % kDepth;
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.pages);
      if (lane == 0) {
        there[warp * kDepth + slot] = ok;
        if (ok) {
          mbar_arrive_expect_tx(full + 8 * slot, kBytes);
          bulk_g2s(ring + slot * kBytes, p.cache.page_tiles<D>(page, in.head) + nth * kBytes, kBytes,
                   full + 8 * slot, policy);
        } else {
          mbar_arrive(full + 8 * slot);
        }
      }
      if (++issued == count) return;
      if (++in.tile == in.s.tile0 + in.s.tiles) {
        next_item<kRows>(p, in);
        start();
      } else if (++nth == per_page) {
        nth = 0;
        ++entry;
        page = next;
        next = entry + 1 < p.width ? p.tables[p.table_stride * in.b + entry + 1] : -1;
      }
    };
    // the first queries are on their way while the first pages are looked up
    if (at.chunk * kRows + (lane >> 2) < at.s.n * p.group)
      prefetch_l1(p.q + 2 * (p.q_row * (at.s.first + (at.chunk * kRows + (lane >> 2)) / p.group) +
                             p.q_head * (at.head * p.group + (at.chunk * kRows + (lane >> 2)) % p.group) + t * (D / 4)));
    start();
    for (int i = 0; i < kDepth && issued < count; ++i) issue();

    uint32_t qe[NT][kWords][2], qo[NT][kWords][2];  // queries: even and odd nibbles' channels
    float sumq[NT][2];
    int place[NT][2];                               // positions of this lane's two rows
    float acc[NT][D / 16][4];
    float top[NT][2], l[NT][2], a1[NT][2], ones[NT][4];
    const float c2 = p.scale * kLog2e;
    const float c1 = kBf ? c2 : c2 * 16777216.f;
    int i = 0;  // tiles done
    while (i < count) {
      const int item_begin = begin + i - (at.tile - at.s.tile0), item_end = item_begin + at.s.tiles;
      const int stop = min(at.s.tile0 + at.s.tiles, at.tile + count - i);
      {
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
            l[nt][c] = a1[nt][c] = ones[nt][c] = ones[nt][c + 2] = 0.f;
          }
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[nt][x][c] = 0.f;
        }
      }

      bool lost = false;
      for (; at.tile < stop; ++at.tile, ++i) {
        const int slot = i % kDepth;
        const uint32_t tile = ring + slot * kBytes;
        if (!mbar_wait_bounded(full + 8 * slot, (i / kDepth) & 1, abort_flag)) {
          lost = true;
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
        ValueRow v0 = value_row(T::up(lds32(tile + off_v_pair(D, g))));
        ValueRow v1 = value_row(T::up(lds32(tile + off_v_pair(D, g + 8))));
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
        if (!whole) {
          // A row of values that stands for NaN counts through its scores where
          // it is seen; where it is not, scale and offset may be anything.
          const bool bad0 = !(fabsf(v0.at_8) <= 3.4e38f), bad1 = !(fabsf(v1.at_8) <= 3.4e38f);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int j = j0 + g + (c < 2 ? 0 : 8);
              const bool seen = j <= place[nt][c & 1] && j < at.s.len &&
                                (p.window == 0 || place[nt][c & 1] - j < p.window);
              if (!seen) {
                x[nt][c] = -CUDART_INF_F;
              } else if (c < 2 ? bad0 : bad1) {
                x[nt][c] = CUDART_NAN_F;
              }
            }
          if (bad0 || j0 + g >= at.s.len) v0.inv_s = v0.at_8 = 0.f;
          if (bad1 || j0 + g + 8 >= at.s.len) v1.inv_s = v1.at_8 = 0.f;
        }
        // The maximum moves only where an argument passes it by more than 8 (a
        // factor of 256, harmless in the sums), so most tiles need no exchange.
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) moves |= x[nt][c] - top[nt][c & 1] > 8.f;
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
              ones[nt][c] *= f[c];
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
        constexpr uint32_t kOnes = 0x3c003c00u;  // 1.0 twice: the sum of the rounded weights
        uint32_t wb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            w[c] = exp2_approx(x[nt][c] - top[nt][c & 1]);
            l[nt][c & 1] = fmaf(w[c], c < 2 ? v0.inv_s : v1.inv_s, l[nt][c & 1]);
            a1[nt][c & 1] = fmaf(w[c], c < 2 ? v0.at_8 : v1.at_8, a1[nt][c & 1]);
          }
          wb[nt][0] = transpose_8x8(Half::down(w[0], w[1]));
          wb[nt][1] = transpose_8x8(Half::down(w[2], w[3]));
          mma_16816<false>(ones[nt], kOnes, kOnes, kOnes, kOnes, wb[nt][0], wb[nt][1]);
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
      }
      if (lost) {
        if (lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
        // the copies that may be in flight land before the CTA's memory is handed on
        for (; i < issued; ++i)
          mbar_wait_bounded(full + 8 * (i % kDepth), (i / kDepth) & 1, drain_flag);
        break;
      }

      // --- the end of an item, or of the run --------------------------------
      const bool all = item_begin >= begin && item_end <= begin + count;
      const bool is_head = item_begin < begin && i < count;
      float* part = is_head ? reinterpret_cast<float*>(smem + Cfg::kOffParts) + warp * kPart
                            : reinterpret_cast<float*>(smem + warp * kDepth * kBytes);
      if (!all && lane == 0)
        segments[2 * warp + (is_head ? 0 : 1)] = {item_begin, item_end, at.b, at.head, at.chunk};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) {
            l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], s);
            a1[nt][c] += __shfl_xor_sync(0xffffffffu, a1[nt][c], s);
          }
          const float over = l[nt][c] == 0.f ? 0.f : 1.f / l[nt][c];
          // this lane has channels [D/8 g, D/8 (g + 1)) of the row
          float y[D / 8];
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            y[2 * x] = (fmaf(acc[nt][x][c], 16777216.f, -8.f * ones[nt][c]) + a1[nt][c]) * over;
            y[2 * x + 1] = (fmaf(acc[nt][x][c + 2], 1048576.f, -8.f * ones[nt][c]) + a1[nt][c]) * over;
          }
          const int r = nt * 8 + 2 * t + c, row = at.chunk * kRows + r;
          if (row >= at.s.n * p.group) continue;
          if (all) {
            uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(at.s.first + row / p.group) * p.q_heads +
                                         at.head * p.group + row % p.group) * D + D / 8 * g);
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
      if (i < count) next_item<kRows>(p, at);
    }
  }
  __syncthreads();
  if (*abort_flag) return;

  // --- parts of this CTA's warps, joined -------------------------------------
  auto part_of = [&](int s) -> const float* {
    return s & 1 ? reinterpret_cast<const float*>(smem + (s >> 1) * kDepth * kBytes)
                 : reinterpret_cast<const float*>(smem + Cfg::kOffParts) + (s >> 1) * kPart;
  };
  auto store = [&](const Segment& seg, const Span& sp, int r, int c, const float4& x) {
    const int row = seg.chunk * kRows + r;
    *reinterpret_cast<uint2*>(
        p.out + 2 * ((static_cast<int64_t>(sp.first + row / p.group) * p.q_heads + seg.head * p.group +
                      row % p.group) * D + c)) = make_uint2(T::down(x.x, x.y), T::down(x.z, x.w));
  };
  int open[2] = {-1, -1};  // segments of the items that other CTAs share: from before, into the next
#pragma unroll 1
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
    const int side = seg.begin < cta_begin ? 0 : 1;
    float* to = p.partials + (2ll * blockIdx.x + side) * kPart;
    if (!all) open[side] = s0;
#pragma unroll 1
    for (int r = threadIdx.x; r < rows; r += Cfg::kThreads) {
      float m = kLowest, sum = 0.f;
#pragma unroll 1
      for (int s = s0; s < s1; ++s)
        if (segments[s].begin >= 0) m = fmaxf(m, part_of(s)[kRows * D + r]);
#pragma unroll 1
      for (int s = s0; s < s1; ++s) {
        if (segments[s].begin < 0) continue;
        const float w = part_of(s)[kRows * D + kRows + r] * exp2_approx(part_of(s)[kRows * D + r] - m);
        join_w[s * kRows + r] = w;
        sum += w;
      }
      const float over = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
      for (int s = s0; s < s1; ++s) join_w[s * kRows + r] *= over;
      if (!all) to[kRows * D + r] = m, to[kRows * D + kRows + r] = sum;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * (D / 4); i += Cfg::kThreads) {
      const int r = i / (D / 4);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int s = s0; s < s1; ++s) {
        if (segments[s].begin < 0) continue;
        const float w = join_w[s * kRows + r];
        const float4 v = *reinterpret_cast<const float4*>(part_of(s) + 4 * i);
        x = make_float4(fmaf(w, v.x, x.x), fmaf(w, v.y, x.y), fmaf(w, v.z, x.z), fmaf(w, v.w, x.w));
      }
      if (all) {
        store(seg, sp, r, 4 * (i % (D / 4)), x);
      } else {
        *reinterpret_cast<float4*>(to + 4 * i) = x;
      }
    }
    s0 = s1;
  }
  if (open[0] < 0 && open[1] < 0) return;

  // --- items of several CTAs: the last to bring its part joins them ----------
  __threadfence();
  __syncthreads();
  float* weights = reinterpret_cast<float*>(smem);               // [ctas][rows]: the rings are done with
  float4* sheets = reinterpret_cast<float4*>(smem + Cfg::kRing); // [sheets][rows * D / 4]: so are the parts
  static_assert(Cfg::kThreads * 16 <= Cfg::kWarps * kPart * 4, "sheets");
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    if (open[side] < 0) continue;
    const Segment seg = segments[open[side]];
    const int c0 = seg.begin / quota, c1 = (seg.end - 1) / quota;
    if (threadIdx.x == 0) *last_flag = atomicAdd(p.counters + c0, 1) == c1 - c0;
    __syncthreads();
    if (*last_flag) {
      __threadfence();
      if (threadIdx.x == 0) p.counters[c0] = 0;
      const Span sp = span_of<kRows>(p, seg.b);
      const int rows = min(kRows, sp.n * p.group - seg.chunk * kRows), ctas = c1 - c0 + 1;
      auto from = [&](int c) -> const float* {
        return p.partials + (2ll * (c0 + c) + (c == 0 ? 1 : 0)) * kPart;
      };
#pragma unroll 1
      for (int r = warp; r < rows; r += Cfg::kWarps) {  // a warp a row
        float m = kLowest, sum = 0.f;
#pragma unroll 1
        for (int c = lane; c < ctas; c += 32) m = fmaxf(m, __ldcg(from(c) + kRows * D + r));
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
#pragma unroll 1
        for (int c = lane; c < ctas; c += 32) {
          const float w = __ldcg(from(c) + kRows * D + kRows + r) * exp2_approx(__ldcg(from(c) + kRows * D + r) - m);
          weights[c * kRows + r] = w;
          sum += w;
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        const float over = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
        for (int c = lane; c < ctas; c += 32) weights[c * kRows + r] *= over;
      }
      __syncthreads();
      // few rows: several sheets of threads, each over some of the CTAs
      const int sheet = rows * (D / 4), count = max(1, min(256 / sheet, ctas));
#pragma unroll 1
      for (int i0 = threadIdx.x; i0 < count * sheet; i0 += Cfg::kThreads) {
        const int i = i0 % sheet, r = i / (D / 4);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = i0 / sheet; c < ctas; c += count) {
          const float w = weights[c * kRows + r];
          const float4 v = __ldcg(reinterpret_cast<const float4*>(from(c) + 4 * i));
          x = make_float4(fmaf(w, v.x, x.x), fmaf(w, v.y, x.y), fmaf(w, v.z, x.z), fmaf(w, v.w, x.w));
        }
        if (count == 1) {
          store(seg, sp, r, 4 * (i % (D / 4)), x);
        } else {
          sheets[i0] = x;
        }
      }
      if (count > 1) {
        __syncthreads();
#pragma unroll 1
        for (int i = threadIdx.x; i < sheet; i += Cfg::kThreads) {
          float4 x = sheets[i];
#pragma unroll 1
          for (int c = 1; c < count; ++c) {
            const float4 v = sheets[c * sheet + i];
            x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
          }
          store(seg, sp, i / (D / 4), 4 * (i % (D / 4)), x);
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace kv4
}  // namespace sm100
