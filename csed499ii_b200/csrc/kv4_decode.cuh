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
// the weights w = p s.  They go into the products as halves: one for a bf16
// model (11 bits, where a result has 8), the sum of two for an fp16 model (22
// bits; with one the error of a result was 1.2 to 1.5 times that of a result
// rounded once, and 16 x 1024 tokens of 32 heads took 25.2 us instead of 27.6).
// The exponential gives w itself, its argument is the score plus log2 s, and the
// running maximum is that of these arguments: a half then holds the weights that
// matter whatever sizes the values have, and p is w / s in 32 bits.  sum(p) and
// the offset term take the weights as they are, and the codes act as if centred
// on 7.5: a rounding error meets at most 7.5 steps of its row's scale, never its
// offset, which can be 2^15 scales (with rounded weights in the offset term one
// wide row among 20000 narrow ones moved the result by 5 times what its rounding
// allows).
//
// mma.m16n8k16 takes 16 tokens (scores) or 16 channels (result) as its rows
// and 8 query rows as its columns; the 8 query heads of a group fill it.  Codes
// become 16-bit operands with one AND per two of them: an integer c < 16 in
// the low bits of a half is the subnormal c * 2^-24, and c << 4 is c * 2^-20,
// both exact in the product; for bf16 queries the codes are OR-ed into the
// mantissa of 128 (128 + c) and the offset term takes the 128 back.
//
// Work is dealt in steps of two tiles: all steps of all (request, head) pairs in
// a row, cut into equal runs, one per warp, whatever the lengths are.  A warp
// streams its run through its own ring of bulk copies, over the borders of
// pairs; what it has of a pair that other warps share is joined in the CTA
// through shared memory, and between CTAs through the workspace by whichever
// finishes last, in CTA order, so results do not depend on timing.
//
// Measured at 8 key/value heads of 128 and 8 query heads each: one request of
// 131072 tokens (142.8 MB, fp16) in 50.6 us, 64 of up to 8192 (256 MB, bf16) in 82 us,
// 2.8 and 3.1 TB/s of 6.55 measured for a copy.  Instructions bound it: 372 a warp and
// tile in the first (its start and joins among them), two fifths of the time on the
// integer pipe to turn codes into operands, at the 51% of issue slots that 16 warps of
// 128 registers fill.  Those registers are not quite enough: D = 128 with one column
// tile spills 88 bytes for fp16 models and 76 for bf16, D = 64 with two 448 and 256
// (8 warps of 255 do not spill there: from 5% less time to 15% more).  Launch, first
// bytes, and joins in the CTA and over CTAs are about 16 us of the 50.
#pragma once

#include <math_constants.h>

#include "kv4_format.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kDecodeBatch = 1024;    // requests of a launch: 4 bytes of shared memory each
constexpr int kStepTokens = 2 * kTile;  // a step: two tiles
constexpr int kLeastSteps = 16;         // of a CTA: fewer are not worth sharing an item
constexpr int kRoundSteps = 32;         // a CTA takes up to so many more to end with an item

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
  int pad;               // 1: rows past the last request are set to zero; 2: those before the first are
  int alone;             // 1: no other kernel serves the requests that are left alone
  int q_heads;
  int group;             // query heads per key/value head
  int window;            // 0: none
  int most;              // requests with more query rows a group than this are left alone
  float scale;
  int* counters;         // [grid], zero between launches
  float* partials;       // [grid][2] parts
  int* status;
  int stalled;           // CTA whose first warp waits for more than comes (-1: none), for tests
};

template <int D, int NT>
struct DecodeCfg {
  // One CTA an SM: the fewer parts an item has, the sooner they are joined.
  static constexpr int kWarps = D == 128 && NT == 2 ? 8 : 16;  // 252 registers, 128
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kDepth = 2;             // steps in a warp's ring
  static constexpr int kSlot = 2 * tile_bytes(D);
  static constexpr int kRows = 8 * NT;         // query rows of an item
  static constexpr int kPart = kRows * (D + 2);  // floats: results, maxima, sums
  static constexpr int kRing = kWarps * kDepth * kSlot;
  static constexpr int kOffParts = kRing;
  static constexpr int kOffTokens = kOffParts + kWarps * kPart * 4;
  static constexpr int kOffPre = kOffTokens + kWarps * 32 * 20;
  static constexpr int kOffMisc = kOffPre + kDecodeBatch * 4;
  static constexpr int kSmem = kOffMisc + 1280;
  // a warp's last part takes the place of its ring
  static_assert(kPart * 4 <= kDepth * kSlot, "part does not fit the ring");
  static_assert((kWarps + kRows) * (2 * D + 8) * 4 <= kRing, "sheets do not fit the rings");
};

// Tokens of a request: what its table can hold, and few enough that a step past the
// last one still has a 32-bit position.
__device__ __forceinline__ int held_tokens(int len, int width, int page_size) {
  const int64_t room = min(static_cast<int64_t>(width) * page_size, static_cast<int64_t>(0x7fffff00));
  return max(static_cast<int>(min(static_cast<int64_t>(len), room)), 0);
}

// What a launch knows about one request.
struct Span {
  int first, n, len;    // query rows, tokens
  int step0, steps;     // that any of its rows sees
  int chunks;           // of query rows
};

template <int ROWS>
__device__ __forceinline__ Span span_of(const DecodeParams& p, int b) {
  Span s;
  s.first = p.starts ? min(max(p.starts[b], 0), p.rows) : p.row0 + b;
  s.n = p.starts ? min(p.starts[b + 1], p.rows) - s.first : 1;
  s.len = held_tokens(p.lens[b], p.width, p.cache.page_size);
  const int64_t rows = static_cast<int64_t>(s.n) * p.group;
  const bool mine = s.n > 0 && rows <= p.most;
  s.chunks = mine ? (static_cast<int>(rows) + ROWS - 1) / ROWS : 0;
  const int from = p.window && s.len - s.n >= p.window ? s.len - s.n - p.window + 1 : 0;
  s.step0 = from / kStepTokens;
  s.steps = mine && s.len > 0 ? (s.len - 1) / kStepTokens + 1 - s.step0 : 0;
  return s;
}

// One item (a request, a key/value head, ROWS of its query rows) and a step.
struct Walk {
  Span s;
  int b, head, chunk, step;  // step of the request
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
  const int steps = max(w.s.steps, 1);
  const int item = off / steps;
  w.step = w.s.step0 + off - item * steps;
  w.head = item / max(w.s.chunks, 1);
  w.chunk = item - w.head * max(w.s.chunks, 1);
  return w;
}

// To the first step of the next item; only called while there is one.
template <int ROWS>
__device__ __forceinline__ void next_item(const DecodeParams& p, Walk& w) {
  if (++w.chunk == w.s.chunks) {
    w.chunk = 0;
    if (++w.head == p.cache.heads) {
      w.head = 0;
      do {
        w.s = span_of<ROWS>(p, ++w.b);
      } while (w.s.steps == 0 && w.b + 1 < p.batch);
    }
  }
  w.step = w.s.step0;
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

// The same with a fresh accumulator.
template <bool BF16>
__device__ __forceinline__ void mma_16816_z(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  }
}

// The same for halves, begun with (c0, c1, c2, c3).
__device__ __forceinline__ void mma_16816_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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

// The middle of the codes: values are held as what they are off it and their value
// at it, so that for values around zero neither's sum is much larger than the result.
constexpr float kMid = 7.5f;

// What the weights need to know of a row of values: its scale's logarithm and
// reciprocal, and its value at code kMid over the scale.
//
// The sum of the weights is kept as sum(w / s), so 1 / s has to leave room for a
// long sum in 32 bits: a scale below 2^-90 (bf16 values below 2^-75) counts as
// 2^-90.  One below 2^-30 of the offset changes no value that 32 bits hold.  A
// row without a scale has all codes 0, so any scale tells the same values; its
// weights are to outweigh nobody else's, who would lose theirs in the rounding to
// half: 2^-10 of the offset is below what its own value adds to the result, and
// 2^-60 for a row of zeros is in the middle of what scales can be.
struct ValueRow {
  float log_s, inv_s, at_mid;
};
__device__ __forceinline__ ValueRow value_row(float2 pair) {
  const float s = pair.x > 0.f ? fmaxf(fmaxf(pair.x, fabsf(pair.y) * 0x1p-30f), 0x1p-90f)
                               : fmaxf(fabsf(pair.y) * 0x1p-10f, 0x1p-60f);
  ValueRow r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r.log_s) : "f"(s));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv_s) : "f"(s));
  r.at_mid = fmaf(pair.y, r.inv_s, kMid);
  return r;
}

// What there is of an item in one place: results (already divided by the sum),
// the running maximum of the weights' arguments (less kWeightTop) and the sum of
// the weights over 2 to it.
struct Segment {
  int begin, end;        // the item's place in the row of all steps; begin < 0: none
  int b, head, chunk;
};

constexpr float kLowest = -3.0e38f;

// A weight in half is 2^kWeightTop where its argument is the maximum, which moves
// once an argument passes it by kLag: weights reach 2^kMoveAt, and what lies 2^-31
// below the largest is still held.  With 1 for the largest a half rounds below
// 2^-14 and ends at 2^-24: 32767 keys that weigh 2^-20 of a first one, 2^-5
// together, had errors of 1.4 times what the rounding of weights allows, and keys
// that weigh 2^-26 were lost.
constexpr float kWeightTop = 7.f, kLag = 8.f, kMoveAt = kWeightTop + kLag;

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
  return x;
}

// Channels [N lane, N (lane + 1)) of a row.
template <int N>
struct Slice {
  float x[N];
  __device__ __forceinline__ void add(float w, const float* row, int lane) {
    if constexpr (N == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(row) + lane);
      x[0] = fmaf(w, v.x, x[0]), x[1] = fmaf(w, v.y, x[1]);
      x[2] = fmaf(w, v.z, x[2]), x[3] = fmaf(w, v.w, x[3]);
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(row) + lane);
      x[0] = fmaf(w, v.x, x[0]), x[1] = fmaf(w, v.y, x[1]);
    }
  }
  __device__ __forceinline__ void add_shared(float w, const float* row, int lane) {
    if constexpr (N == 4) {
      const float4 v = reinterpret_cast<const float4*>(row)[lane];
      x[0] = fmaf(w, v.x, x[0]), x[1] = fmaf(w, v.y, x[1]);
      x[2] = fmaf(w, v.z, x[2]), x[3] = fmaf(w, v.w, x[3]);
    } else {
      const float2 v = reinterpret_cast<const float2*>(row)[lane];
      x[0] = fmaf(w, v.x, x[0]), x[1] = fmaf(w, v.y, x[1]);
    }
  }
  __device__ __forceinline__ void put(float* row, int lane) const {
    if constexpr (N == 4) {
      reinterpret_cast<float4*>(row)[lane] = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      reinterpret_cast<float2*>(row)[lane] = make_float2(x[0], x[1]);
    }
  }
};

template <class T, int D, int NT>
__global__ void __launch_bounds__(DecodeCfg<D, NT>::kThreads, 1)
    kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  using Cfg = DecodeCfg<D, NT>;
  constexpr int kWarps = Cfg::kWarps, kRows = Cfg::kRows, kPart = Cfg::kPart, kDepth = Cfg::kDepth;
  constexpr int kBytes = tile_bytes(D), kSlot = Cfg::kSlot;
  constexpr int kWords = D / 32;  // code words of a lane in a row of keys
  constexpr bool kBf = T::kBf16;
  constexpr int kTerms = kBf ? 1 : 2;  // halves that a weight is the sum of
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre = reinterpret_cast<int*>(smem + Cfg::kOffPre);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffMisc);            // [warps][depth]
  int* there = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 256);               // [warps][depth]
  Segment* segments = reinterpret_cast<Segment*>(smem + Cfg::kOffMisc + 384);    // [warps][2]
  int* sums = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 1024);               // [3][warps]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kOffMisc + 1216);
  volatile int* drain_flag = abort_flag + 1;
  int* last_flag = reinterpret_cast<int*>(smem + Cfg::kOffMisc + 1224);          // [2]
  static_assert(sizeof(Segment) * 32 <= 640, "shared memory");

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  if (lane < kDepth)
    mbar_init(smem_addr(bars + kDepth * warp + lane), warp == 0 && static_cast<int>(blockIdx.x) == p.stalled ? 2 : 1);
  if (lane < 2) segments[2 * warp + lane].begin = -1;
  if (threadIdx.x == 0) *abort_flag = *drain_flag = 0;
  fence_mbar_init();

  grid_dependency_wait();
  grid_dependency_launch();

  // --- the row of all steps: where each request's end is -------------------
  int total = 0;  // the host keeps it below 2^30
  int longest = 0, shortest = 0x7fffffff;  // items
  for (int b0 = 0; b0 < p.batch; b0 += Cfg::kThreads) {
    const int b = b0 + threadIdx.x;
    int x = 0, most = 0, least = 0x7fffffff;
    if (b < p.batch) {
      const Span s = span_of<kRows>(p, b);
      x = p.cache.heads * s.chunks * s.steps;
      most = s.steps;
      if (x > 0) least = s.steps;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, i);
      if (lane >= i) x += y;
    }
    if (lane == 31) sums[warp] = x, sums[kWarps + warp] = most, sums[2 * kWarps + warp] = least;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i == warp) x += all;
      all += sums[i];
      longest = max(longest, sums[kWarps + i]);
      shortest = min(shortest, sums[2 * kWarps + i]);
    }
    if (b < p.batch) pre[b] = total + x;
    total += all;
    __syncthreads();
  }

  // --- rows that see nothing, and rows that nobody serves ---------------------
  {
    const int64_t row_bytes = 2ll * p.q_heads * D;
#pragma unroll 1
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (pre[b] != (b ? pre[b - 1] : 0)) continue;
      const Span s = span_of<kRows>(p, b);
      if (s.chunks == 0 && (s.n <= 0 || !p.alone)) continue;
      const uint32_t x = s.chunks == 0 ? 0x7fff7fffu : 0u;  // NaN in either type
#pragma unroll 1
      for (int64_t i = 16 * threadIdx.x; i < s.n * row_bytes; i += 16 * Cfg::kThreads)
        *reinterpret_cast<uint4*>(p.out + s.first * row_bytes + i) = make_uint4(x, x, x, x);
    }
    const int before = p.starts && p.pad & 2 ? min(max(p.batch ? p.starts[0] : 0, 0), p.rows) : 0;
    const int end = !p.starts || !(p.pad & 1) ? p.rows : min(max(p.batch ? p.starts[p.batch] : 0, before), p.rows);
#pragma unroll 1
    for (int i = blockIdx.x; i < before + p.rows - end; i += gridDim.x) {
      const int64_t row = i < before ? i : end + i - before;
#pragma unroll 1
      for (int64_t j = 16 * threadIdx.x; j < row_bytes; j += 16 * Cfg::kThreads)
        *reinterpret_cast<uint4*>(p.out + row * row_bytes + j) = make_uint4(0, 0, 0, 0);
    }
  }

  // --- this CTA's steps -----------------------------------------------------
  // Joining an item over CTAs costs about as much as kRoundSteps steps of one.
  // Where all items are as long, a CTA's share is rounded up to whole ones if
  // that takes no more, or else every item gets the same CTAs to itself.  (16
  // requests of 32 heads: 27.6 us at 1024 tokens each, 28.1 at 1000 to 1015.)
  const int ctas = gridDim.x, cta = blockIdx.x;
  int quota = (total + ctas - 1) / ctas, per_item = 0;  // CTAs that an item has to itself
  const bool even = longest == shortest;
  const int whole = even ? (quota + longest - 1) / longest * longest : 0;
  if (even && whole - quota <= kRoundSteps) {
    quota = whole;
  } else if (even && total / longest <= ctas) {
    quota = max((longest - 1) / (ctas / (total / longest)) + 1, kLeastSteps);
    per_item = (longest - 1) / quota + 1;
  } else {
    quota = max(quota, kLeastSteps);
  }
  if (per_item ? cta / per_item >= total / longest : static_cast<int64_t>(quota) * cta >= total) return;
  const int cta_begin = per_item ? cta / per_item * longest + cta % per_item * quota : quota * cta;
  const int cta_end = min(cta_begin + quota, per_item ? (cta / per_item + 1) * longest : total);
  // first and last CTA of the item in [begin, end)
  auto first_cta = [&](int begin) { return per_item ? begin / longest * per_item : begin / quota; };
  auto last_cta = [&](int begin, int end) {
    return per_item ? begin / longest * per_item + per_item - 1 : (end - 1) / quota;
  };
  const int share = (cta_end - cta_begin + kWarps - 1) / kWarps;
  const int begin = min(cta_begin + share * warp, cta_end);
  const int count = min(begin + share, cta_end) - begin;

  // --- this warp's run ------------------------------------------------------
  if (count > 0) {
    const uint32_t ring = smem_addr(smem) + warp * kDepth * kSlot;
    const uint32_t full = smem_addr(bars + kDepth * warp);
    // of each token of a step: key scale, key offset, log2 of the value scale
    float* tokens = reinterpret_cast<float*>(smem + Cfg::kOffTokens) + warp * 160;
    float2* token_sums = reinterpret_cast<float2*>(tokens + 96);  // 1 / value scale, value at code kMid / scale
    Walk at = walk_to<kRows>(p, pre, begin);
    // the first queries are on their way while the first pages are looked up
    {
      const int r = at.chunk * kRows + g;
      if (r < at.s.n * p.group)
        prefetch_l1(p.q + 2 * (p.q_row * (at.s.first + r / p.group) +
                               p.q_head * (at.head * p.group + r % p.group) + t * (D / 4)));
    }

    // The copies run ahead of the work: `in` is the place of the next one, and
    // its pages are looked up a step early.
    Walk in = at;
    const int per_page = p.cache.page_size / kTile;
    const uint64_t policy = policy_evict_first();
    int issued = 0, entry, nth, page0, page1;  // nth tile of the table's entry
    auto look_up = [&](bool both) {
      const int* table = p.tables + p.table_stride * in.b + entry;
      if (both) page0 = table[0];
      page1 = page0;
      if (nth + 1 == per_page) page1 = (2 * in.step + 1) * kTile < in.s.len ? table[1] : -1;
    };
    auto start = [&]() {
      entry = 2 * in.step / per_page;
      nth = 2 * in.step - entry * per_page;
      look_up(true);
    };
    auto issue = [&]() {
      const int slot = issued % kDepth;
      if (lane == 0) {
        const bool ok0 = static_cast<uint32_t>(page0) < static_cast<uint32_t>(p.cache.pages);
        const bool ok1 = static_cast<uint32_t>(page1) < static_cast<uint32_t>(p.cache.pages);
        const uint32_t dst = ring + slot * kSlot, bar = full + 8 * slot;
        there[warp * kDepth + slot] = (ok0 ? 1 : 0) | (ok1 ? 2 : 0);
        if (nth + 1 < per_page && ok0) {  // both tiles of one page
          mbar_arrive_expect_tx(bar, 2 * kBytes);
          bulk_g2s(dst, p.cache.tile<D>(page0, in.head, nth), 2 * kBytes, bar, policy);
        } else if (ok0 || ok1) {
          mbar_arrive_expect_tx(bar, (ok0 ? kBytes : 0) + (ok1 ? kBytes : 0));
          if (ok0) bulk_g2s(dst, p.cache.tile<D>(page0, in.head, nth), kBytes, bar, policy);
          if (ok1) bulk_g2s(dst + kBytes, p.cache.page_tiles<D>(page1, in.head), kBytes, bar, policy);
        } else {
          mbar_arrive(bar);
        }
      }
      if (++issued == count) return;
      if (++in.step == in.s.step0 + in.s.steps) {
        next_item<kRows>(p, in);
        start();
      } else {
        nth += 2;
        const int old = entry;
        while (nth >= per_page) nth -= per_page, ++entry;
        look_up(entry != old);
      }
    };
    start();
    for (int i = 0; i < kDepth && issued < count; ++i) issue();

    uint32_t qe[NT][kWords][2], qo[NT][kWords][2];  // queries: even and odd nibbles' channels
    float sumq[NT][2];
    int place[NT][2];                               // positions of this lane's two rows
    float acc[NT][D / 16][4];
    float top[NT][2], l[NT][2], a1[NT][2];
    const float c2 = p.scale * kLog2e;
    const float c1 = kBf ? c2 : c2 * 16777216.f;
    int i = 0;  // steps done
    while (i < count) {
      const int item_begin = begin + i - (at.step - at.s.step0), item_end = item_begin + at.s.steps;
      const int stop = min(at.s.step0 + at.s.steps, at.step + count - i);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = at.chunk * kRows + nt * 8 + g;
        const int token = r / p.group, h = at.head * p.group + r - token * p.group;
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
              x = make_uint4(src[8 * w] | src[8 * w + 1] << 16, src[8 * w + 2] | src[8 * w + 3] << 16,
                             src[8 * w + 4] | src[8 * w + 5] << 16, src[8 * w + 6] | src[8 * w + 7] << 16);
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
          l[nt][c] = a1[nt][c] = 0.f;
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[nt][x][c] = 0.f;
      }

      bool lost = false;
      for (; at.step < stop; ++at.step, ++i) {
        const int slot = i % kDepth;
        const uint32_t data = ring + slot * kSlot;
        if (!mbar_wait_bounded(full + 8 * slot, (i / kDepth) & 1, abort_flag)) {
          lost = true;
          break;
        }
        const int j0 = at.step * kStepTokens;
        // Scale and offset of this lane's token, for all lanes.  A token that is
        // not there weighs nothing, whatever lies in its place; a row of values
        // that stands for NaN counts through its scores.
        {
          const uint32_t tile = data + (lane >> 4) * kBytes;
          const float2 kp = T::up(lds32(tile + off_k_pair(D, lane & 15)));
          const ValueRow v = value_row(T::up(lds32(tile + off_v_pair(D, lane & 15))));
          float4 x = make_float4(kp.x * c1, (kBf ? fmaf(kp.x, -128.f, kp.y) : kp.y) * c2, v.log_s, v.inv_s);
          float at_mid = v.at_mid;
          if (!(fabsf(at_mid) <= 3.4e38f)) x.y = CUDART_NAN_F, x.w = at_mid = 0.f;
          if (j0 + lane >= at.s.len || !(there[warp * kDepth + slot] >> (lane >> 4) & 1))
            x = make_float4(0.f, 0.f, -CUDART_INF_F, 0.f), at_mid = 0.f;
          tokens[lane] = x.x;
          tokens[32 + lane] = x.y;
          tokens[64 + lane] = x.z;
          token_sums[lane] = make_float2(x.w, at_mid);
        }
        __syncwarp();
        // the arguments of the weights
        float x[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t tile = data + u * kBytes;
          uint32_t k0[kWords], k1[kWords];
          if constexpr (D == 128) {
            const uint4 y = lds128(tile + 16 * lane), z = lds128(tile + 512 + 16 * lane);
            k0[0] = y.x, k0[1] = y.y, k0[2] = y.z, k0[3] = y.w;
            k1[0] = z.x, k1[1] = z.y, k1[2] = z.z, k1[3] = z.w;
          } else {
            const uint2 y = lds64(tile + 8 * lane), z = lds64(tile + 256 + 8 * lane);
            k0[0] = y.x, k0[1] = y.y;
            k1[0] = z.x, k1[1] = z.y;
          }
          float e[NT][4], o[NT][4];
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const uint32_t h0 = k0[w] >> 8, h1 = k1[w] >> 8;
            const uint32_t ea0 = key_even<kBf>(k0[w]), ea1 = key_even<kBf>(k1[w]);
            const uint32_t ea2 = key_even<kBf>(h0), ea3 = key_even<kBf>(h1);
            const uint32_t oa0 = key_odd<kBf>(k0[w]), oa1 = key_odd<kBf>(k1[w]);
            const uint32_t oa2 = key_odd<kBf>(h0), oa3 = key_odd<kBf>(h1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (w == 0) {
                mma_16816_z<kBf>(e[nt], ea0, ea1, ea2, ea3, qe[nt][w][0], qe[nt][w][1]);
                mma_16816_z<kBf>(o[nt], oa0, oa1, oa2, oa3, qo[nt][w][0], qo[nt][w][1]);
              } else {
                mma_16816<kBf>(e[nt], ea0, ea1, ea2, ea3, qe[nt][w][0], qe[nt][w][1]);
                mma_16816<kBf>(o[nt], oa0, oa1, oa2, oa3, qo[nt][w][0], qo[nt][w][1]);
              }
            }
          }
          const float3 y = make_float3(tokens[16 * u + g], tokens[32 + 16 * u + g], tokens[64 + 16 * u + g]);
          const float3 z = make_float3(tokens[16 * u + g + 8], tokens[40 + 16 * u + g], tokens[72 + 16 * u + g]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float dot = fmaf(o[nt][c], kBf ? 1.f : 0.0625f, e[nt][c]);
              x[u][nt][c] = c < 2 ? fmaf(y.x, dot, fmaf(y.y, sumq[nt][c & 1], y.z))
                                  : fmaf(z.x, dot, fmaf(z.y, sumq[nt][c & 1], z.z));
            }
        }
        // rows that see less than others
        if ((at.s.n > 1 && j0 + kStepTokens > at.s.len - at.s.n + 1) || (p.window != 0 && at.s.len - j0 > p.window)) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int j = j0 + 16 * u + g + (c < 2 ? 0 : 8);
                if (j > place[nt][c & 1] || (p.window != 0 && place[nt][c & 1] - j >= p.window))
                  x[u][nt][c] = -CUDART_INF_F;
              }
        }
        // The maximum moves only where an argument passes it by more than kLag, so
        // most steps need no exchange.
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            moves |= fmaxf(fmaxf(x[0][nt][c], x[0][nt][c + 2]), fmaxf(x[1][nt][c], x[1][nt][c + 2])) >
                     top[nt][c] + kMoveAt;
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float m = fmaxf(fmaxf(x[0][nt][c], x[0][nt][c + 2]), fmaxf(x[1][nt][c], x[1][nt][c + 2]));
              m = fmaxf(top[nt][c], m - kWeightTop);
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              f[c] = exp2_approx(top[nt][c] - m);
              top[nt][c] = m;
              l[nt][c] *= f[c];
              a1[nt][c] *= f[c];
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
        // Weights, and their sums.
        constexpr uint32_t kOnes = 0x3c003c00u;  // 1.0 twice
        uint32_t wb[2][NT][kTerms][2];
        float ones[NT][4];  // the step's sum of the rounded weights
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float2 s0 = token_sums[16 * u + g], s1 = token_sums[16 * u + g + 8];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              w[c] = exp2_approx(x[u][nt][c] - top[nt][c & 1]);
              l[nt][c & 1] = fmaf(w[c], c < 2 ? s0.x : s1.x, l[nt][c & 1]);
              a1[nt][c & 1] = fmaf(w[c], c < 2 ? s0.y : s1.y, a1[nt][c & 1]);
            }
            const uint32_t w01 = Half::down(w[0], w[1]), w23 = Half::down(w[2], w[3]);
            wb[u][nt][0][0] = transpose_8x8(w01);
            wb[u][nt][0][1] = transpose_8x8(w23);
            if constexpr (kTerms == 2) {
              const float2 r01 = Half::up(w01), r23 = Half::up(w23);
              w[0] -= r01.x, w[1] -= r01.y, w[2] -= r23.x, w[3] -= r23.y;
#pragma unroll
              for (int c = 0; c < 4; ++c) a1[nt][c & 1] = fmaf(-kMid, w[c], a1[nt][c & 1]);
              wb[u][nt][kTerms - 1][0] = transpose_8x8(Half::down(w[0], w[1]));
              wb[u][nt][kTerms - 1][1] = transpose_8x8(Half::down(w[2], w[3]));
            }
            if (u == 0) {
              mma_16816_z<false>(ones[nt], kOnes, kOnes, kOnes, kOnes, wb[u][nt][0][0], wb[u][nt][0][1]);
            } else {
              mma_16816<false>(ones[nt], kOnes, kOnes, kOnes, kOnes, wb[u][nt][0][0], wb[u][nt][0][1]);
            }
          }
        }
        // Result.  A step's products are summed by themselves, begun with kMid times
        // the rounded weights taken off, and added to the others in binary32: the tensor
        // cores cut a sum off at 2^-23 of it with every product added, a bias over a
        // long run of one warp (131071 keys that weigh 2^-26 of a first one had 1.13
        // times the error that the rounding of weights allows).  It takes 4% of the time.
        constexpr float kLess = -kMid * 0x1p-24f;
        constexpr int kOctets = D / 64;
        uint32_t va[2][kOctets], vb[2][kOctets], vc[2][kOctets], vd[2][kOctets];  // tokens 2t, 2t+1, 2t+8, 2t+9
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t tile = data + u * kBytes;
          if constexpr (D == 128) {
            const uint4 y = lds128(tile + 8 * D + 16 * lane), z = lds128(tile + 12 * D + 16 * lane);
            va[u][0] = y.x, va[u][1] = y.y, vb[u][0] = y.z, vb[u][1] = y.w;
            vc[u][0] = z.x, vc[u][1] = z.y, vd[u][0] = z.z, vd[u][1] = z.w;
          } else {
            const uint2 y = lds64(tile + 8 * D + 8 * lane), z = lds64(tile + 12 * D + 8 * lane);
            va[u][0] = y.x, vb[u][0] = y.y;
            vc[u][0] = z.x, vd[u][0] = z.y;
          }
        }
#pragma unroll
        for (int o = 0; o < kOctets; ++o)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float sums[NT][2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t sel = half ? 0x7632 : 0x5410;
              const uint32_t y = prmt_b32(va[u][o], vb[u][o], sel), z = prmt_b32(vc[u][o], vd[u][o], sel);
#pragma unroll
              for (int odd = 0; odd < 2; ++odd) {
                const uint32_t yo = odd ? y >> 8 : y, zo = odd ? z >> 8 : z;
                const uint32_t c0 = yo & 0x000f000fu, c1 = yo & 0x00f000f0u;
                const uint32_t c2 = zo & 0x000f000fu, c3 = zo & 0x00f000f0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int i = 0; i < kTerms; ++i) {
                    float(&to)[4] = sums[nt][odd];
                    const uint32_t b0 = wb[u][nt][i][0], b1 = wb[u][nt][i][1];
                    if (u == 0 && i == 0) {
                      mma_16816_from(to, c0, c1, c2, c3, b0, b1, ones[nt][0] * kLess, ones[nt][1] * kLess,
                                     ones[nt][0] * (16.f * kLess), ones[nt][1] * (16.f * kLess));
                    } else {
                      mma_16816<false>(to, c0, c1, c2, c3, b0, b1);
                    }
                  }
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int odd = 0; odd < 2; ++odd)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[nt][4 * o + 2 * half + odd][c] += sums[nt][odd][c];
          }
        __syncwarp();  // the slot and the tokens' numbers are read
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
                            : reinterpret_cast<float*>(smem + warp * kDepth * kSlot);
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
          const float rest = a1[nt][c];
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            y[2 * x] = fmaf(acc[nt][x][c], 16777216.f, rest) * over;
            y[2 * x + 1] = fmaf(acc[nt][x][c + 2], 1048576.f, rest) * over;
          }
          const int r = nt * 8 + 2 * t + c, row = at.chunk * kRows + r;
          if (row >= at.s.n * p.group) continue;
          if (all) {
            const int token = row / p.group;
            uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(at.s.first + token) * p.q_heads +
                                         at.head * p.group + row - token * p.group) * D + D / 8 * g);
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

  // --- parts of this CTA's warps, joined: a warp a row -------------------------
  using Row = Slice<D / 32>;
  auto store = [&](const Segment& seg, const Span& sp, int r, const Row& x) {
    const int row = seg.chunk * kRows + r, token = row / p.group;
    uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(sp.first + token) * p.q_heads + seg.head * p.group +
                                 row - token * p.group) * D + D / 32 * lane);
    if constexpr (D == 128) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(T::down(x.x[0], x.x[1]), T::down(x.x[2], x.x[3]));
    } else {
      *reinterpret_cast<uint32_t*>(dst) = T::down(x.x[0], x.x[1]);
    }
  };
  auto part_of = [&](int s) -> const float* {
    return s & 1 ? reinterpret_cast<const float*>(smem + (s >> 1) * kDepth * kSlot)
                 : reinterpret_cast<const float*>(smem + Cfg::kOffParts) + (s >> 1) * kPart;
  };
  int open0 = -1, open1 = -1;  // segments of the items that other CTAs share: from before, into the next
  if (*abort_flag) {
    // The others still wait to be counted (or find their counter as it must be next
    // time): what this CTA shares is handed on as a part that is NaN.
    if (threadIdx.x < 2) {
      const int at = threadIdx.x ? cta_end - 1 : cta_begin;
      const Walk w = walk_to<kRows>(p, pre, at);
      const int begin = at - (w.step - w.s.step0), end = begin + w.s.steps;
      const bool shared = threadIdx.x ? begin >= cta_begin && end > cta_end : begin < cta_begin;
      segments[threadIdx.x] = {shared ? begin : -1, end, w.b, w.head, w.chunk};
      float* to = p.partials + (2ll * blockIdx.x + threadIdx.x) * kPart + kRows * D;
      for (int r = 0; r < kRows; ++r) to[r] = 0.f, to[kRows + r] = CUDART_NAN_F;
    }
    __syncthreads();
    if (segments[0].begin >= 0) open0 = 0;
    if (segments[1].begin >= 0) open1 = 1;
  } else {
    const int mine = lane < 2 * kWarps ? segments[lane].begin : -1;
    uint32_t left = __ballot_sync(0xffffffffu, mine >= 0);
    int unit = 0;
    while (left) {
      const int s0 = __ffs(left) - 1;
      const Segment seg = segments[s0];
      const uint32_t group = __ballot_sync(0xffffffffu, mine == seg.begin);
      left &= ~group;
      const bool all = seg.begin >= cta_begin && seg.end <= cta_end;
      const int side = seg.begin < cta_begin ? 0 : 1;
      if (!all) (side ? open1 : open0) = s0;
      const Span sp = span_of<kRows>(p, seg.b);
      const int rows = min(kRows, sp.n * p.group - seg.chunk * kRows);
#pragma unroll 1
      for (int r = 0; r < rows; ++r, ++unit) {
        if (unit % kWarps != warp) continue;
        const bool in = group >> lane & 1;
        const float m = in ? part_of(lane)[kRows * D + r] : kLowest;
        const float top_all = warp_max(m);
        float w = in ? part_of(lane)[kRows * D + kRows + r] * exp2_approx(m - top_all) : 0.f;
        const float sum = warp_sum(w);
        w *= sum == 0.f ? 0.f : 1.f / sum;
        Row x = {};
#pragma unroll 1
        for (uint32_t rest = group; rest; rest &= rest - 1) {
          const int s = __ffs(rest) - 1;
          x.add_shared(__shfl_sync(0xffffffffu, w, s), part_of(s) + r * D, lane);
        }
        if (all) {
          store(seg, sp, r, x);
        } else {
          float* to = p.partials + (2ll * blockIdx.x + side) * kPart;
          x.put(to + r * D, lane);
          if (lane == 0) to[kRows * D + r] = top_all, to[kRows * D + kRows + r] = sum;
        }
      }
    }
  }
  if (open0 < 0 && open1 < 0) return;

  // --- items of several CTAs: the last to bring its part joins them ----------
  __threadfence();
  __syncthreads();
  if (threadIdx.x < 2) {
    const int s = threadIdx.x ? open1 : open0;
    int last = 0;
    if (s >= 0) {
      const int c0 = first_cta(segments[s].begin), c1 = last_cta(segments[s].begin, segments[s].end);
      last = atomicAdd(p.counters + c0, 1) == c1 - c0;
      if (last) p.counters[c0] = 0;
    }
    last_flag[threadIdx.x] = last;
  }
  __syncthreads();
  if (!last_flag[0] && !last_flag[1]) return;
  __threadfence();
  // A warp a row, or several, each over some of the CTAs.  How many is the item's
  // alone: the order of the sums must not depend on which CTA is last for what.
  int rows_of[2], split_of[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    rows_of[side] = 0;
    split_of[side] = 1;
    if (last_flag[side]) {
      const Segment& seg = segments[side ? open1 : open0];
      rows_of[side] = min(kRows, span_of<kRows>(p, seg.b).n * p.group - seg.chunk * kRows);
      split_of[side] = max(kWarps / rows_of[side], 1);
    }
  }
  const int units0 = rows_of[0] * split_of[0], units = units0 + rows_of[1] * split_of[1];
  float* sheets = reinterpret_cast<float*>(smem);  // [units][D + 4]: the rings are done with
#pragma unroll 1
  for (int unit = warp; unit < units; unit += kWarps) {
    const int side = unit >= units0, split = split_of[side], at = side ? unit - units0 : unit;
    const int r = at / split, sub = at - r * split;
    const Segment seg = segments[side ? open1 : open0];
    const int c0 = first_cta(seg.begin), parts = last_cta(seg.begin, seg.end) - c0 + 1;
    auto from = [&](int c) -> const float* {
      return p.partials + (2ll * (c0 + c) + (c == 0 ? 1 : 0)) * kPart;
    };
    float top_all = kLowest, sum = 0.f;
    Row x = {};
#pragma unroll 1
    for (int base = sub; base < parts; base += 32 * split) {
      const int c = base + split * lane;
      const float m = c < parts ? __ldcg(from(c) + kRows * D + r) : kLowest;
      const float n = c < parts ? __ldcg(from(c) + kRows * D + kRows + r) : 0.f;
      const float top1 = fmaxf(top_all, warp_max(m)), f = exp2_approx(top_all - top1);
      const float w = n * exp2_approx(m - top1);
      top_all = top1;
      sum = fmaf(sum, f, warp_sum(w));
#pragma unroll
      for (int y = 0; y < D / 32; ++y) x.x[y] *= f;
      const int here = min(32, (parts - base + split - 1) / split);
#pragma unroll 1
      for (int y = 0; y < here; y += 8) {
#pragma unroll
        for (int z = 0; z < 8; ++z) {  // past the end: the last one again, times nothing
          const float wz = __shfl_sync(0xffffffffu, w, (y + z) & 31);
          x.add(y + z < here ? wz : 0.f, from(base + split * min(y + z, here - 1)) + r * D, lane);
        }
      }
    }
    const float over = split > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int y = 0; y < D / 32; ++y) x.x[y] *= over;
    if (split > 1) {
      x.put(sheets + unit * (D + 4), lane);
      if (lane == 0) sheets[unit * (D + 4) + D] = top_all, sheets[unit * (D + 4) + D + 1] = sum;
    } else {
      store(seg, span_of<kRows>(p, seg.b), r, x);
    }
  }
  if (split_of[0] == 1 && split_of[1] == 1) return;
  __syncthreads();
#pragma unroll 1
  for (int row = warp; row < rows_of[0] + rows_of[1]; row += kWarps) {
    const int side = row >= rows_of[0], split = split_of[side], r = side ? row - rows_of[0] : row;
    if (split == 1) continue;
    const float* sheet = sheets + ((side ? units0 : 0) + r * split) * (D + 4);
    float top_all = kLowest, sum = 0.f;
    Row x = {};
#pragma unroll 1
    for (int y = 0; y < split; ++y) top_all = fmaxf(top_all, sheet[y * (D + 4) + D]);
#pragma unroll 1
    for (int y = 0; y < split; ++y, sheet += D + 4) {
      const float f = exp2_approx(sheet[D] - top_all);
      sum = fmaf(sheet[D + 1], f, sum);
      x.add_shared(f, sheet, lane);
    }
    const float over = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int y = 0; y < D / 32; ++y) x.x[y] *= over;
    const Segment seg = segments[side ? open1 : open0];
    store(seg, span_of<kRows>(p, seg.b), r, x);
  }
}

}  // namespace kv4
}  // namespace sm100
