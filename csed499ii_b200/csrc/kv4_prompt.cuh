// Attention over the 4-bit cache for requests with many query rows (prompts,
// pieces of prompts), on tcgen05.
//
// 4 * D operations per visible (query, key) pair and head bound it.  A CTA
// takes 256 query rows of one key/value head (rows are (token, head of the
// group) pairs, so all heads of a group share what is read) as two tiles of
// 128, and walks over the keys in steps of 128:
//
//   S = Q (C_k - 8)^T     tcgen05.mma, Q and the codes in shared memory
//   P                     in the softmax warps' registers, back to tensor
//                         memory in the place of S
//   O += P (C_v - 8)      tcgen05.mma, P from tensor memory
//
// As in the decode kernel the operands are codes, exact in 16 bits, and the
// rows' scales and offsets stay in 32 bits: a score is s_k S + z_k sum(q) with
// z = offset + 8 scale, the exponential gives the weight w = p s_v that goes
// back, and sum(p) = sum(w / s_v) and sum(p z_v) = sum(w z_v / s_v), one number
// a row, join the result at the end.  That costs the softmax warps three more
// multiply-adds a pair than plain attention, in two-wide f32x2 instructions,
// and saves every rounding but the weights'.
//
// Four warps each turn key and value codes into operand tiles (two stages of
// each), a thread per query tile issues its products (one thread issues a
// product of 128 x 128 x 16 every ~90 cycles, the tensor core could take one
// every 64), and four warps per query tile do the softmax, one row a thread.
// While one query tile is in its softmax the other one's products run.  The running maximum is only moved when an argument passes it by more than
// 8 (a factor of 256): then the step's weights are made again, more slowly, and
// the accumulator in tensor memory is scaled, which is rare after the first
// steps.  Steps that some row does not see whole go the slow way too.
#pragma once

#include <math_constants.h>

#include "kv4_decode.cuh"
#include "marlin24_prefill.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kPromptBatch = 8192;  // requests of a launch
constexpr int kPromptThreads = 20 * 32;
// Registers a thread: 96 at launch, then as below (256 * 168 + 256 * 56 + 128 * 32 = 640 * 96).
constexpr int kSoftmaxRegs = 168, kOperandRegs = 56, kIssueRegs = 32;
constexpr int kStep = 128;          // keys of a step

struct PromptParams {
  Cache cache;
  const uint8_t* q;      // element (row, head, c) at q_row * row + q_head * head + c
  int64_t q_row, q_head;
  int q_aligned;         // 1: every row of q starts on a 16-byte boundary
  uint8_t* out;          // [rows][q_heads][D]
  const int* tables;     // [batch][table_stride], `width` entries used
  int64_t table_stride;
  int width;
  const int* lens;       // tokens of each request in the cache, the step's own among them
  const int* starts;     // [batch + 1] first row of each request
  int batch;
  int rows;              // of q
  int q_heads;
  int group;             // query heads per key/value head
  int window;            // 0: none
  int most;              // requests with at most this many query rows a group are left alone
  float scale;
  int* status;
};

template <int D>
struct PromptCfg {
  static constexpr int kQ = 128 * D * 2;       // a query tile
  static constexpr int kK = kStep * D * 2;     // a key or value tile
  static constexpr int kOffK = 2 * kQ;         // two stages
  static constexpr int kOffV = kOffK + 2 * kK; // two stages
  static constexpr int kOffPairs = kOffV + 2 * kK;     // [4] Constants
  static constexpr int kOffMisc = kOffPairs + 4 * 64 * 40;
  static constexpr int kSmem = kOffMisc + 1024 + 1024;  // and room to align
  static constexpr uint32_t kColS = 0, kColO = 256, kCols = 512;
};

__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_store_32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void tmem_store_16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_store_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

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
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Eight codes (nibbles 0..7 of `w`) less 8 as 16-bit numbers, in the order
// 0, 4, 1, 5, 2, 6, 3, 7.
template <bool BF16>
__device__ __forceinline__ uint4 centred(uint32_t w) {
  uint4 r;
  if constexpr (BF16) {
    const uint32_t k136 = 0x43084308u;  // 128 + 8 twice
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t y = lop3<kLutAndOr>(w >> (4 * i), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 z = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y),
                                       *reinterpret_cast<const __nv_bfloat162*>(&k136));
      x[i] = *reinterpret_cast<const uint32_t*>(&z);
    }
    r = make_uint4(x[0], x[1], x[2], x[3]);
  } else {
    half2 a, b, c, d;
    dequant_pair(w, a, b);
    dequant_pair(w >> 8, c, d);
    r = make_uint4(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b),
                   *reinterpret_cast<uint32_t*>(&c), *reinterpret_cast<uint32_t*>(&d));
  }
  return r;
}

template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

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

// The rows of a request that this kernel serves, as 256-row items.
__device__ __forceinline__ int prompt_items(const PromptParams& p, int b) {
  const int first = min(max(p.starts[b], 0), p.rows);
  const int64_t rows = static_cast<int64_t>(min(p.starts[b + 1], p.rows) - first) * p.group;
  return rows > p.most ? static_cast<int>((rows + 255) / 256) : 0;
}

// What the softmax needs to know of a step's keys, two by two.
struct Constants {
  float4 key[kStep / 2];   // scales, values at code 8, both times scale * log2 e
  float4 value[kStep / 2]; // ValueRow: log_s, inv_s
  float2 at_8[kStep / 2];
};

// Arguments of the weights of keys 2i and 2i + 1 of a step, from their products.
__device__ __forceinline__ F2 arguments(const Constants& k, int i, uint32_t s0, uint32_t s1, F2 sumq) {
  const float4 ks = k.key[i], vs = k.value[i];
  return fma2(pack2(ks.x, ks.y), pack2(__uint_as_float(s0), __uint_as_float(s1)),
              fma2(pack2(ks.z, ks.w), sumq, pack2(vs.x, vs.y)));
}

template <class T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    kv4_prompt_kernel(const __grid_constant__ PromptParams p) {
  using Cfg = PromptCfg<D>;
  constexpr int kBytes = tile_bytes(D);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Constants* constants = reinterpret_cast<Constants*>(smem + Cfg::kOffPairs);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffMisc);
  const uint32_t bar = smem_addr(bars);
  // barriers
  const uint32_t q_ready = bar, k_full = bar + 16, k_empty = bar + 32, v_full = bar + 48,
                 v_empty = bar + 64, s_full = bar + 80, p_ready = bar + 96, o_done = bar + 112,
                 c_full = bar + 128 /* four */, finished = bar + 160;
  uint64_t* tile_at = bars + 24;                                        // keys' and values' [4][8]
  uint32_t* valid = reinterpret_cast<uint32_t*>(bars + 88);             // [4][4]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 96);
  volatile int* drain_flag = abort_flag + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 97);
  int* sums = reinterpret_cast<int*>(bars + 98);                        // [20]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y;

  // --- which rows -------------------------------------------------------------
  int* pre = reinterpret_cast<int*>(smem);  // where the tiles will be
  int total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPromptThreads) {
    const int b = b0 + threadIdx.x;
    int x = b < p.batch ? prompt_items(p, b) : 0;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, i);
      if (lane >= i) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < kPromptThreads / 32; ++i) {
      if (i == warp) x += all;
      all += sums[i];
    }
    if (b < p.batch) pre[b] = total + x;
    total += all;
    __syncthreads();
  }
  // the last items first: within a request they have the most keys
  const int item = total - 1 - static_cast<int>(blockIdx.x);
  if (item < 0) return;
  const int b = first_above(pre, p.batch, item);
  const int tile = item - (b ? pre[b - 1] : 0);
  const int first = min(max(p.starts[b], 0), p.rows), n = min(p.starts[b + 1], p.rows) - first;
  const int64_t room = static_cast<int64_t>(p.width) * p.cache.page_size;
  const int len = static_cast<int>(min(static_cast<int64_t>(p.lens[b]), room));
  const int rows = min(256, n * p.group - tile * 256);
  const int tiles_q = rows > 128 ? 2 : 1;
  const int before = len - n;  // position of the request's row 0
  const int lo_pos = before + tile * 256 / p.group, hi_pos = before + (tile * 256 + rows - 1) / p.group;
  const int from = p.window && lo_pos >= p.window ? lo_pos - p.window + 1 : 0;
  const int to = min(len, hi_pos + 1);
  const int step0 = from / kStep;
  const int steps = to > from ? (to + kStep - 1) / kStep - step0 : 0;
  __syncthreads();  // `pre` is read

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_ready + 8 * i, 4);
      mbar_init(k_full + 8 * i, 4);
      mbar_init(k_empty + 8 * i, tiles_q);
      mbar_init(v_full + 8 * i, 4);
      mbar_init(v_empty + 8 * i, tiles_q);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 4);
      mbar_init(o_done + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(c_full + 8 * i, 4);
    mbar_init(finished, tiles_q);
    *abort_flag = *drain_flag = 0;
    fence_mbar_init();
  }
  if (warp == 16) tmem_alloc(smem_addr(tmem_slot), Cfg::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  auto wait = [&](uint32_t at, int phase) {  // one thread
    ok = ok && mbar_wait_spin_sleep_bounded(at, phase & 1, abort_flag);
    return ok;
  };
  auto wait_warp = [&](uint32_t at, int phase) {
    ok = __all_sync(0xffffffffu, ok && mbar_wait_spin_sleep_bounded(at, phase & 1, abort_flag));
    return ok;
  };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    take_registers<kSoftmaxRegs>();
    const int qi = warp >> 2, row = (warp & 3) * 32 + lane;
    if (qi < tiles_q) {
      const int r = tile * 256 + qi * 128 + row;
      const int token = r / p.group, h = head * p.group + r % p.group;
      const bool live = qi * 128 + row < rows;
      // this row of Q, its channels in the order that `centred` gives the codes
      float sumq = 0.f;
      {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) +
                              p.q_row * (first + token) + p.q_head * h;
        const uint32_t dst = smem_addr(smem) + qi * Cfg::kQ + row * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live) {
            if (p.q_aligned) {
              x = *reinterpret_cast<const uint4*>(src + 8 * c);
            } else {
              uint32_t y[4];
#pragma unroll
              for (int z = 0; z < 4; ++z)
                y[z] = src[8 * c + 2 * z] | static_cast<uint32_t>(src[8 * c + 2 * z + 1]) << 16;
              x = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
          const float2 f0 = T::up(x.x), f1 = T::up(x.y), f2 = T::up(x.z), f3 = T::up(x.w);
          sumq += ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
          sts128(dst + (c >> 3) * (128 * 128) + (((c & 7) ^ (row & 7)) << 4),
                 make_uint4(prmt(x.x, x.z, 0x5410), prmt(x.x, x.z, 0x7632), prmt(x.y, x.w, 0x5410),
                            prmt(x.y, x.w, 0x7632)));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready + 8 * qi);

      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + lanes + Cfg::kColS + 128 * qi;
      const uint32_t o_at = tmem + lanes + Cfg::kColO + D * qi;
      const int pos = before + token;
      const int tile_lo = before + (tile * 256 + qi * 128) / p.group;
      const int tile_hi = before + (tile * 256 + min(rows, qi * 128 + 128) - 1) / p.group;
      float top = kLowest, l = 0.f, off = 0.f;
      for (int it = 0; it < steps; ++it) {
        const int buf = it & 3;
        if (!wait_warp(c_full + 8 * buf, it >> 2) || !wait_warp(s_full + 8 * qi, it)) break;
        tc_fence_after();
        const Constants& k = constants[buf];
        const int j0 = (step0 + it) * kStep;
        const bool whole = j0 + kStep <= tile_lo + 1 && (p.window == 0 || tile_hi - j0 < p.window) &&
                           (valid[4 * buf] & valid[4 * buf + 1] & valid[4 * buf + 2] & valid[4 * buf + 3]) ==
                               0xffffffffu;
        const F2 q2 = pack2(sumq, sumq);
        bool done = false;
        if (whole && it > 0) {
          // the step with the maximum as it is
          uint32_t weights[64];
          float mx[2] = {kLowest, kLowest};
          F2 l2[2] = {0, 0}, off2[2] = {0, 0};
          const F2 top2 = pack2(-top, -top);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32(s_at + 32 * c, s);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 y = unpack2(add2(arguments(k, 16 * c + i, s[2 * i], s[2 * i + 1], q2), top2));
              mx[i & 1] = max3(mx[i & 1], y.x, y.y);
              const float2 w = make_float2(exp2_approx(y.x), exp2_approx(y.y));
              const F2 w2 = pack2(w.x, w.y);
              const float4 vs = k.value[16 * c + i];
              const float2 z = k.at_8[16 * c + i];
              l2[i & 1] = fma2(w2, pack2(vs.z, vs.w), l2[i & 1]);
              off2[i & 1] = fma2(w2, pack2(z.x, z.y), off2[i & 1]);
              weights[16 * c + i] = Half::down(w.x, w.y);
            }
          }
          done = !__any_sync(0xffffffffu, fmaxf(mx[0], mx[1]) > 8.f);
          if (done) {
            const float2 la = unpack2(add2(l2[0], l2[1])), oa = unpack2(add2(off2[0], off2[1]));
            l += la.x + la.y;
            off += oa.x + oa.y;
            tmem_store_32(s_at, weights);
            tmem_store_32(s_at + 32, weights + 32);
          }
        }
        if (!done) {
          // With the maximum of the step first.  What a row does not see has no
          // weight, whatever lies in its place.
          const int back = p.window ? p.window : 0x7fffffff;  // a query sees less far than this
          auto unseen = [&](int j, uint32_t there) {
            return j > pos || pos - j >= back || !(there >> (j & 31) & 1);
          };
          float mx = kLowest;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32(s_at + 32 * c, s);
            const uint32_t there = valid[4 * buf + c];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 x = unpack2(arguments(k, 16 * c + i, s[2 * i], s[2 * i + 1], q2));
              const int j = j0 + 32 * c + 2 * i;
              if (!unseen(j, there)) mx = fmaxf(mx, x.x);
              if (!unseen(j + 1, there)) mx = fmaxf(mx, x.y);
            }
          }
          if (__any_sync(0xffffffffu, mx > top + 8.f)) {
            const float f = exp2_approx(top - fmaxf(top, mx));
            top = fmaxf(top, mx);
            l *= f;
            off *= f;
            if (it > 0) {
              if (!wait_warp(o_done + 8 * qi, it - 1)) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o_at + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_store_32(o_at + 32 * c, o);
              }
            }
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32(s_at + 32 * c, s);
            const uint32_t there = valid[4 * buf + c];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 x = unpack2(arguments(k, 16 * c + i, s[2 * i], s[2 * i + 1], q2));
              const float4 vs = k.value[16 * c + i];
              const float2 z = k.at_8[16 * c + i];
              const int j = j0 + 32 * c + 2 * i;
              float2 w = make_float2(exp2_approx(x.x - top), exp2_approx(x.y - top));
              float2 lw = make_float2(w.x * vs.z, w.y * vs.w), zw = make_float2(w.x * z.x, w.y * z.y);
              if (unseen(j, there)) w.x = lw.x = zw.x = 0.f;
              if (unseen(j + 1, there)) w.y = lw.y = zw.y = 0.f;
              l += lw.x + lw.y;
              off += zw.x + zw.y;
              s[i] = Half::down(w.x, w.y);
            }
            // its place is that of products already read
            tmem_store_16(s_at + 16 * c, s);
          }
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 8 * qi);
      }
      if (steps > 0 && wait_warp(o_done + 8 * qi, steps - 1)) tc_fence_after();
      const float over = l == 0.f ? 0.f : 1.f / l;
      uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(first + token) * p.q_heads + h) * D);
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (steps > 0) tmem_ld32(o_at + 32 * c, o);
          if (!live) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float a = __uint_as_float(o[8 * i + 2 * x]), d = __uint_as_float(o[8 * i + 2 * x + 1]);
              w[x] = l == 0.f || steps == 0 ? 0u : T::down((a + off) * over, (d + off) * over);
            }
            *reinterpret_cast<uint4*>(dst + 64 * c + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  } else if (warp < 16) {
    // ------------------------------------------- codes to operand tiles
    // Warps 8-11 the keys' (and what the softmax needs to know), 12-15 the
    // values'.  Codes are in registers a step ahead; where a step's tiles lie is
    // looked up two steps ahead.  Once a wait has given up these warps run on
    // without waiting: they meet at a barrier every step, which none of them
    // may leave alone.
    give_registers<kOperandRegs>();
    const bool keys = warp < 12;
    const int dw = warp & 3, id = dw * 32 + lane, meet = keys ? 1 : 2;
    const int per_page = p.cache.page_size / kTile;
    uint64_t* tiles = tile_at + (keys ? 0 : 32);
    auto look_up = [&](int it) {  // where the step's eight cache tiles are
      if (dw == 0 && lane < 8 && it < steps) {
        const int t = (step0 + it) * 8 + lane;
        uint64_t at = 0;
        if (static_cast<int64_t>(t) * kTile < len) {
          const int page = p.tables[p.table_stride * b + t / per_page];
          if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.pages))
            at = reinterpret_cast<uint64_t>(p.cache.page_tiles<D>(page, head) + t % per_page * kBytes);
        }
        tiles[8 * (it & 3) + lane] = at;
      }
    };
    auto tile_of = [&](int it, int i) { return reinterpret_cast<const uint8_t*>(tiles[8 * (it & 3) + i]); };
    look_up(0);
    look_up(1);
    named_bar_sync(meet, 128);
    if (keys) {
      constexpr int kUnits = D / 32;  // 16-byte loads of a thread
      const float c2 = p.scale * kLog2e;
      uint4 codes[kUnits];
      uint32_t kp = 0, vp = 0;
      bool here = false;
      auto load = [&](int it) {
        if (it >= steps) return;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int rest = (u * 128 + id) >> 3, chunk = rest % kUnits, half = rest / kUnits;
          const uint8_t* src = tile_of(it, half >> 1);
          codes[u] = src ? *reinterpret_cast<const uint4*>(src + off_k(D, (half & 1) * 8 + (lane & 7)) + 16 * chunk)
                         : make_uint4(0, 0, 0, 0);
        }
        const uint8_t* src = tile_of(it, id >> 4);
        here = src != nullptr && (step0 + it) * kStep + id < len;
        kp = here ? *reinterpret_cast<const uint32_t*>(src + off_k_pair(D, id & 15)) : 0u;
        vp = here ? *reinterpret_cast<const uint32_t*>(src + off_v_pair(D, id & 15)) : 0u;
      };
      load(0);
      for (int it = 0; it < steps; ++it) {
        const int stage = it & 1, buf = it & 3;
        look_up(it + 2);
        if (it >= 2) wait_warp(k_empty + 8 * stage, (it >> 1) - 1);
        {
          const float2 ks = T::up(kp);
          const ValueRow v = value_row(T::up(vp));
          Constants& c = constants[buf];
          float* kf = reinterpret_cast<float*>(&c.key[id >> 1]) + (id & 1);
          kf[0] = ks.x * c2;
          kf[2] = fmaf(ks.x, 8.f, ks.y) * c2;
          float* vf = reinterpret_cast<float*>(&c.value[id >> 1]) + (id & 1);
          vf[0] = v.log_s;
          vf[2] = v.inv_s;
          reinterpret_cast<float*>(&c.at_8[id >> 1])[id & 1] = v.at_8;
          const uint32_t mask = __ballot_sync(0xffffffffu, here);
          if (lane == 0) valid[4 * buf + dw] = mask;
          __syncwarp();
          if (lane == 0) mbar_arrive(c_full + 8 * buf);
        }
        const uint32_t dst = smem_addr(smem) + Cfg::kOffK + stage * Cfg::kK;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int rest = (u * 128 + id) >> 3, chunk = rest % kUnits, half = rest / kUnits;
          const int key = half * 8 + (lane & 7);
          const uint32_t w[4] = {codes[u].x, codes[u].y, codes[u].z, codes[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c8 = chunk * 4 + i;  // eighth channel group of the row
            sts128(dst + (c8 >> 3) * (kStep * 128) + key * 128 + (((c8 & 7) ^ (key & 7)) << 4),
                   centred<T::kBf16>(w[i]));
          }
        }
        load(it + 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full + 8 * stage);
        named_bar_sync(meet, 128);
      }
    } else {
      constexpr int kWordsV = D / 64;  // words of codes per token a thread
      const int half = (lane & 7) + 8 * (dw & 1), piece = (lane >> 3) + 4 * (dw >> 1);
      uint32_t w[8 * kWordsV];         // of the eight tokens of a half tile: [token][kWordsV]
      auto load = [&](int it) {
        if (it >= steps) return;
        const uint8_t* src = tile_of(it, half >> 1);
#pragma unroll
        for (int u = 0; u < 2 * kWordsV; ++u) {
          const uint4 x = src ? *reinterpret_cast<const uint4*>(src + off_v(D, (half & 1) * 8, piece) + 16 * u)
                              : make_uint4(0, 0, 0, 0);
          w[4 * u] = x.x, w[4 * u + 1] = x.y, w[4 * u + 2] = x.z, w[4 * u + 3] = x.w;
        }
      };
      load(0);
      for (int it = 0; it < steps; ++it) {
        const int stage = it & 1;
        look_up(it + 2);
        if (it >= 2) wait_warp(v_empty + 8 * stage, (it >> 1) - 1);
        const uint32_t dst = smem_addr(smem) + Cfg::kOffV + stage * Cfg::kK;
#pragma unroll
        for (int o = 0; o < kWordsV; ++o) {
#pragma unroll
          for (int part = 0; part < 4; ++part) {  // channels 2 part and 2 part + 1 of the octet
            half2 even[4], odd[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {  // tokens 2t and 2t + 1
              const uint32_t y = prmt(w[2 * t * kWordsV + o], w[(2 * t + 1) * kWordsV + o], part < 2 ? 0x5410 : 0x7632);
              dequant_pair(y >> (8 * (part & 1)), even[t], odd[t]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int d = piece * (D / 8) + 8 * o + 2 * part + x;
              const half2* z = x ? odd : even;
              sts128(dst + (half >> 3) * (D * 128) + d * 128 + (((half & 7) ^ (d & 7)) << 4),
                     make_uint4(*reinterpret_cast<const uint32_t*>(&z[0]), *reinterpret_cast<const uint32_t*>(&z[1]),
                                *reinterpret_cast<const uint32_t*>(&z[2]), *reinterpret_cast<const uint32_t*>(&z[3])));
            }
          }
        }
        load(it + 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + 8 * stage);
        named_bar_sync(meet, 128);
      }
    }
  } else {
    give_registers<kIssueRegs>();
    const int qi = warp - 16;
    if (lane == 0 && qi < tiles_q && steps > 0) {
      // ---------------------------------------------------------- products
      constexpr uint32_t types = T::kBf16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t id_s = umma_idesc_f16_f32(kStep) | types, id_o = umma_idesc_f16_f32(D);
      const uint32_t base = smem_addr(smem);
      const uint32_t s_at = tmem + Cfg::kColS + 128 * qi, o_at = tmem + Cfg::kColO + D * qi;
      auto scores = [&](int stage) {
        const uint64_t a = umma_desc_sw128_k(base + qi * Cfg::kQ);
        const uint64_t bd = umma_desc_sw128_k(base + Cfg::kOffK + stage * Cfg::kK);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t at = (k >> 2) * (128 * 128) + (k & 3) * 32;
          umma_f16(s_at, a + (at >> 4), bd + (at >> 4), id_s, k > 0);
        }
        umma_commit(s_full + 8 * qi);
        umma_commit(k_empty + 8 * stage);
      };
      if (wait(q_ready + 8 * qi, 0) && wait(k_full, 0)) {
        tc_fence_after();
        scores(0);
        for (int it = 0; it < steps; ++it) {
          const int stage = it & 1, next = (it + 1) & 1;
          if (!wait(v_full + 8 * stage, it >> 1) || !wait(p_ready + 8 * qi, it)) break;
          tc_fence_after();
          const uint64_t bd = umma_desc_sw128_k(base + Cfg::kOffV + stage * Cfg::kK);
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k) {
            const uint32_t at = (k >> 2) * (D * 128) + (k & 3) * 32;
            umma_f16_ts(o_at, s_at + 8 * k, bd + (at >> 4), id_o, it > 0 || k > 0);
          }
          umma_commit(o_done + 8 * qi);
          umma_commit(v_empty + 8 * stage);
          if (it + 1 < steps) {
            if (!wait(k_full + 8 * next, (it + 1) >> 1)) break;
            tc_fence_after();
            scores(next);
          }
        }
      }
      umma_commit(finished);
      mbar_wait_bounded(finished, 0, drain_flag);
    }
  }
  if (!ok && lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kCols);
  }
}

}  // namespace kv4
}  // namespace sm100
