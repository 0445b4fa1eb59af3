// Attention over the 4-bit cache for requests with many query rows (prompts,
// pieces of prompts), on tcgen05.
//
// 4 * D operations per visible (query, key) pair and head bound it, and next to
// them one exponential a pair (16 an SM and cycle, as long as its two products
// of 128 channels take).  A CTA takes 256 query rows of one key/value head
// (rows are (token, head of the group) pairs, so all heads of a group share what
// is read) as two tiles of 128, and walks over the keys in steps of 112 (128
// where D is 64):
//
//   S = Q (C_k - 8)^T     tcgen05.mma, Q and the codes in shared memory
//   P                     in the softmax warps' registers, back to tensor
//                         memory in the place of S
//   O += P 2 (C_v - m)    tcgen05.mma, P from tensor memory; m is a row's middle code
//
// As in the decode kernel the operands are codes, exact in 16 bits, so that
// nothing is rounded but the weights.  Here they are one half for either type: an
// fp16 result has 1.2 to 1.45 times the error of a result rounded once (the weights'
// roundings are as large as its own), and a second product for what the rounding
// leaves, as the decode kernel has, would add half of the step's tensor work and as
// many stores to tensor memory again.  What scales and offsets add is put into
// the same products as 16 more channels, in two or three 16-bit terms each
// (2^-22 of a value): with z = offset / s_k + 8 a key's argument of the
// exponential is s_k (S + z sum(q) + log2 s_v / s_k), so its column of S needs
// one multiply-add; and the columns 1 / s_v and offset / s_v + m next to the
// values' codes give sum(p) and the values' offsets with the result (the weights
// are w = p s_v).  Without them every pair of keys costs the softmax ten
// broadcast reads of shared memory, and those bound it (a prompt of 8192 tokens,
// 32 heads on 8 of 128 channels: 1452 us instead of 1108, before the steps below
// brought it to 808).  They are why a step is 112 keys: two tiles of scores and two
// of 144 channels are all of tensor memory.
//
// What is left to bound it is shared memory: a product of 128 x 112 x 16 reads
// 120 bytes a cycle.  So the scores are read in the fragment form of 16 lanes x
// 8 columns, in which a thread has two neighbouring keys of four rows: one
// 8-byte read of the keys' scales serves 8 products, where one row a thread
// would take a broadcast for every key.
//
// Numbers that the terms cannot hold (a key's or value's scale out of the usual
// range, a row of NaN) are added in 32 bits by a careful form of the step.  So
// is what the weights lose in rounding to half where the values' scales differ
// by more than a factor of 64: a weight p s_v below 2^-21 of the largest is rounded
// more coarsely, which is nothing to the result but could be to sum(p).  A third form
// serves steps that some row does not see whole and steps that move the running
// maximum: the maximum is only moved when an argument passes it by more than kLag,
// which is rare after the first steps.
//
// Four warps each turn key and value codes into operand tiles (two stages of
// each), eight warps per query tile do the softmax (two for 32 rows: one has
// the first 64 keys of a step, one the others, and they agree on whether the
// maximum moves), and one warp issues the products, the first query tile's result and next scores before the second
// one's: so each runs while the other is in its softmax.
//
// Where requests are too few to fill the GPU, an item's keys are shared out over
// several CTAs in runs of steps; each leaves its rows' results with their maxima
// and sums in the workspace, and a second kernel joins them in order.
//
// The prompt above takes 808 us, 680 TFLOP/s of 1661 measured for a large matrix
// product.  Of a step's 4900 cycles (256 rows, 112 keys) the products take 2200 and
// a tile's softmax 2800, of which eight warps with 88 registers hide too little
// latency: each 16 keys are a load from tensor memory and then 16 exponentials a
// thread.  Loading the next 16 keys ahead needs 16 registers more than there are
// (spilled: 1020 us; as it is, 24 bytes are spilled at D = 128 and 50 at D = 64).  An item's beginning and end take 35000 cycles, 15% of it.
#pragma once

#include <math_constants.h>

#include "kv4_decode.cuh"
#include "marlin24_prefill.cuh"

namespace sm100 {
namespace kv4 {

constexpr int kPromptBatch = 8192;  // requests of a launch
constexpr int kPromptThreads = 28 * 32;
// Registers a thread: 72 at launch, then as below (512 * 88 + 256 * 56 + 128 * 40 = 896 * 72).
constexpr int kSoftmaxRegs = 88, kOperandRegs = 56, kIssueRegs = 40;

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
  int split;             // CTAs of a head that the keys of its items may be shared out over; 0: they are not
  float* partials;       // [CTAs] parts of items that are
  int* status;
};

constexpr int kSplitBatch = 1024;  // requests of a launch that shares out keys
// Steps of a CTA where keys are shared out: an item costs a CTA about as much as
// four steps before and after its own.
constexpr int kLeastPromptSteps = 4;

// The tensor cores cut a sum off at 2^-23 of it with every product added, which is
// a bias over many keys (131071 that weigh 2^-26 of a first one had 3.7 times the
// error that the rounding of weights allows).  After so many steps (about 900
// products of a channel) the results so far go to the softmax warps' local memory,
// are added to in binary32 there, and the products begin anew.
constexpr int kFreshSteps = 128;

// What the careful form of a step needs to know of its keys (the usual one
// reads the scales alone).
struct Numbers {
  float scale[128];  // of the key, times scale * log2 e
  float z[128];      // the key's value at code 8 over its scale
  float log_s[128], inv_s[128], at_mid[128];  // of the value
};

template <int D>
struct PromptCfg {
  static constexpr int kStep = D == 128 ? 112 : 128;  // keys of a step
  static constexpr int kTiles = kStep / kTile;
  static constexpr int kN = D + 16;                   // columns of the result: channels and sums
  // operand tiles of 128-byte rows (64 numbers), and of 32-byte rows (the 16 more)
  static constexpr int kQ = 128 * D * 2, kQx = 128 * 32;
  static constexpr int kK = kStep * D * 2, kKx = kStep * 32;
  static constexpr int kV = 2 * kN * 128;
  static constexpr int kOffK = 2 * kQ;                // two stages of each
  static constexpr int kOffV = kOffK + 2 * kK;
  static constexpr int kOffQx = kOffV + 2 * kV;
  static constexpr int kOffKx = kOffQx + 2 * kQx;
  static constexpr int kOffNumbers = kOffKx + 2 * kKx;  // four stages
  static constexpr int kOffRows = kOffNumbers + 4 * sizeof(Numbers);  // [tile][half][row] of two numbers
  static constexpr int kOffMiddles = kOffRows + 2 * 2 * 128 * 8;  // [stage][key]: 1024 + twice a value's middle, a half
  static constexpr int kOffMisc = kOffMiddles + 4 * 256;
  static constexpr int kSmem = kOffMisc + 1280 + 1024;  // and room to align
  static_assert(kSmem <= kPrefillSmemBudget && kK % 1024 == 0 && kV % 1024 == 0 && kKx % 256 == 0, "tiles");
  static constexpr uint32_t kColS = 0, kColO = 2 * kStep, kCols = 512;
  static_assert(kColO + 2 * kN <= kCols, "tensor memory");
};

// Shared-memory matrix descriptor, K-major operand of 32-byte rows, swizzled:
// groups of 8 rows 256 bytes apart, swizzle mode 6.
__device__ __forceinline__ uint64_t umma_desc_sw32_k(uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(1u) << 16;
  d |= static_cast<uint64_t>(256u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(6u) << 61;
  return d;
}

// Products issued by a whole warp, of which one thread does it: where the code
// around them does not diverge their operands stay in uniform registers (a
// product of 128 x 144 x 16 every 74 cycles; issued from a branch of one lane,
// every 160).  N products along 64 channels or keys, 32 bytes apart in both
// operands (8 columns in tensor memory).
template <int N>
__device__ __forceinline__ void warp_umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  static_assert(N == 1 || N == 4, "products");
  if constexpr (N == 1) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
        "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
template <int N>
__device__ __forceinline__ void warp_umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  static_assert(N == 3 || N == 4, "products");
  if constexpr (N == 3) {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b64 b1, b2;\n\t.reg .b32 a1, a2;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "add.s32 a1, %1, 8;\n\tadd.s64 b1, %2, 2;\n\tadd.s32 a2, %1, 16;\n\tadd.s64 b2, %2, 4;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "add.s32 a1, %1, 8;\n\tadd.s64 b1, %2, 2;\n\tadd.s32 a2, %1, 16;\n\tadd.s64 b2, %2, 4;\n\t"
        "add.s32 a3, %1, 24;\n\tadd.s64 b3, %2, 6;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// The same thread's: arrives on `bar` once all its products so far are done.
__device__ __forceinline__ void warp_umma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}

__device__ __forceinline__ void tmem_load_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Waits for this thread's loads; `r` is what they brought (named here so that
// no use of it moves before the wait).
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
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

// Fragments of 16 lanes: N groups of 8 columns as 32-bit numbers (a thread has
// columns 2 (lane % 4) and the next of rows lane / 4 and lane / 4 + 8), and N
// groups of 4 columns (column lane % 4 of the same rows).
__device__ __forceinline__ void tmem_load_fragment(uint32_t taddr, uint32_t* r) {  // 16 columns
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_store_fragment(uint32_t taddr, const uint32_t* v) {
  if constexpr (N == 2) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3])
                 : "memory");
  } else if constexpr (N == 4) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    static_assert(N == 8, "groups");
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
  }
}

__device__ __forceinline__ void tmem_store_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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

// Twice what the codes in nibbles `at` of either half of `q` are off their rows'
// middles (`middle` is 1024 + twice those).
__device__ __forceinline__ half2 twice_off(uint32_t q, int at, half2 middle) {
  const uint32_t x = lop3<kLutAndOr>(at ? q >> (4 * at - 1) : q << 1, 0x001e001eu, 0x64006400u);  // 1024 + 2 c
  return __hsub2(*reinterpret_cast<const half2*>(&x), middle);
}

template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Whether any thread of the barrier's says so.
__device__ __forceinline__ bool named_bar_any(int id, int threads, bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<int>(x)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
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

// The first number of two in 16 bits, widened again.
template <class T>
__device__ __forceinline__ float rounded(float x) {
  return T::up(T::down(x, 0.f)).x;
}

// The 16 more channels, as 16-bit pairs: of a row of Q and of a key their
// product is z sum(q) + log.  Halves in two terms each, and `log` in either of
// two sizes; bf16 in three.
template <class T>
__device__ __forceinline__ void query_terms(float sum, uint4 (&x)[2]) {
  const float h = rounded<T>(sum), m = rounded<T>(sum - h);
  if constexpr (T::kBf16) {
    x[0] = make_uint4(T::down(h, h), T::down(m, m), T::down(h, sum - h - m), T::down(1.f, 1.f));
    x[1] = make_uint4(T::down(1.f, 0.f), 0u, 0u, 0u);
  } else {
    x[0] = make_uint4(T::down(h, m), T::down(h, 1.f), T::down(1.f, 16384.f), T::down(16384.f, 0.f));
    x[1] = make_uint4(0u, 0u, 0u, 0u);
  }
}
template <class T>
__device__ __forceinline__ void key_terms(float z, float log, uint4 (&x)[2]) {
  const float zh = rounded<T>(z), zm = rounded<T>(z - zh);
  if constexpr (T::kBf16) {
    const float a = rounded<T>(log), b = rounded<T>(log - a);
    x[0] = make_uint4(T::down(zh, zm), T::down(zh, zm), T::down(z - zh - zm, zh), T::down(a, b));
    x[1] = make_uint4(T::down(log - a - b, 0.f), 0u, 0u, 0u);
  } else {
    const bool large = fabsf(log) > 60000.f;
    const float y = large ? log * (1.f / 16384.f) : log;
    const float a = rounded<T>(y), b = y - a;
    x[0] = make_uint4(T::down(zh, zh), T::down(zm, large ? 0.f : a), T::down(large ? 0.f : b, large ? a : 0.f),
                      T::down(large ? b : 0.f, 0.f));
    x[1] = make_uint4(0u, 0u, 0u, 0u);
  }
}
// ... and what they hold: false for NaN too.
template <class T>
__device__ __forceinline__ bool terms_hold(float z, float log) {
  return T::kBf16 ? fabsf(z) < 1e30f && fabsf(log) < 1e30f : fabsf(z) < 60000.f && fabsf(log) < 1e9f;
}
// A value's row with the code nearest to its zero as the middle, in halves of a code:
// what codes are off it sums up to the result itself, and its own value is at most a
// quarter of the scale (more where a row does not reach zero).  With one middle for
// all rows, codes and middles of values that are not symmetric about zero have sums
// that cancel, and what the tensor cores cut off either stays: 30 times the error of
// a result rounded once for exponentially distributed values less their mean, 20000 keys
// of like weight.
struct MiddleRow : ValueRow {
  float twice;  // the middle, 0..30
};
__device__ __forceinline__ MiddleRow middle_row(float2 pair) {
  MiddleRow r;
  static_cast<ValueRow&>(r) = value_row(pair);
  r.twice = rintf(fminf(fmaxf(-2.f * pair.y * r.inv_s, 0.f), 30.f));
  r.at_mid = fmaf(pair.y, r.inv_s, 0.5f * r.twice);
  return r;
}
// The values' two numbers go into halves, a quarter of inv_s in 2^-9..2^15.
__device__ __forceinline__ bool sums_hold(const ValueRow& v) {
  return v.inv_s >= 0x1p-7f && v.inv_s <= 0x1p17f && fabsf(v.at_mid) < 60000.f;
}

// Inclusive prefix sums of the requests' items in `pre`, and their total.
template <int Threads>
__device__ __forceinline__ int prompt_prefix(const PromptParams& p, int* pre, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += Threads) {
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
    for (int i = 0; i < Threads / 32; ++i) {
      if (i == warp) x += all;
      all += sums[i];
    }
    if (b < p.batch) pre[b] = total + x;
    total += all;
    __syncthreads();
  }
  return total;
}

// 256 query rows of a request, and the keys that any of them sees.
struct PromptItem {
  int b, tile;
  int first, n, len;     // the request's rows and tokens
  int rows;              // of the item
  int before;            // position of the request's row 0
  int step0, steps;
};
template <int Step>
__device__ __forceinline__ PromptItem prompt_item(const PromptParams& p, const int* pre, int item) {
  PromptItem x;
  x.b = first_above(pre, p.batch, item);
  x.tile = item - (x.b ? pre[x.b - 1] : 0);
  x.first = min(max(p.starts[x.b], 0), p.rows);
  x.n = min(p.starts[x.b + 1], p.rows) - x.first;
  x.len = held_tokens(p.lens[x.b], p.width, p.cache.page_size);
  x.rows = min(256, x.n * p.group - x.tile * 256);
  x.before = x.len - x.n;
  const int lo = x.before + x.tile * 256 / p.group, hi = x.before + (x.tile * 256 + x.rows - 1) / p.group;
  const int from = p.window && lo >= p.window ? lo - p.window + 1 : 0;
  const int to = min(x.len, hi + 1);
  x.step0 = from / Step;
  x.steps = to > from ? (to + Step - 1) / Step - x.step0 : 0;
  return x;
}

// How an item's steps are shared out over at most `most` CTAs.
struct Shares {
  int parts, steps;  // of a part
  __device__ __forceinline__ Shares(int all, int most) {
    steps = max((all + most - 1) / most, min(all, kLeastPromptSteps));
    parts = steps ? (all + steps - 1) / steps : 1;
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    kv4_prompt_kernel(const __grid_constant__ PromptParams p) {
  using Cfg = PromptCfg<D>;
  constexpr int kStep = Cfg::kStep, kTiles = Cfg::kTiles, kN = Cfg::kN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Numbers* numbers = reinterpret_cast<Numbers*>(smem + Cfg::kOffNumbers);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffMisc);
  const uint32_t bar = smem_addr(bars);
  // barriers
  // `spent`, for step t in [0, steps]: result t - 1 and scores t are done with
  const uint32_t q_ready = bar, k_full = bar + 16, v_full = bar + 32, spent = bar + 48,
                 s_full = bar + 64, p_ready = bar + 80, c_full = bar + 96 /* four */,
                 finished = bar + 128;
  uint64_t* tile_at = bars + 24;                                        // keys' and values' [4][8]
  uint32_t* valid = reinterpret_cast<uint32_t*>(bars + 88);             // [4][4] keys that are there
  uint32_t* plain_k = valid + 16;                                       // ... whose numbers the terms hold
  uint32_t* plain_v = valid + 32;
  int* range = reinterpret_cast<int*>(valid + 48);                      // [4][2][4] exponents of value scales
  int* fine = range + 32;                                               // [4][4] all that are there are plain
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 140);
  volatile int* drain_flag = abort_flag + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 141);
  volatile int* after = reinterpret_cast<volatile int*>(bars + 142);    // [4]
  int* sums = reinterpret_cast<int*>(bars + 144);                       // [28]
  static_assert((144 + 14) * 8 <= 1280, "shared memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y;

  grid_dependency_wait();
  grid_dependency_launch();

  // --- which rows -------------------------------------------------------------
  int* pre = reinterpret_cast<int*>(smem);  // where the tiles will be
  const int total = prompt_prefix<kPromptThreads>(p, pre, sums);
  const int most = p.split && total ? max(gridDim.x / total, 1u) : 1;  // CTAs of an item
  // the last items first: within a request they have the most keys
  const int item = total - 1 - static_cast<int>(blockIdx.x) / most, share = blockIdx.x % most;
  if (item < 0) return;
  const PromptItem x = prompt_item<kStep>(p, pre, item);
  const int b = x.b, tile = x.tile, first = x.first, len = x.len, rows = x.rows, before = x.before;
  const int tiles_q = rows > 128 ? 2 : 1;
  const Shares shares(x.steps, most);
  if (share >= shares.parts) return;
  const int step0 = x.step0 + share * shares.steps, steps = min(shares.steps, x.steps - share * shares.steps);
  __syncthreads();  // `pre` is read

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_ready + 8 * i, 8);
      mbar_init(k_full + 8 * i, 4);
      mbar_init(v_full + 8 * i, 4);
      mbar_init(spent + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(c_full + 8 * i, 4);
    mbar_init(finished, 1);
    *abort_flag = *drain_flag = 0;
    // for the end of the softmax warps, whose registers are few
    after[0] = shares.parts, after[1] = first, after[2] = tile * 256, after[3] = rows;
    fence_mbar_init();
  }
  if (warp == 24) tmem_alloc(smem_addr(tmem_slot), Cfg::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  auto wait_warp = [&](uint32_t at, int phase) {
    ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(at, phase & 1, abort_flag));
    return ok;
  };

  if (warp < 16) {
    // ------------------------------------------------------------- softmax
    take_registers<kSoftmaxRegs>();
    const int qi = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    if (qi < tiles_q) {
      const int r = tile * 256 + qi * 128 + row;
      const int token = r / p.group, h = head * p.group + r % p.group;
      const bool live = qi * 128 + row < rows;
      // the two warps of 32 rows meet here, and leave each other numbers there
      const int meet = 1 + 4 * qi + (warp & 3);
      float2* mine = reinterpret_cast<float2*>(smem + Cfg::kOffRows) + (2 * qi + half) * 128;
      const float2* other = mine + (half ? -128 : 128);
      // A wait that gave up ends both warps' work: neither may miss the other's barriers.
      auto gave_up = [&]() {
        ok = !named_bar_any(meet, 64, !ok);
        return !ok;
      };
      // half of this row of Q, its channels in the order that `centred` gives the codes
      float sumq = 0.f;
      {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) +
                              p.q_row * (first + token) + p.q_head * h;
        const uint32_t dst = smem_addr(smem) + qi * Cfg::kQ + row * 128;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int c = half * (D / 16) + i;
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
        mine[row].x = sumq;
        named_bar_sync(meet, 64);
        sumq = half ? other[row].x + sumq : sumq + other[row].x;
      }
      // a sum that the terms cannot hold is left to the careful form
      const bool big = !T::kBf16 && !(fabsf(sumq) < 60000.f);
      if (half == 0) {
        uint4 x[2];
        query_terms<T>(big ? 0.f : sumq, x);
        const uint32_t dst = smem_addr(smem) + Cfg::kOffQx + qi * Cfg::kQx + row * 32;
        sts128(dst + ((row >> 2 & 1) << 4), x[0]);
        sts128(dst + ((row >> 2 & 1 ^ 1) << 4), x[1]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      const bool usual = !__any_sync(0xffffffffu, big);
      if (lane == 0) mbar_arrive(q_ready + 8 * qi);

      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      constexpr int kRest = kStep / 16 - 4;  // chunks of 16 keys that the second half has; the first has four
      const int chunks = half ? kRest : 4, key0 = 64 * half;
      const uint32_t s_at = tmem + lanes + Cfg::kColS + kStep * qi + key0;
      const uint32_t o_at = tmem + lanes + Cfg::kColO + kN * qi;
      // this thread's rows of the scores: 8 i + lane / 4 of the warp's, i < 4
      const int w0 = qi * 128 + (warp & 3) * 32, t2 = 2 * (lane & 3);
      // positions of this warp's first and last row
      const int lo = before + (tile * 256 + w0) / p.group;
      const int hi = before + (tile * 256 + max(w0, min(rows, w0 + 32) - 1)) / p.group;
      // from a number of each of those rows to that of row `lane`
      auto of_lane = [&](const float (&x)[4]) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = __shfl_sync(0xffffffffu, x[i], (lane & 7) * 4);
          if (lane >> 3 == i) y = z;
        }
        return y;
      };
      float top[4], l[4], off[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) top[i] = kLowest, l[i] = off[i] = 0.f;
      int largest = -1000;  // exponent of a value scale up to here
      // This thread's row of the result up to the last step that was a multiple of
      // kFreshSteps: every second 16 channels, and the sums' 16 columns.
      constexpr int kSettled = D / 32 + 1;
      volatile float settled[16 * kSettled];
      for (int it = 0; it < steps; ++it) {
        const int buf = it & 3;
        wait_warp(c_full + 8 * buf, it >> 2);
        const Numbers& k = numbers[buf];
        const int j0 = (step0 + it) * kStep;
        bool done = false;
        const int4 up = *reinterpret_cast<const int4*>(range + 8 * buf);
        const int4 down = *reinterpret_cast<const int4*>(range + 8 * buf + 4);
        largest = max(largest, max(max(up.x, up.y), max(up.z, up.w)));
        const int smallest = min(min(down.x, down.y), min(down.z, down.w));
        const int4 all_fine = *reinterpret_cast<const int4*>(fine + 4 * buf);
        const bool plain = usual && largest - smallest <= 6 && (all_fine.x & all_fine.y & all_fine.z & all_fine.w);
        wait_warp(s_full + 8 * qi, it);
        if (gave_up()) break;
        tc_fence_after();
        if (plain && it % kFreshSteps != 0 && j0 + kStep <= lo + 1 && (p.window == 0 || hi - j0 < p.window)) {
          // the step with the maximum as it is
          uint32_t weights[2][16];  // of either 16 lanes
          float mx[2] = {kLowest, kLowest};
          F2 top2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) top2[i] = pack2(-top[i], -top[i]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c >= kRest && c >= chunks) break;
            uint32_t s[16];
            tmem_load_fragment(s_at + 16 * c, s);
            tmem_load_fragment(s_at + (16u << 16) + 16 * c, s + 8);
            tmem_loaded(s);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2 ks = *reinterpret_cast<const float2*>(k.scale + key0 + 16 * c + 8 * j + t2);
              const F2 ks2 = pack2(ks.x, ks.y);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t* x = s + 8 * (i >> 1) + 4 * j + 2 * (i & 1);
                const float2 y = unpack2(fma2(ks2, pack2(__uint_as_float(x[0]), __uint_as_float(x[1])), top2[i]));
                mx[j] = max3(mx[j], y.x, y.y);
                weights[i >> 1][4 * c + 2 * j + (i & 1)] = Half::down(exp2_approx(y.x), exp2_approx(y.y));
              }
            }
          }
          done = !named_bar_any(meet, 64, fmaxf(mx[0], mx[1]) > kMoveAt);
          if (done) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t at = s_at + (i ? 16u << 16 : 0u);
              if (kRest == 4 || half == 0) {
                tmem_store_fragment<8>(at, weights[i]);
              } else {
                tmem_store_fragment<4>(at, weights[i]);
                tmem_store_fragment<2>(at + 16, weights[i] + 8);
              }
            }
          }
        }
        if (!done) {
          // With the maximum of the step first.  What a row does not see has no
          // weight, whatever lies in its place.
          uint32_t seen[4];  // keys before the row's last one
          int first_key[4];  // the step's, counted from the row's first one
          float sums[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = before + (tile * 256 + w0 + 8 * i + (lane >> 2)) / p.group;
            const int oldest = p.window && pos >= p.window ? pos - p.window + 1 : 0;
            seen[i] = pos < 0 ? 0 : pos - oldest;
            first_key[i] = pos < 0 ? -1000 : j0 - oldest;  // a row before all keys sees none
            sums[i] = __shfl_sync(0xffffffffu, sumq, 8 * i + (lane >> 2));
          }
          const uint32_t* in_k = plain_k + 4 * buf;
          const uint32_t* in_v = plain_v + 4 * buf;
          auto bit = [&](const uint32_t* mask, int i) { return mask[i >> 5] >> (i & 31) & 1; };
          auto argument = [&](int r, int i, uint32_t s) {  // of key i of the step for row r
            if (static_cast<uint32_t>(first_key[r] + i) > seen[r]) return -CUDART_INF_F;
            float x = __uint_as_float(s);
            if (!bit(valid + 4 * buf, i)) return -CUDART_INF_F;
            const bool held = bit(in_k, i);
            if (!held || !T::kBf16 && !(fabsf(sums[r]) < 60000.f)) x = fmaf(k.z[i], sums[r], x);
            return fmaf(k.scale[i], x, held ? 0.f : k.log_s[i]);
          };
          auto plain_argument = [&](int r, int i, uint32_t s, float scale) {
            const float x = __uint_as_float(s) * scale;
            return static_cast<uint32_t>(first_key[r] + i) > seen[r] ? -CUDART_INF_F : x;
          };
          float mx[4] = {kLowest, kLowest, kLowest, kLowest};
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            uint32_t s[16];
            tmem_load_fragment(s_at + 16 * c, s);
            tmem_load_fragment(s_at + (16u << 16) + 16 * c, s + 8);
            tmem_loaded(s);
            if (plain) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int at = key0 + 16 * c + 8 * j + t2;
                const float2 ks = *reinterpret_cast<const float2*>(k.scale + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint32_t* x = s + 8 * (r >> 1) + 4 * j + 2 * (r & 1);
                  mx[r] = max3(mx[r], plain_argument(r, at, x[0], ks.x), plain_argument(r, at + 1, x[1], ks.y));
                }
              }
            } else
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int r = 2 * (i >> 3) + (i >> 1 & 1);
              mx[r] = fmaxf(mx[r], argument(r, key0 + 16 * c + 8 * (i >> 2 & 1) + t2 + (i & 1), s[i]));
            }
          }
          bool moves = false;
          const int row0 = (warp & 3) * 32 + (lane >> 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            if ((lane & 3) == 0) mine[row0 + 8 * i].y = mx[i];
          }
          named_bar_sync(meet, 64);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mx[i] = fmaxf(mx[i], other[row0 + 8 * i].y);
            moves |= mx[i] > top[i] + kMoveAt;
          }
          if (__any_sync(0xffffffffu, moves) || it % kFreshSteps == 0) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float next = fmaxf(top[i], mx[i] - kWeightTop);
              f[i] = exp2_approx(top[i] - next);
              top[i] = next;
              l[i] *= f[i];
              off[i] *= f[i];
            }
            if (it > 0) {
              const float fl = of_lane(f);
              wait_warp(spent + 8 * (it & 1), it >> 1);
              if (gave_up()) break;
              tc_fence_after();
              if (it % kFreshSteps != 0) {
#pragma unroll 1
                for (int c = half; c < kN / 16; c += 2) {
                  uint32_t o[16];
                  tmem_load_16(o_at + 16 * c, o);
                  tmem_loaded(o);
#pragma unroll
                  for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fl);
                  tmem_store_16(o_at + 16 * c, o);
                }
              }
              if (it >= kFreshSteps) {
#pragma unroll 1
                for (int c = 0; c < kSettled; ++c) {
                  uint32_t o[16] = {};
                  if (it % kFreshSteps == 0) {
                    tmem_load_16(o_at + (c == D / 32 ? D : 32 * c + 16 * half), o);
                    tmem_loaded(o);
                  }
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                    settled[16 * c + i] =
                        (__uint_as_float(o[i]) + (it > kFreshSteps ? settled[16 * c + i] : 0.f)) * fl;
                }
              }
            }
          }
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            uint32_t s[16];
            tmem_load_fragment(s_at + 16 * c, s);
            tmem_load_fragment(s_at + (16u << 16) + 16 * c, s + 8);
            tmem_loaded(s);
            uint32_t weights[8];
            if (plain) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int at = key0 + 16 * c + 8 * j + t2;
                const float2 ks = *reinterpret_cast<const float2*>(k.scale + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint32_t* x = s + 8 * (r >> 1) + 4 * j + 2 * (r & 1);
                  weights[4 * (r >> 1) + 2 * j + (r & 1)] =
                      Half::down(exp2_approx(plain_argument(r, at, x[0], ks.x) - top[r]),
                                 exp2_approx(plain_argument(r, at + 1, x[1], ks.y) - top[r]));
                }
              }
            } else
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 2 * (i >> 2) + (i & 1), at = key0 + 16 * c + 8 * (i >> 1 & 1) + t2;
              const float x0 = argument(r, at, s[2 * i]), x1 = argument(r, at + 1, s[2 * i + 1]);
              const float w0 = exp2_approx(x0 - top[r]), w1 = exp2_approx(x1 - top[r]);
              weights[4 * (i >> 2) + (i & 3)] = Half::down(w0, w1);
              // what the sums' columns do not hold, or what the weights lose
              const float2 w = Half::up(weights[4 * (i >> 2) + (i & 3)]);
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const float rest = (z ? w1 : w0) - (bit(in_v, at + z) ? z ? w.y : w.x : 0.f);
                if ((z ? x1 : x0) != -CUDART_INF_F) {
                  l[r] = fmaf(rest, k.inv_s[at + z], l[r]);
                  off[r] = fmaf(rest, k.at_mid[at + z], off[r]);
                }
              }
            }
            // in the place of products already read
            tmem_store_fragment<2>(s_at + 8 * c, weights);
            tmem_store_fragment<2>(s_at + (16u << 16) + 8 * c, weights + 4);
          }
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 8 * qi);
      }
      // from here on one row a thread
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int z = 1; z < 4; z <<= 1) {
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], z);
          off[i] += __shfl_xor_sync(0xffffffffu, off[i], z);
        }
      float sum = of_lane(l), rest = of_lane(off);
      named_bar_sync(meet, 64);  // the other has read what is there
      mine[row] = make_float2(sum, rest);
      named_bar_sync(meet, 64);
      sum = half ? other[row].x + sum : sum + other[row].x;
      rest = half ? other[row].y + rest : rest + other[row].y;
      // (the last phase of a `spent` can only be told from the one before the one
      // before it once that one is over)
      if (steps > 0 && wait_warp(spent + 8 * (steps - 1 & 1), (steps - 1) >> 1) &&
          wait_warp(spent + 8 * (steps & 1), steps >> 1)) {
        tc_fence_after();
        uint32_t o[16];
        tmem_load_16(o_at + D, o);
        tmem_loaded(o);
        sum += 4.f * (__uint_as_float(o[0]) + __uint_as_float(o[1]));
        rest += __uint_as_float(o[2]) + __uint_as_float(o[3]);
        if (steps > kFreshSteps) {
          const volatile float* more = settled + 16 * (D / 32);
          sum += 4.f * (more[0] + more[1]);
          rest += more[2] + more[3];
        }
      }
      const float over = sum == 0.f ? 0.f : 1.f / sum;
      auto value = [&](uint32_t x) { return fmaf(0.5f, __uint_as_float(x), rest) * over; };  // codes were twice
      const bool whole = after[0] == 1, there = qi * 128 + row < after[3];
      const int at = after[2] + qi * 128 + row, at_token = at / p.group;
      uint8_t* dst = p.out + 2 * ((static_cast<int64_t>(after[1] + at_token) * p.q_heads + head * p.group + at -
                                   at_token * p.group) * D);
      // a part: [16 channels][row][16] results, the rows' maxima and sums
      float* part = p.partials + (blockIdx.y * gridDim.x + blockIdx.x) * (256 * (D + 2)) + qi * 128 + row;
      const float highest = of_lane(top);
      if (!whole && half == 0) {
        part[256 * D] = highest;
        part[256 * (D + 1)] = sum;
      }
      part += 15 * (qi * 128 + row);
      if (ok) {
#pragma unroll 1
        for (int c = half; c < D / 16; c += 2) {
          uint32_t o[16] = {};
          if (steps > 0) {
            tmem_load_16(o_at + 16 * c, o);
            tmem_loaded(o);
          }
          if (!there) continue;
          if (steps > kFreshSteps) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + settled[16 * (c >> 1) + i]);
          }
          if (!whole) {
            float4* to = reinterpret_cast<float4*>(part + c * (256 * 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
              if (sum != 0.f)
                y = make_float4(value(o[4 * i]), value(o[4 * i + 1]), value(o[4 * i + 2]), value(o[4 * i + 3]));
              to[i] = y;
            }
            continue;
          }
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = sum == 0.f ? 0u : T::down(value(o[2 * i]), value(o[2 * i + 1]));
          *reinterpret_cast<uint4*>(dst + 32 * c) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(dst + 32 * c + 16) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
  } else if (warp < 24) {
    // ------------------------------------------- codes to operand tiles
    // Warps 16-19 the keys' (and what the softmax needs to know), 20-23 the
    // values'.  Codes are in registers a step ahead; where a step's tiles lie is
    // looked up two steps ahead.  Once a wait has given up these warps run on
    // without waiting: they meet at a barrier every step, which none of them
    // may leave alone.
    give_registers<kOperandRegs>();
    const bool keys = warp < 20;
    const int dw = warp & 3, id = dw * 32 + lane, meet = keys ? 9 : 10;
    const int per_page = p.cache.page_size / kTile;
    uint64_t* tiles = tile_at + (keys ? 0 : 32);
    auto look_up = [&](int it) {  // where the step's cache tiles are
      if (dw == 0 && lane < kTiles && it < steps) {
        const int t = (step0 + it) * kTiles + lane;
        uint64_t at = 0;
        if (static_cast<int64_t>(t) * kTile < len) {
          const int page = p.tables[p.table_stride * b + t / per_page];
          if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.pages))
            at = reinterpret_cast<uint64_t>(p.cache.tile<D>(page, head, t % per_page));
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
          const uint8_t* src = half < 2 * kTiles ? tile_of(it, half >> 1) : nullptr;
          codes[u] = src ? *reinterpret_cast<const uint4*>(src + off_k(D, (half & 1) * 8 + (lane & 7)) + 16 * chunk)
                         : make_uint4(0, 0, 0, 0);
        }
        const uint8_t* src = id < kStep ? tile_of(it, id >> 4) : nullptr;
        here = src != nullptr && (step0 + it) * kStep + id < len;
        kp = here ? *reinterpret_cast<const uint32_t*>(src + off_k_pair(D, id & 15)) : 0u;
        vp = here ? *reinterpret_cast<const uint32_t*>(src + off_v_pair(D, id & 15)) : 0u;
      };
      load(0);
      for (int it = 0; it < steps; ++it) {
        const int stage = it & 1, buf = it & 3;
        look_up(it + 2);
        if (it >= 2) wait_warp(spent + 8 * stage, (it >> 1) - 1);
        {
          // A row without a scale has all codes 0: any scale tells the same.
          const float2 ks = T::up(kp);
          const float s = ks.x > 0.f ? ks.x : fmaxf(fabsf(ks.y) * 0x1p-10f, 0x1p-10f);
          const float z = __fdividef(ks.y, s) + 8.f, scale = s * c2;
          const MiddleRow v = middle_row(T::up(vp));
          const float log = __fdividef(v.log_s, scale);
          const bool held = here && terms_hold<T>(z, log);
          Numbers& k = numbers[buf];
          k.scale[id] = scale;
          k.z[id] = z;
          k.log_s[id] = v.log_s;
          k.inv_s[id] = v.inv_s;
          k.at_mid[id] = v.at_mid;
          reinterpret_cast<uint16_t*>(smem + Cfg::kOffMiddles + buf * 256)[id] =
              static_cast<uint16_t>(Half::down(1024.f + v.twice, 0.f));
          const uint32_t mask = __ballot_sync(0xffffffffu, here);
          const uint32_t mask_k = __ballot_sync(0xffffffffu, held);
          const uint32_t mask_v = __ballot_sync(0xffffffffu, here && sums_hold(v));
          const bool beyond = id >= kStep || (step0 + it) * kStep + id >= len;
          const int all_fine = __all_sync(0xffffffffu, beyond || (held && sums_hold(v)));
          const int e = static_cast<int>(__float_as_uint(v.inv_s) >> 23);  // 254 less the scale's
          const int up = __reduce_max_sync(0xffffffffu, here ? 254 - e : -1000);
          const int down = __reduce_min_sync(0xffffffffu, here ? 254 - e : 1000);
          if (lane == 0) {
            fine[4 * buf + dw] = all_fine;
            range[8 * buf + dw] = up;
            range[8 * buf + 4 + dw] = down;
            valid[4 * buf + dw] = mask;
            plain_k[4 * buf + dw] = mask_k;
            plain_v[4 * buf + dw] = mask_v;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(c_full + 8 * buf);
          if (id < kStep) {
            uint4 x[2];
            key_terms<T>(held ? z : 0.f, held ? log : 0.f, x);
            const uint32_t dst = smem_addr(smem) + Cfg::kOffKx + stage * Cfg::kKx + id * 32;
            sts128(dst + ((id >> 2 & 1) << 4), x[0]);
            sts128(dst + ((id >> 2 & 1 ^ 1) << 4), x[1]);
          }
        }
        const uint32_t dst = smem_addr(smem) + Cfg::kOffK + stage * Cfg::kK;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int rest = (u * 128 + id) >> 3, chunk = rest % kUnits, half = rest / kUnits;
          if (half >= 2 * kTiles) continue;
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
      const bool serves = half < 2 * kTiles;
      uint32_t vp = 0;                 // of value `id`
      bool here = false;
      // the columns after the sums' are nothing
      for (int i = id; i < 2 * 2 * 12 * 8; i += 128) {
        const int chunk = i & 7, r = (i >> 3) % 12, atom = i / 96 & 1, stage = i / 192;
        sts128(smem_addr(smem) + Cfg::kOffV + stage * Cfg::kV + atom * (kN * 128) + (D + 4 + r) * 128 + 16 * chunk,
               make_uint4(0, 0, 0, 0));
      }
      uint32_t w[8 * kWordsV];         // of the eight tokens of a half tile: [token][kWordsV]
      auto load = [&](int it) {
        if (it >= steps) return;
        const uint8_t* pair = id < kStep ? tile_of(it, id >> 4) : nullptr;
        here = pair != nullptr && (step0 + it) * kStep + id < len;
        vp = here ? *reinterpret_cast<const uint32_t*>(pair + off_v_pair(D, id & 15)) : 0u;
        const uint8_t* src = serves ? tile_of(it, half >> 1) : nullptr;
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
        if (it >= 2) wait_warp(spent + 8 * (stage ^ 1), (it - 1) >> 1);
        const uint32_t dst = smem_addr(smem) + Cfg::kOffV + stage * Cfg::kV;
        if (id < kStep) {
          const MiddleRow v = middle_row(T::up(vp));
          const bool held = here && sums_hold(v);
          const float inv = held ? 0.25f * v.inv_s : 0.f, z = held ? v.at_mid : 0.f;
          const float h = rounded<Half>(inv), zh = rounded<Half>(z);
          const uint32_t x = Half::down(h, inv - h), y = Half::down(zh, z - zh);
          const uint32_t at = dst + (id >> 6) * (kN * 128) + 2 * (id & 7);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint16_t number = static_cast<uint16_t>((r < 2 ? x : y) >> (16 * (r & 1)));
            asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + (D + r) * 128 + (((id >> 3 & 7) ^ ((D + r) & 7)) << 4)),
                         "h"(number)
                         : "memory");
          }
        }
        wait_warp(c_full + 8 * (it & 3), it >> 2);  // the middles are there
        half2 middle[4];                            // of tokens 2t and 2t + 1
        {
          const uint4 x = lds128(smem_addr(smem) + Cfg::kOffMiddles + (it & 3) * 256 + 16 * half);
          const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int t = 0; t < 4; ++t) middle[t] = *reinterpret_cast<const half2*>(&y[t]);
        }
        if (serves)
#pragma unroll
        for (int o = 0; o < kWordsV; ++o) {
#pragma unroll
          for (int part = 0; part < 4; ++part) {  // channels 2 part and 2 part + 1 of the octet
            half2 even[4], odd[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {  // tokens 2t and 2t + 1
              const uint32_t y = prmt(w[2 * t * kWordsV + o], w[(2 * t + 1) * kWordsV + o], part < 2 ? 0x5410 : 0x7632);
              even[t] = twice_off(y, 2 * (part & 1), middle[t]);
              odd[t] = twice_off(y, 2 * (part & 1) + 1, middle[t]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int d = piece * (D / 8) + 8 * o + 2 * part + x;
              const half2* z = x ? odd : even;
              sts128(dst + (half >> 3) * (kN * 128) + d * 128 + (((half & 7) ^ (d & 7)) << 4),
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
    if (__shfl_sync(0xffffffffu, warp, 0) == 24 && steps > 0) {
      // ---------------------------------------------------------- products
      constexpr uint32_t types = T::kBf16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t id_s = umma_idesc_f16_f32(kStep) | types, id_o = umma_idesc_f16_f32(kN);
      const uint32_t base = smem_addr(smem), t0 = __shfl_sync(0xffffffffu, tmem, 0);
      auto scores = [&](int qi, int stage) {
        const uint64_t q_desc = umma_desc_sw128_k(base + qi * Cfg::kQ);
        const uint64_t k_desc = umma_desc_sw128_k(base + Cfg::kOffK + stage * Cfg::kK);
        const uint32_t s_at = t0 + Cfg::kColS + kStep * qi;
        warp_umma_ss<4>(s_at, q_desc, k_desc, id_s, 0);
        if constexpr (D == 128) warp_umma_ss<4>(s_at, q_desc + (128 * 128 >> 4), k_desc + (kStep * 128 >> 4), id_s, 1);
        warp_umma_ss<1>(s_at, umma_desc_sw32_k(base + Cfg::kOffQx + qi * Cfg::kQx),
                     umma_desc_sw32_k(base + Cfg::kOffKx + stage * Cfg::kKx), id_s, 1);
        warp_umma_commit(s_full + 8 * qi);
      };
      bool go = wait_warp(k_full, 0);
      for (int qi = 0; qi < tiles_q && go; ++qi) {
        go = wait_warp(q_ready + 8 * qi, 0);
        if (!go) break;
        tc_fence_after();
        scores(qi, 0);
      }
      warp_umma_commit(spent);
      for (int it = 0; it < steps && go; ++it) {
        const int stage = it & 1, next = (it + 1) & 1;
        const bool more = it + 1 < steps;
        go = wait_warp(v_full + 8 * stage, it >> 1) && (!more || wait_warp(k_full + 8 * next, (it + 1) >> 1));
        for (int qi = 0; qi < tiles_q && go; ++qi) {
          go = wait_warp(p_ready + 8 * qi, it);
          if (!go) break;
          tc_fence_after();
          const uint64_t v_desc = umma_desc_sw128_k(base + Cfg::kOffV + stage * Cfg::kV);
          const uint32_t s_at = t0 + Cfg::kColS + kStep * qi, o_at = t0 + Cfg::kColO + kN * qi;
          warp_umma_ts<4>(o_at, s_at, v_desc, id_o, it % kFreshSteps != 0);
          warp_umma_ts<kStep / 16 - 4>(o_at, s_at + 64, v_desc + (kN * 128 >> 4), id_o, 1);
          if (more) scores(qi, next);
        }
        warp_umma_commit(spent + 8 * next);
      }
      warp_umma_commit(finished);
      mbar_wait_bounded(finished, 0, drain_flag);
    }
  }
  if (!ok && lane == 0) atomicOr(p.status, kStatusFullWaitTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 24) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kCols);
  }
}

// The parts of items whose keys were shared out: a thread joins 16 channels of a
// row, a CTA 32 rows.
template <class T, int D>
__global__ void __launch_bounds__(2 * D) kv4_prompt_join_kernel(const __grid_constant__ PromptParams p) {
  __shared__ int pre[kSplitBatch], sums[2 * D / 32];
  grid_dependency_wait();
  grid_dependency_launch();
  const int total = prompt_prefix<2 * D>(p, pre, sums);
  const int item = total - 1 - static_cast<int>(blockIdx.x / 8);
  if (item < 0) return;
  // gridDim.x is 8 times the most items there can be; the other kernel's is p.split
  const int most = max(p.split / total, 1);
  const PromptItem x = prompt_item<PromptCfg<D>::kStep>(p, pre, item);
  const Shares shares(x.steps, most);
  const int row = blockIdx.x % 8 * 32 + threadIdx.x % 32, c = threadIdx.x / 32;
  if (shares.parts < 2 || row >= x.rows) return;
  constexpr int kPart = 256 * (D + 2);
  const float* part = p.partials + (static_cast<int>(blockIdx.y) * p.split + (total - 1 - item) * most) * kPart;
  float top = kLowest;
#pragma unroll 8
  for (int i = 0; i < shares.parts; ++i) top = fmaxf(top, __ldcg(part + i * kPart + 256 * D + row));
  float y[16] = {}, sum = 0.f;
#pragma unroll 2
  for (int i = 0; i < shares.parts; ++i) {
    const float* at = part + i * kPart;
    const float w = __ldcg(at + 256 * (D + 1) + row) * exp2_approx(__ldcg(at + 256 * D + row) - top);
    sum += w;
    const float4* from = reinterpret_cast<const float4*>(at + (c * 256 + row) * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = __ldcg(from + j);
      y[4 * j] = fmaf(w, v.x, y[4 * j]), y[4 * j + 1] = fmaf(w, v.y, y[4 * j + 1]);
      y[4 * j + 2] = fmaf(w, v.z, y[4 * j + 2]), y[4 * j + 3] = fmaf(w, v.w, y[4 * j + 3]);
    }
  }
  const float over = sum == 0.f ? 0.f : 1.f / sum;
  const int r = x.tile * 256 + row, token = r / p.group, h = blockIdx.y * p.group + r % p.group;
  uint4* dst = reinterpret_cast<uint4*>(
      p.out + 2 * ((static_cast<int64_t>(x.first + token) * p.q_heads + h) * D + 16 * c));
#pragma unroll
  for (int j = 0; j < 2; ++j)
    dst[j] = make_uint4(T::down(y[8 * j] * over, y[8 * j + 1] * over), T::down(y[8 * j + 2] * over, y[8 * j + 3] * over),
                        T::down(y[8 * j + 4] * over, y[8 * j + 5] * over),
                        T::down(y[8 * j + 6] * over, y[8 * j + 7] * over));
}

}  // namespace kv4
}  // namespace sm100
