// C ABI and launches of the 4-bit paged key/value cache (kv4_*.cuh).
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/sm100_marlin.h"
#include "kv4_cache.cuh"
#include "kv4_decode.cuh"
#include "kv4_prompt.cuh"
#include "kv4_schedule.cuh"

namespace sm100 {

// sm100_marlin.cu
int cuda_fail(cudaError_t e);
int kernel_status(int dev, int** out);  // device address of the status word
int sm_count(int dev, int* sms);
bool overlap_enabled();                 // programmatic launches (sm100_marlin_set_overlap)

namespace {

using namespace kv4;

// Makes `dev` current for a launch; the caller's device comes back on scope exit.
struct OnDevice {
  int prev = -1;
  cudaError_t error;
  explicit OnDevice(int dev) : error(cudaGetDevice(&prev)) {
    if (error == cudaSuccess && prev != dev) {
      error = cudaSetDevice(dev);
    } else {
      prev = -1;
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

int launched(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? SM100_MARLIN_OK : cuda_fail(e);
}

// A launch that may begin while the kernel before it on the stream ends.  Every
// kernel here waits for that one before it touches global memory, and only then
// lets the next one begin: a GEMM fetches its weights before it waits, and a
// kernel before this one may be writing them.
template <class Params>
cudaError_t launch(void (*kernel)(Params), dim3 grid, int threads, int smem, cudaStream_t stream, const Params& p) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = overlap_enabled() ? 1 : 0;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, p);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_cache(const void* cache, int pages, int heads, int page_size, int dim, int dtype) {
  if (dim != 64 && dim != 128) return SM100_MARLIN_ERR_KERN_SHAPE;
  if (dtype != SM100_MARLIN_FP16 && dtype != SM100_MARLIN_BF16) return SM100_MARLIN_ERR_ARGUMENT;
  if (pages < 0 || heads <= 0 || page_size <= 0 || page_size % kTile != 0)
    return SM100_MARLIN_ERR_PROB_SHAPE;
  if (static_cast<int64_t>(pages) * page_size > 0x7fffffffll) return SM100_MARLIN_ERR_PROB_SHAPE;
  if (!cache && pages > 0) return SM100_MARLIN_ERR_ARGUMENT;
  return aligned(cache, 16) ? SM100_MARLIN_OK : SM100_MARLIN_ERR_ALIGNMENT;
}

// The opt-in to more than 48 KB of shared memory, once per kernel and device.
template <auto Kernel>
int allow_smem(int dev, int bytes) {
  static std::atomic<uint64_t> done{0};
  if (dev >= 0 && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return SM100_MARLIN_OK;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e);
  if (dev >= 0 && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return SM100_MARLIN_OK;
}

// Requests with at most this many query rows for a key/value head go to the
// decode kernel, others to the prompt kernel.  At 64 requests, 8 heads of 128, over
// 4096 tokens: 48 rows take 348 us here and 409 there, 64 rows 451 and 410 (bf16: 391
// and 420); 128 rows over 2048 tokens 453 and 242.
constexpr int kFewRows = 64;

std::atomic<int> stalled_cta{-1};  // sm100_marlin_kv4_stall

// Counters of the decode kernel's grid, then either kernel's parts.
constexpr size_t kCounterBytes = 4096;
constexpr size_t kPromptPart = 256 * (128 + 2);
static_assert(kPromptPart >= 2 * DecodeCfg<128, 2>::kPart, "parts");
size_t workspace_bytes(int sms) {
  return kCounterBytes + static_cast<size_t>(sms) * kPromptPart * sizeof(float);
}

template <class T, int D, int NT>
int launch_decode(DecodeParams p, int sms, int dev, cudaStream_t stream) {
  using Cfg = DecodeCfg<D, NT>;
  const int bad = allow_smem<kv4_decode_kernel<T, D, NT>>(dev, Cfg::kSmem);
  if (bad) return bad;
  // The kernel keeps a sum per request in shared memory, and counts steps in 32
  // bits: larger batches go in slices.  What it can meet counts here, not what the
  // caller says of the lengths.
  const int64_t all = static_cast<int64_t>(p.starts ? p.rows : 1) * p.group, most = all < p.most ? all : p.most;
  const int64_t steps = (static_cast<int64_t>(p.width) * p.cache.page_size / kStepTokens + 1) *
                        p.cache.heads * ((most + Cfg::kRows - 1) / Cfg::kRows);  // of a request, at most
  const int64_t fit = 0x3fffffffll / steps;
  if (fit < 1) return SM100_MARLIN_ERR_PROB_SHAPE;
  const int slice = static_cast<int>(fit < kDecodeBatch ? fit : kDecodeBatch), batch = p.batch;
  int done = 0;
  do {
    const int n = batch - done < slice ? batch - done : slice;
    p.batch = n;
    p.pad = (done + n == batch ? 1 : 0) | (done == 0 ? 2 : 0);
    const cudaError_t e = launch(kv4_decode_kernel<T, D, NT>, dim3(sms), Cfg::kThreads, Cfg::kSmem, stream, p);
    if (e != cudaSuccess) return cuda_fail(e);
    p.lens += n;
    p.tables += n * p.table_stride;
    p.row0 += n;
    if (p.starts) p.starts += n;
    done += n;
  } while (done < batch);
  return launched(cudaSuccess);
}

template <class T, int D>
int launch_prompt(PromptParams p, int sms, int dev, cudaStream_t stream) {
  const int bad = allow_smem<kv4_prompt_kernel<T, D>>(dev, PromptCfg<D>::kSmem);
  if (bad) return bad;
  // No more items than full ones and one rest for each request that is served;
  // CTAs without an item leave at once.
  const int64_t rows = static_cast<int64_t>(p.rows) * p.group;
  const int heads = p.cache.heads;
  for (int done = 0, batch = p.batch; done < batch; done += kPromptBatch) {
    p.batch = batch - done < kPromptBatch ? batch - done : kPromptBatch;
    const int64_t rests = rows / (p.most + 1);
    const int64_t items = rows / 256 + (rests < p.batch ? rests : p.batch);
    if (items > 0) {
      // Items that leave half of the GPU idle share out their keys, if they can have
      // enough of them (a last launch joins them): 256 rows of each of 8 heads over 16384
      // tokens take 87 us instead of 392.
      const int64_t keys = static_cast<int64_t>(p.width) * p.cache.page_size;
      p.split = batch <= kSplitBatch && 2 * items * heads <= sms && keys >= 2 * kLeastPromptSteps * PromptCfg<D>::kStep
                    ? sms / heads
                    : 0;
      cudaError_t e = launch(kv4_prompt_kernel<T, D>, dim3(p.split ? p.split : static_cast<unsigned>(items), heads),
                             kPromptThreads, PromptCfg<D>::kSmem, stream, p);
      if (e == cudaSuccess && p.split)
        e = launch(kv4_prompt_join_kernel<T, D>, dim3(static_cast<unsigned>(8 * items), heads), 2 * D, 0, stream, p);
      if (e != cudaSuccess) return cuda_fail(e);
    }
    p.lens += p.batch;
    p.tables += p.batch * p.table_stride;
    p.starts += p.batch;
  }
  return launched(cudaSuccess);
}

// f(T{}, std::integral_constant-like D) for the cache's type and head size.
template <int D>
struct Dim {
  static constexpr int value = D;
};
template <class F>
int dispatch(int dtype, int dim, F&& f) {
  if (dtype == SM100_MARLIN_FP16) return dim == 64 ? f(Half{}, Dim<64>{}) : f(Half{}, Dim<128>{});
  return dim == 64 ? f(Bf16{}, Dim<64>{}) : f(Bf16{}, Dim<128>{});
}

}  // namespace
}  // namespace sm100

using namespace sm100;
using namespace sm100::kv4;

extern "C" {

int sm100_marlin_kv4_schedule(const int* new_lens, const int* lens, int* block_tables,
                              int64_t table_stride, int width, int batch, int* free_pages,
                              int capacity, const int* free_count, int rows, int page_size,
                              int* lens_out, int* free_count_out, int* starts, int* slots,
                              int* positions, int* fate, int dev, void* stream) {
  if (batch < 0 || batch > kMaxBatch || rows < 0 || width < 0 || capacity < 0 || page_size <= 0)
    return SM100_MARLIN_ERR_PROB_SHAPE;
  if (!free_count || !free_count_out || !starts || (batch > 0 && (!new_lens || !lens || !lens_out || !fate)) ||
      (batch > 0 && width > 0 && !block_tables) || (capacity > 0 && !free_pages) ||
      (rows > 0 && (!slots || !positions)))
    return SM100_MARLIN_ERR_ARGUMENT;
  OnDevice on(dev);
  if (on.error != cudaSuccess) return cuda_fail(on.error);
  const ScheduleParams p{new_lens, lens, block_tables, table_stride, width, batch, free_pages,
                         capacity, free_count, rows, page_size, lens_out, free_count_out, starts,
                         slots, positions, fate};
  const int smem = 20 * batch;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        kv4_schedule_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 20 * kMaxBatch);
    if (e != cudaSuccess) return cuda_fail(e);
  }
  // One CTA where the new lengths or the new count lie in what is read: the others
  // would read it while it writes.
  auto overlap = [](const int* a, int64_t n, const int* b, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + 4 * m && y < x + 4 * n && n > 0 && m > 0;
  };
  bool in_place = overlap(lens_out, batch, free_count, 1) || overlap(free_count_out, 1, free_count, 1);
  for (const int* in : {new_lens, lens})
    in_place |= overlap(lens_out, batch, in, batch) || overlap(free_count_out, 1, in, batch);
  const int ctas = in_place ? 1 : 1 + (rows > batch ? rows : batch) / kScheduleThreads;
  return launched(launch(kv4_schedule_kernel, dim3(ctas < 148 ? ctas : 148), kScheduleThreads, smem,
                         static_cast<cudaStream_t>(stream), p));
}

int sm100_marlin_kv4_append(const void* k, int64_t k_row, int64_t k_head, const void* v,
                            int64_t v_row, int64_t v_head, void* cache, int pages, int kv_heads,
                            int page_size, int head_dim, int dtype, const int* slots, int tokens,
                            int dev, void* stream) {
  const int bad = check_cache(cache, pages, kv_heads, page_size, head_dim, dtype);
  if (bad) return bad;
  if (tokens < 0 || static_cast<int64_t>(tokens) * kv_heads > 0x7fffffffll) return SM100_MARLIN_ERR_PROB_SHAPE;
  if (tokens == 0) return SM100_MARLIN_OK;
  if (!k || !v || !slots) return SM100_MARLIN_ERR_ARGUMENT;
  if (!aligned(k, 2) || !aligned(v, 2)) return SM100_MARLIN_ERR_ALIGNMENT;
  OnDevice on(dev);
  if (on.error != cudaSuccess) return cuda_fail(on.error);
  const bool vector = aligned(k, 16) && aligned(v, 16) && ((k_row | k_head | v_row | v_head) & 7) == 0;
  const AppendParams p{{static_cast<uint8_t*>(cache), pages, kv_heads, page_size},
                       static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), k_row, k_head,
                       v_row, v_head, slots, tokens, vector};
  const int64_t threads = static_cast<int64_t>(tokens) * kv_heads * kRowLanes;
  return dispatch(dtype, head_dim, [&](auto type, auto dim) {
    return launched(launch(kv4_append_kernel<decltype(type), decltype(dim)::value>,
                           dim3(static_cast<unsigned>((threads + kCacheThreads - 1) / kCacheThreads)), kCacheThreads, 0,
                           static_cast<cudaStream_t>(stream), p));
  });
}

int sm100_marlin_kv4_read(const void* cache, int pages, int kv_heads, int page_size, int head_dim,
                          int dtype, const int* slots, int tokens, void* k, void* v, int dev,
                          void* stream) {
  const int bad = check_cache(cache, pages, kv_heads, page_size, head_dim, dtype);
  if (bad) return bad;
  if (tokens < 0 || static_cast<int64_t>(tokens) * kv_heads > 0x7fffffffll) return SM100_MARLIN_ERR_PROB_SHAPE;
  if (tokens == 0) return SM100_MARLIN_OK;
  if (!k || !v || !slots) return SM100_MARLIN_ERR_ARGUMENT;
  if (!aligned(k, 16) || !aligned(v, 16)) return SM100_MARLIN_ERR_ALIGNMENT;
  OnDevice on(dev);
  if (on.error != cudaSuccess) return cuda_fail(on.error);
  const ReadParams p{{static_cast<uint8_t*>(const_cast<void*>(cache)), pages, kv_heads, page_size},
                     static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), slots, tokens};
  const int64_t threads = static_cast<int64_t>(tokens) * kv_heads * kRowLanes;
  return dispatch(dtype, head_dim, [&](auto type, auto dim) {
    return launched(launch(kv4_read_kernel<decltype(type), decltype(dim)::value>,
                           dim3(static_cast<unsigned>((threads + kCacheThreads - 1) / kCacheThreads)), kCacheThreads, 0,
                           static_cast<cudaStream_t>(stream), p));
  });
}

int sm100_marlin_kv4_attention(const void* q, int64_t q_row, int64_t q_head, const void* cache,
                               int pages, int kv_heads, int page_size, int head_dim, int dtype,
                               const int* block_tables, int64_t table_stride, int width,
                               const int* lens, const int* starts, int batch, int rows, int q_heads,
                               int max_new, int window, float scale, void* out, void* workspace,
                               size_t workspace_bytes, int dev, void* stream) {
  const int bad = check_cache(cache, pages, kv_heads, page_size, head_dim, dtype);
  if (bad) return bad;
  if (batch < 0 || rows < 0 || width < 0 || q_heads <= 0 || q_heads % kv_heads != 0 || max_new < 0 ||
      (!starts && rows != batch))
    return SM100_MARLIN_ERR_PROB_SHAPE;
  if (window < 0) return SM100_MARLIN_ERR_ARGUMENT;
  if (rows == 0) return SM100_MARLIN_OK;
  if (!q || !out || (batch > 0 && (!lens || (width > 0 && !block_tables)))) return SM100_MARLIN_ERR_ARGUMENT;
  if (!aligned(q, 2) || !aligned(out, 16)) return SM100_MARLIN_ERR_ALIGNMENT;
  OnDevice on(dev);
  if (on.error != cudaSuccess) return cuda_fail(on.error);
  int sms = 0;
  int* status = nullptr;
  const int failed = sm_count(dev, &sms) | kernel_status(dev, &status);
  if (failed) return failed;
  if (!workspace || workspace_bytes < sm100::workspace_bytes(sms)) return SM100_MARLIN_ERR_SCRATCH;
  if (!aligned(workspace, 16)) return SM100_MARLIN_ERR_ALIGNMENT;
  // a window that holds all that a table can is none
  if (window >= static_cast<int64_t>(width) * page_size) window = 0;
  const Cache c{static_cast<uint8_t*>(const_cast<void*>(cache)), pages, kv_heads, page_size};
  const int group = q_heads / kv_heads;
  const bool vector = aligned(q, 16) && ((q_row | q_head) & 7) == 0;
  const int few_rows = group > kFewRows ? group : kFewRows;  // a single token is always few
  const int64_t most = static_cast<int64_t>(starts ? max_new : 1) * group;
  const DecodeParams few{c, static_cast<const uint8_t*>(q), q_row, q_head, vector,
                         static_cast<uint8_t*>(out), block_tables, table_stride, width, lens, starts,
                         0, batch, rows, 1, most <= few_rows, q_heads, group, window, few_rows, scale,
                         static_cast<int*>(workspace),
                         reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes), status,
                         stalled_cta.load(std::memory_order_relaxed)};
  const PromptParams many{c, static_cast<const uint8_t*>(q), q_row, q_head, vector, static_cast<uint8_t*>(out),
                          block_tables, table_stride, width, lens, starts, batch, rows, q_heads,
                          group, window, few_rows, scale, 0, few.partials, status};
  const cudaStream_t on_stream = static_cast<cudaStream_t>(stream);
  return dispatch(dtype, head_dim, [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    const int bad = most <= 8 ? launch_decode<T, D, 1>(few, sms, dev, on_stream)
                              : launch_decode<T, D, 2>(few, sms, dev, on_stream);
    return bad || most <= few_rows ? bad : launch_prompt<T, D>(many, sms, dev, on_stream);
  });
}

int sm100_marlin_kv4_stall(int cta) {
  if (cta < -1) return SM100_MARLIN_ERR_ARGUMENT;
  stalled_cta.store(cta, std::memory_order_relaxed);
  return SM100_MARLIN_OK;
}

size_t sm100_marlin_kv4_workspace_bytes(int dev) {
  int sms = 0;
  return sm_count(dev, &sms) ? 0 : workspace_bytes(sms);
}

}  // extern "C"
