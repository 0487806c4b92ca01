// Host/device declarations of the paged key-value cache operators (append,
// decode, evict) and of token scoring.
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace rp {

// Codes these kernels record in the device status word.
constexpr int kStatusBadPage = 0x201;    // a page id outside the pool
constexpr int kStatusBadLength = 0x202;  // a length below 0 or past the page table, bad starts
constexpr int kStatusBadToken = 0x203;   // a token id past the vocabulary

// Positions that a page table addresses, at most: loops over them step past the
// end by a grid's stride (4096 a CTA cluster, 1024 positions a CTA of the weights'
// launch), which has to fit an int.
constexpr int kMaxPositions = 0x7FFFFFFF - (1 << 23);

// Value types of a cache (rp_kv_dtype).
constexpr int kKvBf16 = 0, kKvF16 = 1, kKvE4m3 = 2;

// One pool of pages: row (page, head, slot) of K at k + (page * s_page +
// head * s_head + slot * s_slot) * element size, D elements; V alike.  e4m3
// rows have one fp32 scale each at ks / vs[(page * heads + head) * page_size
// + slot].
struct PagedPool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int64_t s_page, s_head, s_slot;
  int dtype, num_pages, heads, page_size, D;
};

// Page tables and lengths of B sequences: position p of sequence b is slot
// p % page_size of page table[b * stride + p / page_size].
struct PagedTable {
  const int32_t* table;
  int64_t stride;
  int pages;  // entries a row
  const int32_t* lengths;
  int B;
};

// Accumulated attention weights: sequence b, KV head h, position p at
// w + b * s_seq + h * s_head + p.
struct KeyWeights {
  float* w;
  int64_t s_seq, s_head;
};

struct AppendArgs {
  PagedPool kv;
  PagedTable t;
  const uint16_t* k_new;  // element (token, head, d)
  const uint16_t* v_new;
  int64_t k_tok, k_head, v_tok, v_head;  // element strides
  int in_f16;
  int tokens;
  const int32_t* starts;  // (B + 1) first new token of each sequence; null: one each
  KeyWeights weights;     // null w: none; else zeroed at the new positions
  int32_t* lengths_out;   // (B,)
  int* status;
};
cudaError_t launch_paged_append(const AppendArgs& a, cudaStream_t st);

struct PagedDecodeArgs {
  PagedPool kv;
  PagedTable t;
  const uint16_t* q;  // (B, Hq, D)
  int64_t q_seq, q_head;
  int q_f16;
  int Hq;
  float scale_log2;  // softmax scale * log2(e)
  uint16_t* out;     // (B, Hq, D) in the query's type
  int64_t o_seq, o_head;
  float* lse;          // (B, Hq) natural log, or null
  KeyWeights weights;  // null w: none
  void* workspace;
  int* status;
};
size_t paged_decode_workspace(const PagedPool& kv, int B, int Hq, int table_pages, bool weights);
cudaError_t launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t st);

struct EvictArgs {
  PagedPool kv;
  PagedTable t;
  KeyWeights weights;
  const int32_t* out_table;  // (B, out_pages)
  int64_t out_stride;
  int out_pages;
  int budget, recent;
  int32_t* kept;         // (B, heads, budget) positions in order, -1 past the end
  int32_t* lengths_out;  // (B,)
  float* weights_out;    // (B, heads, out_pages * page_size), 0 past the end
  int* status;
};
cudaError_t launch_paged_evict(const EvictArgs& a, cudaStream_t st);

constexpr int kMaxTop = 64;
struct ScoreArgs {
  const void* logits;  // row r at logits + r * stride elements
  int64_t stride;
  int dtype;  // rp_dtype
  int rows, vocab, top;
  const int64_t* tokens;  // (rows,); negative: none
  float* logprobs;        // (rows,)
  float* entropy;         // (rows,)
  float* top_logprobs;    // (rows, top)
  int64_t* top_ids;       // (rows, top)
  int* status;
};
cudaError_t launch_token_logprobs(const ScoreArgs& a, cudaStream_t st);

// Bytes of which every stride of the pool is a multiple (a power of two), if a
// row's offset then fits 32 bits; else 0.  A contiguous pool's unit is a row or
// more, so that only pools of terabytes, or of odd strides and over 64 GB, have
// none.
inline int64_t pool_unit(const PagedPool& kv) {
  const int64_t size = kv.dtype == kKvE4m3 ? 1 : 2, all = (kv.s_page | kv.s_head | kv.s_slot) * size;
  const int64_t unit = all == 0 ? 16 : all & -all;
  const int64_t rows[3] = {kv.num_pages - 1, kv.heads - 1, kv.page_size - 1};
  const int64_t strides[3] = {kv.s_page, kv.s_head, kv.s_slot};
  uint64_t span = 0;  // in units
  for (int i = 0; i < 3; ++i) {
    const uint64_t n = static_cast<uint64_t>(strides[i] * size / unit);
    if (rows[i] == 0) continue;
    if (n > 0xFFFFFFFFu) return 0;
    span += n * static_cast<uint64_t>(rows[i]);
  }
  return span > 0xFFFFFFFFu || unit > 0x80000000LL ? 0 : unit;
}

// Per-device settings of the launchers are kept for this many devices.
constexpr int kMaxDevices = 64;
inline int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}
// SMs of a device (148 on a whole B200), 0 if it cannot be asked.
inline int sm_count(int dev) {
  static std::atomic<int> known[kMaxDevices];
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
    known[dev].store(n, std::memory_order_relaxed);
  return n;
}

#ifdef __CUDACC__
// Programmatic launches: what follows may be launched; what came before is
// complete and its memory visible.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A launch that may begin while the launch before it ends (its kernel waits
// for that one's end itself).
template <typename F, typename A>
cudaError_t launch_after(F* kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, const A& arg) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, arg);
}

// Length of sequence b, held to what its page table can address.
__device__ __forceinline__ int table_length(const PagedTable& t, int page_size, int b, int* status) {
  const int n = t.lengths[b];
  const int64_t cap = static_cast<int64_t>(t.pages) * page_size;
  if (n < 0 || n > cap) {
    atomicCAS(status, 0, kStatusBadLength);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}

// Element offset of row (page of position p, head, slot), or -1 (with the
// status recorded) for a page id outside the pool.
__device__ __forceinline__ int64_t row_offset(const PagedPool& kv, const int32_t* table_row, int p,
                                              int head, int* status) {
  const int page = table_row[p / kv.page_size];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(kv.num_pages)) {
    atomicCAS(status, 0, kStatusBadPage);
    return -1;
  }
  return page * kv.s_page + head * kv.s_head + (p % kv.page_size) * kv.s_slot;
}

// Index of that row's scales.
__device__ __forceinline__ int64_t scale_index(const PagedPool& kv, const int32_t* table_row, int p,
                                               int head) {
  return (static_cast<int64_t>(table_row[p / kv.page_size]) * kv.heads + head) * kv.page_size +
         p % kv.page_size;
}
#endif

}  // namespace rp
