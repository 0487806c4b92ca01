// Paged key-value cache: append and evict (see include/repercep_b200.h).
#include "internal.h"
#include "paged.h"
#include "quant_common.cuh"

namespace rp {
namespace {

constexpr int kAppendThreads = 256;

// New rows into the cache.  A row of D 16-bit values is D / 8 16-byte
// vectors, one a thread, so a warp holds 256 / D rows; K and V of a row are
// loaded together.  Rows are numbered (token, head), as the input has them.
// e4m3: the amax of a row is a shuffle over its D / 8 lanes, and the steps
// are the quantizer's (quant_common.cuh), so the bytes are those of the
// row-wise quantizer.  Reads 4 D bytes and writes 2 D (or 4 D) a row.
template <int D, bool E4M3, bool F16>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  constexpr int kLanes = D / 8;  // threads a row
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x;
  const int H = a.kv.heads, B = a.t.B;
  if (gid < B) {
    const int n = table_length(a.t, a.kv.page_size, static_cast<int>(gid), a.status);
    const int64_t add = a.starts ? static_cast<int64_t>(a.starts[gid + 1]) - a.starts[gid] : 1;
    a.lengths_out[gid] = static_cast<int>(n + (add > 0 ? add : 0));
  }
  const int64_t r = gid / kLanes;
  const int c = static_cast<int>(gid % kLanes);
  if (r >= static_cast<int64_t>(a.tokens) * H) return;  // whole rows: the shuffles below stay in a row
  const int t = static_cast<int>(r / H), h = static_cast<int>(r % H);
  int b = t, first = t;
  if (a.starts) {  // the sequence with starts[b] <= t < starts[b + 1]
    if (t < a.starts[0] || t >= a.starts[B]) return;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.starts[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    first = a.starts[b];
  }
  const int64_t pos = static_cast<int64_t>(table_length(a.t, a.kv.page_size, b, a.status)) + (t - first);
  if (pos < 0 || pos >= static_cast<int64_t>(a.t.pages) * a.kv.page_size) {
    if (c == 0) atomicCAS(a.status, 0, kStatusBadLength);
    return;
  }
  const int p = static_cast<int>(pos);
  const int32_t* row = a.t.table + b * a.t.stride;
  const int64_t off = row_offset(a.kv, row, p, h, a.status);
  if (off < 0) return;
  const uint4 k = __ldg(reinterpret_cast<const uint4*>(a.k_new + t * a.k_tok + h * a.k_head) + c);
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(a.v_new + t * a.v_tok + h * a.v_head) + c);
  if constexpr (E4M3) {
    uint32_t mk = quant::absmax8(k), mv = quant::absmax8(v);
    const unsigned lanes = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1) << (threadIdx.x & 31 & ~(kLanes - 1));
#pragma unroll
    for (int s = kLanes / 2; s > 0; s /= 2) {
      mk = max(mk, __shfl_xor_sync(lanes, mk, s));
      mv = max(mv, __shfl_xor_sync(lanes, mv, s));
    }
    const float sk = quant::scale_from_amax_bits<F16>(mk), sv = quant::scale_from_amax_bits<F16>(mv);
    reinterpret_cast<uint2*>(a.kv.k + off)[c] = quant::quant8_any<F16>(k, __frcp_rn(sk), isfinite(sk));
    reinterpret_cast<uint2*>(a.kv.v + off)[c] = quant::quant8_any<F16>(v, __frcp_rn(sv), isfinite(sv));
    if (c == 0) {
      const int64_t i = scale_index(a.kv, row, p, h);
      a.kv.ks[i] = sk;
      a.kv.vs[i] = sv;
    }
  } else {
    reinterpret_cast<uint4*>(a.kv.k + 2 * off)[c] = k;
    reinterpret_cast<uint4*>(a.kv.v + 2 * off)[c] = v;
  }
  if (a.weights.w && c == 0) a.weights.w[b * a.weights.s_seq + h * a.weights.s_head + p] = 0.f;
}

template <int D>
cudaError_t append_d(const AppendArgs& a, unsigned grid, cudaStream_t st) {
  if (a.kv.dtype != kKvE4m3) append_kernel<D, false, false><<<grid, kAppendThreads, 0, st>>>(a);
  else if (a.in_f16) append_kernel<D, true, true><<<grid, kAppendThreads, 0, st>>>(a);
  else append_kernel<D, true, false><<<grid, kAppendThreads, 0, st>>>(a);
  return cudaGetLastError();
}

// Weights order: a key is larger when the weight is; -0 equals 0 and any NaN
// is above +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;

__device__ __forceinline__ int block_sum(int x, int* buf) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if (lane == 0) buf[warp] = x;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < kSelectThreads / 32 ? buf[lane] : 0);
}

// Exclusive prefix of x over the block's threads; *total: the sum.
__device__ __forceinline__ int block_prefix(int x, int* buf, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int y = x;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    const int z = __shfl_up_sync(0xffffffffu, y, s);
    if (lane >= s) y += z;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = y;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    if (w < warp) before += buf[w];
    all += buf[w];
  }
  *total = all;
  return before + y - x;
}

// Positions to keep, one CTA per (sequence, head): the threshold is the
// largest key with at least `want` candidates at or above it, found bit by
// bit; ties at it go to the lowest positions.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ int buf[kSelectThreads / 32];
  const int h = blockIdx.x, b = blockIdx.y, H = a.kv.heads;
  const int n = table_length(a.t, a.kv.page_size, b, a.status);
  const int keep = min(n, a.budget);
  const float* w = a.weights.w + b * a.weights.s_seq + h * a.weights.s_head;
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * H + h) * a.budget;
  const int64_t out_cap = static_cast<int64_t>(a.out_pages) * a.kv.page_size;
  float* wo = a.weights_out + (static_cast<int64_t>(b) * H + h) * out_cap;
  if (h == 0 && threadIdx.x == 0) a.lengths_out[b] = keep;
  const int older = n > a.budget ? n - a.recent : n;   // candidates [0, older)
  const int want = n > a.budget ? a.budget - a.recent : n;
  uint32_t thr = 0;
  int above = 0;  // candidates above thr
  if (want < older) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = thr | (1u << bit);
      int c = 0;
      for (int i = threadIdx.x; i < older; i += kSelectThreads) c += weight_key(w[i]) >= t;
      if (block_sum(c, buf) >= want) thr = t;
    }
    int c = 0;
    for (int i = threadIdx.x; i < older; i += kSelectThreads) c += weight_key(w[i]) > thr;
    above = block_sum(c, buf);
  }
  int out = 0, ties = want - above;  // ties still to take
  for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t key = i < older ? weight_key(w[i]) : 0;
    const bool all = want >= older;
    const bool tie = !all && i < older && key == thr;
    int n_tie = 0, n_out = 0;
    const int tie_at = block_prefix(tie, buf, &n_tie);
    const bool take = i < n && (i >= older || all || key > thr || (tie && tie_at < ties));
    const int at = out + block_prefix(take, buf, &n_out);
    if (take) {
      kept[at] = i;
      wo[at] = w[i];
    }
    ties -= min(n_tie, ties);
    out += n_out;
  }
  for (int i = keep + threadIdx.x; i < a.budget; i += kSelectThreads) kept[i] = -1;
  for (int64_t i = keep + threadIdx.x; i < out_cap; i += kSelectThreads) wo[i] = 0.f;
}

// Rows to their new places, one warp per kept row.
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a, int row_bytes) {
  const int lane = threadIdx.x & 31;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z, H = a.kv.heads;
  if (j >= a.budget) return;
  const int p = a.kept[(static_cast<int64_t>(b) * H + h) * a.budget + j];
  if (p < 0) return;
  const int32_t* from_row = a.t.table + b * a.t.stride;
  const int32_t* to_row = a.out_table + b * a.out_stride;
  const int64_t from = row_offset(a.kv, from_row, p, h, a.status);
  const int64_t to = row_offset(a.kv, to_row, j, h, a.status);
  if (from < 0 || to < 0) return;
  const int size = a.kv.dtype == kKvE4m3 ? 1 : 2;
  for (int c = lane * 16; c < row_bytes; c += 512) {
    const uint4 k = *reinterpret_cast<const uint4*>(a.kv.k + from * size + c);
    const uint4 v = *reinterpret_cast<const uint4*>(a.kv.v + from * size + c);
    *reinterpret_cast<uint4*>(a.kv.k + to * size + c) = k;
    *reinterpret_cast<uint4*>(a.kv.v + to * size + c) = v;
  }
  if (a.kv.ks && lane == 0) {
    const int64_t i = scale_index(a.kv, from_row, p, h), o = scale_index(a.kv, to_row, j, h);
    a.kv.ks[o] = a.kv.ks[i];
    a.kv.vs[o] = a.kv.vs[i];
  }
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs& a, cudaStream_t st) {
  const int64_t threads = static_cast<int64_t>(a.tokens) * a.kv.heads * (a.kv.D / 8);
  const int64_t grid = ((threads > a.t.B ? threads : a.t.B) + kAppendThreads - 1) / kAppendThreads;
  if (grid == 0) return cudaSuccess;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const unsigned g = static_cast<unsigned>(grid);
  switch (a.kv.D) {
    case 32: return append_d<32>(a, g, st);
    case 64: return append_d<64>(a, g, st);
    case 128: return append_d<128>(a, g, st);
    case 256: return append_d<256>(a, g, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_paged_evict(const EvictArgs& a, cudaStream_t st) {
  evict_select_kernel<<<dim3(a.kv.heads, a.t.B), kSelectThreads, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const dim3 grid((a.budget + 7) / 8, a.kv.heads, a.t.B);
  evict_move_kernel<<<grid, 256, 0, st>>>(a, a.kv.D * (a.kv.dtype == kKvE4m3 ? 1 : 2));
  return cudaGetLastError();
}

}  // namespace rp
