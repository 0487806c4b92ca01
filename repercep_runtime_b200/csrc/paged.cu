// Paged key-value cache: append and evict (see include/repercep_b200.h).
#include <cooperative_groups.h>

#include <atomic>

#include "internal.h"
#include "paged.h"
#include "quant_common.cuh"

namespace rp {
namespace {

namespace cg = cooperative_groups;

constexpr int kAppendThreads = 256;

// New rows into the cache.  A row of D 16-bit values is D / 8 16-byte
// vectors; a thread takes one, or for an e4m3 cache two, so that it stores 16
// bytes of K and of V each time (8 took 139 us where 16 take 115).  A CTA takes
// a run of rows, numbered (token, head) as the input has them.  While the K and
// V vectors of a thread's U rows are on their way, one thread per token finds
// its sequence, page and slot (done by every thread for every row, this took
// twice the time of the rest).  e4m3: the steps are the quantizer's
// (quant_common.cuh), so the bytes are those of the row-wise quantizer; K's and
// V's amax share the words of one shuffle reduction over the row's D / 16 lanes,
// and each lane then divides for one of the 2 U scales.  Reads 4 D bytes and
// writes 2 D (or 4 D) a row, bound by HBM.  Measured: 48 prompts of 512 to 4099
// tokens, 8 heads of 128, into an e4m3 cache 113 us, 6.3 TB/s (replayed in a
// graph), into a bf16 one 147, 6.3 TB/s; one token of 64 sequences 2.4 us.
template <int D, bool E4M3, bool F16, int U>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  constexpr int kVecs = E4M3 ? 2 : 1;               // 16-byte vectors of a thread: it writes 16 bytes of K and of V
  constexpr int kLanes = D / 8 / kVecs;             // threads a row
  constexpr int kAtOnce = kAppendThreads / kLanes;  // rows a CTA takes at once
  constexpr int kTokens = kAtOnce * U;              // tokens of a CTA, at most
  __shared__ int64_t offset[kTokens];               // of (token, head 0), -1: left out
  __shared__ int64_t scale_at[E4M3 ? kTokens : 1];
  __shared__ int64_t weight_at[kTokens];
  const uint32_t H = a.kv.heads, B = a.t.B;
  const int c = threadIdx.x % kLanes;
  const uint32_t rows = static_cast<uint32_t>(a.tokens) * H, begin = blockIdx.x * kTokens;
  const uint32_t r0 = begin + threadIdx.x / kLanes;
  const uint32_t next_tok = kAtOnce / H, next_head = kAtOnce % H;
  uint4 k[U][kVecs], v[U][kVecs];
  uint32_t tok[U], head[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t r = r0 + u * kAtOnce;
    tok[u] = u == 0 ? r / H : tok[u - 1] + next_tok;
    head[u] = u == 0 ? r - tok[u] * H : head[u - 1] + next_head;
    if (head[u] >= H) {
      head[u] -= H;
      ++tok[u];
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      k[u][i] = v[u][i] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        k[u][i] = __ldg(reinterpret_cast<const uint4*>(a.k_new + tok[u] * a.k_tok + head[u] * a.k_head) + c * kVecs + i);
        v[u][i] = __ldg(reinterpret_cast<const uint4*>(a.v_new + tok[u] * a.v_tok + head[u] * a.v_head) + c * kVecs + i);
      }
    }
  }
  for (uint32_t i = blockIdx.x * kAppendThreads + threadIdx.x; i < B; i += gridDim.x * kAppendThreads) {
    const int n = table_length(a.t, a.kv.page_size, i, a.status);
    int add = 1;
    if (a.starts) {  // the tokens of it that there are
      const int s0 = a.starts[i], s1 = a.starts[i + 1];
      if (s0 < 0 || s1 < s0 || s1 > a.tokens) atomicCAS(a.status, 0, kStatusBadLength);
      add = max(0, min(max(s1, 0), a.tokens) - max(s0, 0));
    }
    // what the table holds is counted; a negative length takes no token and stays: as a 0, the
    // next call's would go over position 0
    const int64_t after = min(static_cast<int64_t>(n) + add, static_cast<int64_t>(a.t.pages) * a.kv.page_size);
    a.lengths_out[i] = a.t.lengths[i] < 0 ? a.t.lengths[i] : static_cast<int>(after);
  }
  const uint32_t t0 = begin / H, t1 = (min(begin + kTokens, rows) + H - 1) / H;  // the run's tokens
  for (uint32_t i = threadIdx.x; begin < rows && i < t1 - t0; i += kAppendThreads) {
    const int t = static_cast<int>(t0 + i);
    int b = t, first = t;
    bool ok = true;
    if (a.starts) {  // the sequence with starts[b] <= t < starts[b + 1]
      ok = t >= __ldg(a.starts) && t < __ldg(a.starts + B);
      int lo = 0, hi = static_cast<int>(B) - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (__ldg(a.starts + mid) <= t) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      first = max(0, __ldg(a.starts + b));
    }
    int64_t off = -1;
    if (ok) {
      const int n = a.t.lengths[b];
      const int64_t pos = static_cast<int64_t>(n) + (t - first);
      if (n < 0 || pos >= static_cast<int64_t>(a.t.pages) * a.kv.page_size) {
        atomicCAS(a.status, 0, kStatusBadLength);
      } else {
        const int p = static_cast<int>(pos);
        const int32_t* row = a.t.table + b * a.t.stride;
        off = row_offset(a.kv, row, p, 0, a.status);
        if (E4M3 && off >= 0) scale_at[i] = scale_index(a.kv, row, p, 0);
        weight_at[i] = b * a.weights.s_seq + p;
      }
    }
    offset[i] = off;
  }
  __syncthreads();
  int64_t off[U];  // of the row; -1: left out
#pragma unroll
  for (int u = 0; u < U; ++u) {
    off[u] = -1;
    if (r0 + u * kAtOnce < rows && offset[tok[u] - t0] >= 0)
      off[u] = offset[tok[u] - t0] + static_cast<int64_t>(head[u]) * a.kv.s_head;
  }
  if constexpr (E4M3) {
    uint32_t m[U];  // amax bits: K's in the low half, V's in the high one
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = max(quant::absmax8(k[u][0]), quant::absmax8(k[u][1])) |
             max(quant::absmax8(v[u][0]), quant::absmax8(v[u][1])) << 16;
#pragma unroll
      for (int x = kLanes / 2; x > 0; x /= 2) m[u] = __vmaxu2(m[u], __shfl_xor_sync(0xffffffffu, m[u], x));
    }
    constexpr int kRounds = (2 * U + kLanes - 1) / kLanes;
    float mul[kRounds];  // of scale j = c + round * kLanes: row j / 2, K or V
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int j = c + i * kLanes;
      uint32_t mine = m[0], at_tok = tok[0], at_head = head[0];
      bool store = off[0] >= 0;
#pragma unroll
      for (int u = 1; u < U; ++u)
        if (j / 2 == u) {
          mine = m[u];
          at_tok = tok[u];
          at_head = head[u];
          store = off[u] >= 0;
        }
      const float scale = quant::scale_from_amax_bits<F16>(j % 2 ? mine >> 16 : mine & 0xffffu);
      mul[i] = __frcp_rn(scale);
      if (j < 2 * U && store)
        (j % 2 ? a.kv.vs : a.kv.ks)[scale_at[at_tok - t0] + static_cast<int64_t>(at_head) * a.kv.page_size] = scale;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float qk = __shfl_sync(0xffffffffu, mul[2 * u / kLanes], 2 * u % kLanes, kLanes);
      const float qv = __shfl_sync(0xffffffffu, mul[(2 * u + 1) / kLanes], (2 * u + 1) % kLanes, kLanes);
      if (off[u] < 0) continue;
      // a scale that is inf or NaN has a reciprocal that is not positive
      const uint2 k0 = quant::quant8_any<F16>(k[u][0], qk, qk > 0.f), k1 = quant::quant8_any<F16>(k[u][1], qk, qk > 0.f);
      const uint2 v0 = quant::quant8_any<F16>(v[u][0], qv, qv > 0.f), v1 = quant::quant8_any<F16>(v[u][1], qv, qv > 0.f);
      reinterpret_cast<uint4*>(a.kv.k + off[u])[c] = make_uint4(k0.x, k0.y, k1.x, k1.y);
      reinterpret_cast<uint4*>(a.kv.v + off[u])[c] = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (off[u] < 0) continue;
      reinterpret_cast<uint4*>(a.kv.k + 2 * off[u])[c] = k[u][0];
      reinterpret_cast<uint4*>(a.kv.v + 2 * off[u])[c] = v[u][0];
    }
  }
  if (a.weights.w && c == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (off[u] >= 0) a.weights.w[weight_at[tok[u] - t0] + head[u] * a.weights.s_head] = 0.f;
  }
}

template <int D, int U>
cudaError_t append_u(const AppendArgs& a, cudaStream_t st) {
  const int kRows = kAppendThreads / (D / 8) * (a.kv.dtype == kKvE4m3 ? 2 : 1) * U;  // of a CTA
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.kv.heads;
  int64_t grid = (rows + kRows - 1) / kRows;
  if (grid < 1) grid = 1;  // lengths_out
  const unsigned g = static_cast<unsigned>(grid);
  if (a.kv.dtype != kKvE4m3) append_kernel<D, false, false, U><<<g, kAppendThreads, 0, st>>>(a);
  else if (a.in_f16) append_kernel<D, true, true, U><<<g, kAppendThreads, 0, st>>>(a);
  else append_kernel<D, true, false, U><<<g, kAppendThreads, 0, st>>>(a);
  return cudaGetLastError();
}

// Two rows a thread once the GPU is full all the same (2048 threads an SM):
// the 48 prompts take 115 us with two, 132 with one, 145 with four; 49k rows of
// e4m3, which fill two thirds of it, 12.2 us with two and 11.2 with one.
template <int D>
cudaError_t append_d(const AppendArgs& a, cudaStream_t st) {
  const int64_t threads = static_cast<int64_t>(a.tokens) * a.kv.heads * (D / 8 / (a.kv.dtype == kKvE4m3 ? 2 : 1));
  return threads >= 2LL * 2048 * sm_count(current_device()) ? append_u<D, 2>(a, st) : append_u<D, 1>(a, st);
}

// Weights order: a key is larger when the weight is; -0 equals 0 and any NaN
// is above +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// The weight of a key (0 for -0, one NaN for all).
__device__ __forceinline__ float key_weight(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// ---- selection
//
// One cluster of CTAs per (sequence, KV head): each CTA keeps the keys of its
// slice of the row in shared memory, and the threshold (the want-th largest
// key) is found in at most three passes over them, 11, 11 and 10 bits at a
// time, with a histogram per CTA that every CTA of the cluster adds up through
// distributed shared memory: sums of 8 bins first, then the bins of one such
// sum.  (All 2048 bins at once take 4500 cycles a pass; counting the lanes of a
// bin by ballots or a match before one add costs more than the adds, also where
// weights are equal: 57 us against 52 for two long sequences.)  Two passes more
// count and place what is kept in order, so ties at the threshold go to the
// lowest positions.  Reads each weight from HBM once; bound by the latency of
// its few dependent passes, which the split over a cluster shortens.  Measured
// (replayed in a graph, with the move of the 64 rows kept): 16 rows of 70001 and
// 98303 weights 19 us, 128 rows of 1001 to 16385 18 us.
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
static_assert(kSelThreads >= 256, "a thread for every sum of 8 bins");
constexpr int kSelBatch = 8;  // keys of a thread in flight
constexpr int kBins = 2048;
constexpr int kCoarse = kBins / 8;
constexpr int kSelCluster = 16;        // CTAs of a row, at most (8 where a GPU cannot hold 16)
constexpr int kSliceAim = 4096;        // positions of a CTA that a larger cluster is not taken for
constexpr int kSliceHeld = 44 * 1024;  // positions of a CTA held in shared memory, at most

struct SelectShared {
  int4 hist[3][kBins / 4];
  int4 coarse[3][kCoarse / 4];
  int above[kSelWarps], ties[kSelWarps];  // of each warp's run
  int part_above, part_ties;              // of this CTA's slice
  int scan[kSelWarps];
  int digit, left, whole;
};

// HELD: every slice fits the shared memory; else keys are made from the
// weights again in each pass.
template <bool HELD>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t slice[];
  __shared__ SelectShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int h = blockIdx.x / parts, b = blockIdx.y, H = a.kv.heads;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  launch_next();
  const int n = table_length(a.t, a.kv.page_size, b, a.status);
  const int keep = min(n, a.budget);
  const float* w = a.weights.w + b * a.weights.s_seq + h * a.weights.s_head;
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * H + h) * a.budget;
  const int64_t out_cap = static_cast<int64_t>(a.out_pages) * a.kv.page_size;
  float* wo = a.weights_out + (static_cast<int64_t>(b) * H + h) * out_cap;
  const int stride = parts * kSelThreads, first = part * kSelThreads + t;
  // candidates [0, older), of which `want` stay; what is behind them stays whole
  const bool cut = n > a.budget;
  const int older = cut ? n - a.recent : n, want = cut ? a.budget - a.recent : n;
  const bool search = cut && want > 0;  // the same in the whole cluster
  const int per = (older + parts - 1) / parts, i0 = min(older, part * per);
  const int count = search ? min(older, i0 + per) - i0 : 0;
  if (HELD) {  // all of a thread's weights in flight at once
    for (int i = t; i < count; i += kSelThreads)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(slice + i)), "l"(w + i0 + i) : "memory");
  }
  if (blockIdx.x == 0 && t == 0) a.lengths_out[b] = keep;
  for (int i = keep + first; i < a.budget; i += stride) kept[i] = -1;
  for (int64_t i = keep + first; i < out_cap; i += stride) wo[i] = 0.f;
  for (int i = (cut ? older : 0) + first; i < n; i += stride) {
    kept[want - (cut ? older : want) + i] = i;
    wo[want - (cut ? older : want) + i] = w[i];
  }
  if (!search) return;

  for (int i = t; i < 3 * kBins / 4; i += kSelThreads) (&sh.hist[0][0])[i] = make_int4(0, 0, 0, 0);
  if (HELD) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    // a thread makes keys of the weights that it brought in itself
#pragma unroll 4
    for (int i = t; i < count; i += kSelThreads) slice[i] = weight_key(__uint_as_float(slice[i]));
  }
  __syncthreads();
  const auto key_at = [&](int i) { return HELD ? slice[i] : weight_key(__ldg(w + i0 + i)); };

  uint32_t thr = 0;
  int left = want;  // rank of the threshold among the keys that share its known bits
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 2 ? 10 : 11, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    int* hist = reinterpret_cast<int*>(sh.hist[pass]);
    for (int base = warp * 32; base < count; base += kSelBatch * kSelThreads) {
      uint32_t key[kSelBatch];
      bool in[kSelBatch];
#pragma unroll
      for (int u = 0; u < kSelBatch; ++u) {
        const int i = base + u * kSelThreads + lane;
        key[u] = i < count ? key_at(i) : 0;
        // equal known bits (all, in the first pass)
        in[u] = i < count && (pass == 0 || (key[u] ^ thr) >> (shift + bits) == 0);
      }
#pragma unroll
      for (int u = 0; u < kSelBatch; ++u) {
        if (in[u]) atomicAdd(&hist[(key[u] >> shift) & ((1 << bits) - 1)], 1);
      }
    }
    __syncthreads();
    if (t < kCoarse) {
      const int4 x = sh.hist[pass][2 * t], y = sh.hist[pass][2 * t + 1];
      reinterpret_cast<int*>(sh.coarse[pass])[t] = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    // a sum of 8 bins a thread, from the top: the one in which the running count reaches `left`
    int c = 0, before = 0;
    if (t < kCoarse) {
#pragma unroll
      for (int q = 0; q < kSelCluster; ++q)
        if (q < parts) c += reinterpret_cast<const int*>(cluster.map_shared_rank(&sh, q)->coarse[pass])[kCoarse - 1 - t];
      before = c;
#pragma unroll
      for (int s = 1; s < 32; s *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, before, s);
        if (lane >= s) before += x;
      }
      if (lane == 31) sh.scan[warp] = before;
    }
    __syncthreads();
    if (t < kCoarse) {
      before -= c;
#pragma unroll
      for (int i = 0; i < kCoarse / 32; ++i) before += i < warp ? sh.scan[i] : 0;
      if (before < left && before + c >= left) {
        sh.digit = kCoarse - 1 - t;
        sh.left = left - before;
      }
    }
    __syncthreads();
    // its bins, by one warp: lane i sums bin 7 - i % 8 over every fourth CTA
    if (warp == 0) {
      const int group = sh.digit, rest = sh.left, bin = group * 8 + 7 - (lane & 7);
      int m = 0;
#pragma unroll
      for (int i = 0; i < kSelCluster / 4; ++i) {
        const int q = (lane >> 3) + 4 * i;
        if (q < parts) m += reinterpret_cast<const int*>(cluster.map_shared_rank(&sh, q)->hist[pass])[bin];
      }
      m += __shfl_xor_sync(0xffffffffu, m, 8);
      m += __shfl_xor_sync(0xffffffffu, m, 16);
      int run = m;
#pragma unroll
      for (int s = 1; s < 8; s *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, run, s, 8);
        if ((lane & 7) >= s) run += x;
      }
      __syncwarp();
      if (lane < 8 && run - m < rest && run >= rest) {
        sh.digit = bin;
        sh.left = rest - (run - m);
        sh.whole = run == rest;
      }
    }
    __syncthreads();
    thr |= static_cast<uint32_t>(sh.digit) << shift;
    left = sh.left;  // among the keys of this bin; after the last pass, the ties to take
    if (sh.whole) {  // all of the bin stays: what is above the key below it (no key is 0)
      thr -= 1;
      left = 0;
      break;
    }
  }

  // ---- places: each warp a run of the slice, in order
  const int run = (count + kSelWarps - 1) / kSelWarps, r0 = min(count, warp * run), r1 = min(count, r0 + run);
  int above = 0, ties = 0;
#pragma unroll 8
  for (int i = r0 + lane; i < r1; i += 32) {
    const uint32_t key = key_at(i);
    above += key > thr;
    ties += key == thr;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) {
    sh.above[warp] = above;
    sh.ties[warp] = ties;
  }
  __syncthreads();
  int at_above = 0, at_ties = 0;
#pragma unroll
  for (int q = 0; q < kSelWarps; ++q) {
    at_above += q < warp ? sh.above[q] : 0;
    at_ties += q < warp ? sh.ties[q] : 0;
  }
  if (parts > 1) {
    if (t == kSelThreads - 1) {  // of the last warp: the whole slice
      sh.part_above = at_above + above;
      sh.part_ties = at_ties + ties;
    }
    cluster.sync();
    // lane q reads what CTA q's slice holds
    int2 p = make_int2(0, 0);
    if (lane < part) {
      const SelectShared* other = cluster.map_shared_rank(&sh, lane);
      p = make_int2(other->part_above, other->part_ties);
    }
    at_above += __reduce_add_sync(0xffffffffu, p.x);
    at_ties += __reduce_add_sync(0xffffffffu, p.y);
    cluster.barrier_arrive();  // the others' shared memory is read until here
  }
  for (int base = r0; base < r1; base += 32 * kSelBatch) {
    uint32_t gt[kSelBatch], eq[kSelBatch];
    uint32_t key[kSelBatch];
#pragma unroll
    for (int u = 0; u < kSelBatch; ++u) {
      const int i = base + u * 32 + lane;
      key[u] = i < r1 ? key_at(i) : 0;
      gt[u] = __ballot_sync(0xffffffffu, i < r1 && key[u] > thr);
      eq[u] = __ballot_sync(0xffffffffu, i < r1 && key[u] == thr);
    }
#pragma unroll
    for (int u = 0; u < kSelBatch; ++u) {
      const uint32_t below = (1u << lane) - 1;
      const int tie = at_ties + __popc(eq[u] & below);  // ties before this one
      if (((gt[u] >> lane) & 1) || (((eq[u] >> lane) & 1) && tie < left)) {
        const int at = at_above + __popc(gt[u] & below) + min(tie, left);
        kept[at] = i0 + base + u * 32 + lane;
        wo[at] = key_weight(key[u]);
      }
      at_above += __popc(gt[u]);
      at_ties += __popc(eq[u]);
    }
  }
  if (parts > 1) cluster.barrier_wait();
}

// ---- move
//
// Kept rows to their new places: a warp takes 8 rows, their places found by 8
// lanes, with K and V of all of them in flight before the first store.  Bound by
// HBM: 4096 rows of 128 sequences and heads (bf16, D 128) 85 us under the
// profiler, 6.1 TB/s read and written; 100 us with the selection's launch.
constexpr int kMoveRows = 8;
constexpr int kMoveWarps = 8;

template <int ROW>  // bytes of a row
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictArgs a) {
  constexpr int kLanes = ROW / 16;                               // lanes of a row
  constexpr int kTurns = kMoveRows * kLanes > 32 ? kMoveRows * kLanes / 32 : 1;  // vectors of K a lane
  constexpr int kAtOnce = 32 / kLanes;                           // rows of a turn
  const int lane = threadIdx.x & 31;
  const int j0 = (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * kMoveRows, h = blockIdx.y, b = blockIdx.z;
  const int H = a.kv.heads;
  const int j = j0 + lane;
  wait_previous();
  const int p = lane < kMoveRows && j < a.budget ? a.kept[(static_cast<int64_t>(b) * H + h) * a.budget + j] : -1;
  int64_t from = -1, to = -1;
  if (p >= 0) {
    const int32_t* from_row = a.t.table + b * a.t.stride;
    const int32_t* to_row = a.out_table + b * a.out_stride;
    from = row_offset(a.kv, from_row, p, h, a.status);
    to = row_offset(a.kv, to_row, j, h, a.status);
    if (from < 0 || to < 0) {
      to = -1;
    } else if (a.kv.ks) {
      const int64_t i = scale_index(a.kv, from_row, p, h), o = scale_index(a.kv, to_row, j, h);
      const float ks = a.kv.ks[i], vs = a.kv.vs[i];
      a.kv.ks[o] = ks;
      a.kv.vs[o] = vs;
    }
  }
  const int size = a.kv.dtype == kKvE4m3 ? 1 : 2;
  const int col = lane % kLanes * 16;
  uint4 k[kTurns], v[kTurns];
  int64_t dst[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = i * kAtOnce + lane / kLanes;
    const int64_t src = __shfl_sync(0xffffffffu, from, r % 32) * size + col;
    const int64_t d = __shfl_sync(0xffffffffu, to, r % 32);
    dst[i] = d < 0 || r >= kMoveRows ? -1 : d * size + col;
    if (dst[i] >= 0) {
      k[i] = __ldcs(reinterpret_cast<const uint4*>(a.kv.k + src));
      v[i] = __ldcs(reinterpret_cast<const uint4*>(a.kv.v + src));
    }
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i)
    if (dst[i] >= 0) {
      *reinterpret_cast<uint4*>(a.kv.k + dst[i]) = k[i];
      *reinterpret_cast<uint4*>(a.kv.v + dst[i]) = v[i];
    }
}

// Clusters of 16 CTAs are allowed if the device can hold one of them.
template <typename F>
cudaError_t select_clusters(F* kernel, size_t smem, int* most) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kSelCluster);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kSelCluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
  if (e != cudaSuccess) return e;
  *most = clusters > 0 ? kSelCluster : kSelCluster / 2;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs& a, cudaStream_t st) {
  switch (a.kv.D) {
    case 32: return append_d<32>(a, st);
    case 64: return append_d<64>(a, st);
    case 128: return append_d<128>(a, st);
    case 256: return append_d<256>(a, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_paged_evict(const EvictArgs& a, cudaStream_t st) {
  static std::atomic<int> most_parts[kMaxDevices];  // CTAs of a cluster, once this device is set up
  const int dev = current_device();
  int most = most_parts[dev].load(std::memory_order_relaxed);
  if (most == 0) {
    cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSliceHeld * 4);
    if (e == cudaSuccess) e = select_clusters(evict_select_kernel<true>, kSliceHeld * 4, &most);
    int other = 0;
    if (e == cudaSuccess) e = select_clusters(evict_select_kernel<false>, 0, &other);
    if (e != cudaSuccess) return e;
    if (other < most) most = other;
    most_parts[dev].store(most, std::memory_order_relaxed);
  }
  const int64_t cap = static_cast<int64_t>(a.t.pages) * a.kv.page_size;
  int parts = 1;
  // a larger cluster while the slices are long and the GPU holds all CTAs at once: three an SM at
  // slices of kSliceAim, fewer at longer ones, which then run in turns (96 rows of 98303 in
  // clusters of four 80 us, of eight 63, of two 224: those slices do not fit the shared memory)
  while (parts < most && cap > static_cast<int64_t>(parts) * kSliceAim &&
         static_cast<int64_t>(a.kv.heads) * a.t.B * parts * 2 <= 3 * sm_count(dev))
    parts *= 2;
  const int64_t per = (cap + parts - 1) / parts;
  const bool held = per <= kSliceHeld;
  if (static_cast<int64_t>(a.kv.heads) * parts > 0x7FFFFFFF) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.kv.heads * parts, a.t.B);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = held ? static_cast<size_t>(per) * 4 : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = held ? cudaLaunchKernelEx(&cfg, evict_select_kernel<true>, a)
                       : cudaLaunchKernelEx(&cfg, evict_select_kernel<false>, a);
  if (e != cudaSuccess) return e;
  constexpr int kRows = kMoveRows * kMoveWarps;
  const dim3 grid((a.budget + kRows - 1) / kRows, a.kv.heads, a.t.B);
  switch (a.kv.D * (a.kv.dtype == kKvE4m3 ? 1 : 2)) {
    case 32: return launch_after(evict_move_kernel<32>, grid, kMoveWarps * 32, 0, st, a);
    case 64: return launch_after(evict_move_kernel<64>, grid, kMoveWarps * 32, 0, st, a);
    case 128: return launch_after(evict_move_kernel<128>, grid, kMoveWarps * 32, 0, st, a);
    case 256: return launch_after(evict_move_kernel<256>, grid, kMoveWarps * 32, 0, st, a);
    case 512: return launch_after(evict_move_kernel<512>, grid, kMoveWarps * 32, 0, st, a);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rp
