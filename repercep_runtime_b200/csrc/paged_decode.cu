// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b of length n, KV head h and each of the G = Hq / Hkv query
// heads g that share it:
//   s_gj = scale * q_g . k_j,  m_g = max_j s_gj,  l_g = sum_j 2^(s_gj - m_g)
//   out_g = sum_j 2^(s_gj - m_g) v_j / l_g,  lse_g = ln 2 * (m_g + log2 l_g)
// (s in log2 units), and on request w[b, h, j] += sum_g 2^(s_gj - m_g) / l_g.
// A sequence without tokens gives out = 0 and lse = -inf.
//
// Every cached row is read once and meets G queries only, so the kernel is
// bound by HBM: its work is to keep enough bytes in flight on every SM.
//  - Work: the tiles (64 or 128 keys) of all (sequence, KV head) items in one
//    line, cut into equal runs, one per resident CTA, whatever the lengths.  An
//    item inside one run is finished there; an item that a cut splits leaves
//    (m, l, O) partials, at most two per CTA, that a second kernel joins in
//    order.  Workspace and launches do not depend on the lengths, and nothing
//    is atomic: equal inputs give equal bits.
//  - Loads: each warp streams its own slice of every tile through a ring of
//    its own in shared memory (16-byte cp.async, the page ids one step ahead),
//    so there is no CTA-wide barrier between tiles.
//  - Products: keys are the 16 rows of mma.m16n8k16 and the group's queries
//    its 8 columns (S^T = K Q^T, O^T = V^T P^T): a group of up to 8 heads costs
//    one column block.  At the memory's rate they take 15 to 19 % of the tensor
//    pipe's cycles; tcgen05's 128 rows would meet the same few queries.
//  - e4m3 rows are widened to fp16 exactly.  The queries are brought to fp16
//    by a power of two of their row's maximum, the rows' K scales multiply the
//    scores in fp32, and their V scales the softmax weights.  The products of
//    weight and V scale enter fp16 over a running power of two of their own
//    maximum in each column (over the largest V scale alone, a large row of no
//    weight pushed the others' out of fp16's range).  A row whose scale is 0
//    (fp16 rows of zeros or below 1.27e-5, whose scale the quantizer rounds to 0
//    and whose zeros are NaN bytes) is cleared in shared memory first.
//  - Rounding: scores, sums and accumulators are fp32.  For the product with a
//    16-bit V a softmax weight is split into a 16-bit value and the 16-bit
//    remainder, two products each, which cost 1 % of the time; rounded once it
//    added as much error as the output's own rounding (2.2e-3 against 1.7e-3 in
//    all); an fp16 pair holds 2^-36 of the row's largest weight.  With an e4m3
//    cache it is rounded once, with its V scale, to fp16: relative 2^-11, and
//    absolutely 2^-35 of the column's largest such product (two parts there cost
//    2 to 10 %: 233 us for the batch below, 73 for 16 heads a KV head).
// Measured (whole calls, replayed in a graph): two sequences of 115k tokens, 32/8
// heads, fp16 155 us (6.4 TB/s); 64 sequences of 512 to 520, 32/32 heads, bf16 88
// us (6.2 TB/s), with weights 92; 128 of 1 to 8191, 32/8 heads, e4m3, with weights
// 224 us.  Under the profiler, caches flushed: main kernel, join and weights of
// that batch 206, 8 and 21 us, the long case's main kernel 152 us (6.5 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "internal.h"
#include "paged.h"
#include "ptx.cuh"

namespace rp {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kJoinThreads = 512;
constexpr int kMaxCtas = 592;  // CTAs of the main kernel, at most
constexpr int kMinTiles = 2;    // tiles of a CTA's run, at least (but for the last)
// e4m3: a weight times its row's V scale enters fp16 times a power of two of its
// column's, which brings the largest such product to 2^10 or more, falls when one
// exceeds 2^15, rises as the weights fall with their reference, and is at most 2^110.
constexpr float kWeightTop = 32768.f;
constexpr uint32_t kWeightMost = 127 + 110;

template <int KV, int D, int NT>
struct Cfg {
  static constexpr bool kFp8 = KV == kKvE4m3;
  static constexpr bool kBf16 = KV == kKvBf16;
  static constexpr int kRow = D * (kFp8 ? 1 : 2);   // bytes of a row
  static constexpr int kChunks = kRow / 16;         // 16-byte chunks of a row
  static constexpr int kFrags = D / 16 * NT;  // accumulator fragments (float4 a lane)
  // The reference m of a row's weights 2^(s - m) (log2 units): a new one lies kBelow
  // under the maximum, and stays until a score exceeds it by kAbove.  e4m3: weights
  // are at most 1, so that a product with any V scale is finite, and references are
  // whole numbers.  fp16: the largest lie in [2^11, 2^15], so that small ones keep
  // clear of the format's lower end.
  static constexpr float kBelow = kFp8 ? -8.f : kBf16 ? 0.f : 11.f;
  static constexpr float kAbove = kFp8 ? 0.f : kBf16 ? 8.f : 15.f;
  // keys of a warp's step: 16 where that makes 8 KB (a stage holds a warp's accumulators at times)
  static constexpr int kKeys = 32 * kRow >= 8192 && 32 * kRow >= kFrags * 512 ? 16 : 32;
  static constexpr int kTile = kKeys * kWarps;
  static constexpr int kRowsBytes = kKeys * kRow;
  static constexpr int kStage = 2 * kRowsBytes + (kFp8 ? kKeys * 8 : 0);
  static_assert(kStage >= kFrags * 512, "a stage holds a warp's accumulators");
  // 16 KB a warp, so that three CTAs share an SM
  static constexpr int kStages = 2 * kRowsBytes >= 8192 ? 2 : 2 * kRowsBytes >= 4096 ? 4 : 6;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSmem = kWarps * kRing + kWarps * NT * 8 * 8 + kWarps * kStages * 4;
};

// What a CTA left for the join: the item it began (tile 0) without ending it
// and the slot of that partial, and the item it continued (slot 0).
struct Cut {
  int begun, begun_slot, continued, pad;
};

struct Params {
  PagedDecodeArgs a;
  int G;       // query heads of a KV head
  int groups;  // column groups of a KV head (NT * 8 query heads each)
  int shift;   // log2 of the page size, or -1
  // The pool's strides in units of their largest common power of two (bytes):
  // a row's offset is then a 32-bit number.
  uint32_t u_page, u_head, u_slot, unit;
  int grid;    // CTAs of the main kernel
  int score_pitch;
  float4* part_o;  // (grid * 2, kFrags, 32)
  float* part_ml;  // (grid * 2, 2, NT * 8)
  Cut* cuts;       // (grid)
  float* lse2;     // (B, Hq) log2-sum-exp, with weights only
  float* scores;   // (B, Hq, score_pitch) log2 units, with weights only
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Cached rows leave L2 first and scores last: a row is read once (for every
// sequence that names its page), while a later launch reads the scores (e4m3 batch
// with weights: 228 us in all, 234 without the second).  That launch gives their
// lines back: left as they were, they kept part of L2 from the kernels that came
// after (80 MB summed again and again took 20.5 us a pass instead of 16.4, with no
// end).
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ uint64_t evict_last() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void store_kept(float* dst, float x, uint64_t policy) {
  asm volatile("st.global.L2::cache_hint.f32 [%0], %1, %2;" ::"l"(dst), "f"(x), "l"(policy) : "memory");
}
__device__ __forceinline__ float4 load_once(const float* src, uint64_t policy) {
  float4 x;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.f32 {%0, %1, %2, %3}, [%4], %5;"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "l"(src), "l"(policy)
               : "memory");
  return x;
}
// The 128-byte line of `at` leaves L2 when its turn comes.
__device__ __forceinline__ void give_back_line(const float* at) {
  asm volatile("applypriority.global.L2::evict_normal [%0], 128;" ::"l"(reinterpret_cast<uint64_t>(at) & ~127ull)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
               "r"(read ? 16 : 0), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(read ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 8x8 transpose across the warp: (row lane / 4, columns 2 (lane % 4), + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two e4m3 values (low 16 bits) as two fp16, exactly.
__device__ __forceinline__ uint32_t widen_lo(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t y;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ float value16(uint32_t u, bool f16) {
  return f16 ? __half2float(__ushort_as_half(static_cast<uint16_t>(u))) : __uint_as_float(u << 16);
}
__device__ __forceinline__ uint16_t round16(float x, bool f16) {
  return f16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// A place in the line of tiles: sequence, item of the sequence (KV head and
// column group), tile of the item.
struct Place {
  int b, item, tile, n, tiles;
  template <typename C>
  __device__ __forceinline__ void enter(const Params& p) {
    n = table_length(p.a.t, p.a.kv.page_size, b, p.a.status);
    tiles = (n + C::kTile - 1) / C::kTile;
  }
  // The next tile; the line goes on (a sequence without tiles has none of it).
  template <typename C>
  __device__ __forceinline__ void next(const Params& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++item < p.a.kv.heads * p.groups) return;
    item = 0;
    tiles = 0;
    while (++b < p.a.t.B && tiles == 0) {
      enter<C>(p);
      if (tiles > 0) return;
    }
  }
};

// Writes one head's output row elements and its log-sum-exp; (m, l) in log2
// units.
__device__ __forceinline__ void write_lse(const Params& p, int b, int hq, float m, float l) {
  const float y = l == 0.f ? -INFINITY : m + log2f(l);
  if (p.lse2) p.lse2[static_cast<int64_t>(b) * p.a.Hq + hq] = y;
  if (p.a.lse) p.a.lse[static_cast<int64_t>(b) * p.a.Hq + hq] = kLn2 * y;
}

// Dimension of accumulator row r (lane / 4, + 8 for the second half) of
// fragment block dt: e4m3's transposed loads interleave even and odd ones.
template <bool FP8>
__device__ __forceinline__ int dim_of(int dt, int r, int half) {
  return FP8 ? dt * 16 + 2 * r + half : dt * 16 + r + 8 * half;
}

template <int KV, int D, int NT>
__global__ void __launch_bounds__(kThreads) decode_kernel(const Params p) {
  using C = Cfg<KV, D, NT>;
  constexpr int MT = C::kKeys / 16, KS = D / 16, DT = D / 16, S = C::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = lane >> 2, pair = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * C::kRing;
  float* sm_m = reinterpret_cast<float*>(smem + kWarps * C::kRing);
  float* sm_l = sm_m + kWarps * NT * 8;
  uint32_t* live = reinterpret_cast<uint32_t*>(sm_l + kWarps * NT * 8) + warp * S;
  const PagedPool& kv = p.a.kv;
  const int items = kv.heads * p.groups, B = p.a.t.B;

  launch_next();
  // ---- this CTA's run of tiles: a prefix sum over the sequences
  __shared__ long long sums[kWarps];
  __shared__ Place at;
  const int per = (B + kThreads - 1) / kThreads;
  const int b0 = threadIdx.x * per, b1 = min(B, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b)
    mine += (table_length(p.a.t, kv.page_size, b, p.a.status) + C::kTile - 1) / C::kTile;
  long long before = mine;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    const long long x = __shfl_up_sync(0xffffffffu, before, s);
    if (lane >= s) before += x;
  }
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  long long total = 0;
  before -= mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  total *= items;
  // every run up to `runs` has a tile, so an item's parts lie in CTAs next to each other
  const long long runs = min(static_cast<long long>(p.grid), (total + kMinTiles - 1) / kMinTiles);
  const bool idle = blockIdx.x >= runs;
  const long long first = idle ? 0 : total * blockIdx.x / runs, last = idle ? 0 : total * (blockIdx.x + 1) / runs;
  if (first < last && before * items <= first && first < (before + mine) * items) {
    Place x;
    long long skip = first - before * items;
    for (x.b = b0;; ++x.b) {
      x.enter<C>(p);
      if (skip < static_cast<long long>(x.tiles) * items) break;
      skip -= static_cast<long long>(x.tiles) * items;
    }
    x.item = static_cast<int>(skip / x.tiles);
    x.tile = static_cast<int>(skip % x.tiles);
    at = x;
  }
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < B; b += p.grid) {
    if (table_length(p.a.t, kv.page_size, b, p.a.status) > 0) continue;
    for (int i = threadIdx.x; i < p.a.Hq * D; i += kThreads)
      p.a.out[b * p.a.o_seq + (i / D) * p.a.o_head + i % D] = 0;
    for (int i = threadIdx.x; i < p.a.Hq; i += kThreads) write_lse(p, b, i, 0.f, 0.f);
  }
  __syncthreads();
  Cut cut{-1, 0, -1, 0};
  if (first == last) {
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = cut;
    return;
  }
  Place load = at, here = at;
  int to_load = static_cast<int>(last - first), left = to_load;

  // ---- loads: lane's key of the warp's slice, its page id one step ahead
  const int my_key = lane % C::kKeys, my_col = lane % C::kChunks;
  const uint64_t policy = evict_first(), keep = evict_last();
  const uint8_t* k_col = kv.k + my_col * 16;
  const uint8_t* v_col = kv.v + my_col * 16;
  int page = 0;
  const auto fetch_page = [&] {
    const int key = load.tile * C::kTile + warp * C::kKeys + my_key;
    page = -1;
    if (to_load > 0 && key < load.n) {
      const int i = p.shift >= 0 ? key >> p.shift : key / kv.page_size;
      page = __ldg(p.a.t.table + load.b * p.a.t.stride + i);
    }
  };
  const auto issue = [&](int stage) {
    if (to_load > 0) {
      const int key = load.tile * C::kTile + warp * C::kKeys + my_key;
      const int head = load.item / p.groups;
      const uint32_t base = ring + stage * C::kStage;
      bool ok = key < load.n;
      if (ok && static_cast<unsigned>(page) >= static_cast<unsigned>(kv.num_pages)) {
        atomicCAS(p.a.status, 0, kStatusBadPage);
        ok = false;
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) live[stage] = mask;
      uint32_t off = 0;
      if (ok) {
        const uint32_t slot = p.shift >= 0 ? key & (kv.page_size - 1) : key % kv.page_size;
        off = page * p.u_page + head * p.u_head + slot * p.u_slot;
        if constexpr (C::kFp8) {
          const int64_t i = (static_cast<int64_t>(page) * kv.heads + head) * kv.page_size + slot;
          if (lane < C::kKeys) {
            cp_async4(base + 2 * C::kRowsBytes + lane * 4, kv.ks + i, true);
            cp_async4(base + 2 * C::kRowsBytes + (C::kKeys + lane) * 4, kv.vs + i, true);
          }
        }
      } else if constexpr (C::kFp8) {
        if (lane < C::kKeys) {
          cp_async4(base + 2 * C::kRowsBytes + lane * 4, kv.ks, false);
          cp_async4(base + 2 * C::kRowsBytes + (C::kKeys + lane) * 4, kv.vs, false);
        }
      }
      if (key - my_key < load.n) {  // some of the slice is in the sequence: the rest of it is zeroed
#pragma unroll
        for (int i = 0; i < C::kKeys * C::kChunks / 32; ++i) {
          const int r = i * (32 / C::kChunks) + lane / C::kChunks;
          const uint64_t o = static_cast<uint64_t>(__shfl_sync(0xffffffffu, off, r)) * p.unit;
          const bool read = (mask >> r) & 1;
          constexpr int kRsh = C::kRow >= 128 ? 0 : C::kRow == 64 ? 1 : 2;
          constexpr int kMask = C::kChunks >= 8 ? 7 : C::kChunks - 1;
          const uint32_t dst = base + r * C::kRow + ((my_col ^ ((r >> kRsh) & kMask)) << 4);
          cp_async16(dst, k_col + o, read, policy);
          cp_async16(dst + C::kRowsBytes, v_col + o, read, policy);
        }
      }
      --to_load;
      if (to_load > 0) load.next<C>(p);
      fetch_page();
    }
    cp_commit();
  };
  fetch_page();
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(s);
  int stage = 0;

  bool first_segment = true;
  while (left > 0) {
    const int b = here.b, head = here.item / p.groups, g0 = here.item % p.groups * NT * 8;
    const int cols = min(NT * 8, p.G - g0), hq0 = head * p.G + g0;
    const int seg = min(left, here.tiles - here.tile);
    const bool begins = here.tile == 0, ends = here.tile + seg == here.tiles;

    // ---- queries as B operands: column lane / 4, rows 2 (lane % 4) + {0, 1, 8, 9}
    // (e4m3: 4 (lane % 4) + {0..3}, the order in which its K rows come)
    uint32_t q[KS][NT][2];
    float factor[NT][2];  // of the score columns 2 (lane % 4) + {0, 1}
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + row;
      const uint16_t* src = p.a.q + b * p.a.q_seq + (hq0 + min(col, cols - 1)) * p.a.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (C::kFp8) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + ks * 16 + pair * 4));
          q[ks][nt][0] = col < cols ? w.x : 0;
          q[ks][nt][1] = col < cols ? w.y : 0;
        } else {
          const uint32_t x = __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + pair * 2));
          const uint32_t y = __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + pair * 2 + 8));
          q[ks][nt][0] = col < cols ? x : 0;
          q[ks][nt][1] = col < cols ? y : 0;
        }
      }
      if constexpr (C::kFp8) {
        // fp16 queries: times the power of two that brings the row's maximum to [2^13, 2^14)
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            top = fmaxf(top, fmaxf(fabsf(value16(q[ks][nt][i] & 0xffffu, p.a.q_f16)),
                                   fabsf(value16(q[ks][nt][i] >> 16, p.a.q_f16))));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;  // floor(log2 top)
        e = top > 0.f && top < INFINITY ? max(-100, min(e, 127)) : 13;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(max(1, 127 + e - 13)) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            q[ks][nt][i] = pack16<false>(value16(q[ks][nt][i] & 0xffffu, p.a.q_f16) * up,
                                         value16(q[ks][nt][i] >> 16, p.a.q_f16) * up);
        factor[nt][0] = __shfl_sync(0xffffffffu, down, pair * 8) * p.a.scale_log2;
        factor[nt][1] = __shfl_sync(0xffffffffu, down, pair * 8 + 4) * p.a.scale_log2;
      } else {
        factor[nt][0] = factor[nt][1] = p.a.scale_log2;
      }
    }

    float m[NT][2], l[NT][2], o[DT][NT][4];
    float winv[NT][2];  // e4m3: the power of two by which weights with their V scales enter fp16
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      winv[nt][0] = winv[nt][1] = __uint_as_float(kWeightMost << 23);
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][nt][i] = 0.f;
    }

    for (int step = 0; step < seg; ++step) {
      cp_wait<S - 2>();
      __syncwarp();
      const int key0 = here.tile * C::kTile + warp * C::kKeys;
      const uint32_t mask = live[stage];
      const uint32_t kb = ring + stage * C::kStage, vb = kb + C::kRowsBytes;
      issue(stage == 0 ? S - 1 : stage - 1);
      if (key0 < here.n) {
        constexpr int kRsh = C::kRow >= 128 ? 0 : C::kRow == 64 ? 1 : 2;
        constexpr int kMask = C::kChunks >= 8 ? 7 : C::kChunks - 1;
        const auto chunk = [&](uint32_t base, int r, int col) {
          return base + r * C::kRow + ((col ^ ((r >> kRsh) & kMask)) << 4);
        };
        uint8_t* rows = smem + warp * C::kRing + stage * C::kStage;
        const float* scales = reinterpret_cast<const float*>(rows + 2 * C::kRowsBytes);
        if constexpr (C::kFp8) {
          // a row whose scale is 0 is zeros, whatever its bytes (0 times a NaN byte is not)
          const bool no_k = scales[my_key] == 0.f, no_v = scales[C::kKeys + my_key] == 0.f;
          if (__any_sync(0xffffffffu, (no_k || no_v) && ((mask >> my_key) & 1))) {
            const uint32_t k0 = __ballot_sync(0xffffffffu, no_k), v0 = __ballot_sync(0xffffffffu, no_v);
#pragma unroll 1
            for (int r = 0; r < C::kKeys; ++r) {
              uint4* dst = reinterpret_cast<uint4*>(rows + r * C::kRow) + lane;
              if (((k0 >> r) & 1) && lane < C::kChunks) *dst = make_uint4(0, 0, 0, 0);
              if (((v0 >> r) & 1) && lane < C::kChunks) dst[C::kRowsBytes / 16] = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
          }
        }
        // ---- S^T = K Q^T
        float x[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[mt][nt][i] = 0.f;
        const int lr = (lane & 7) + (lane & 8), lc = lane >> 4;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if constexpr (C::kFp8) {
#pragma unroll
            for (int k2 = 0; k2 < KS / 2; ++k2) {
              uint32_t w[4];
              ldsm4(w, chunk(kb, mt * 16 + lr, 2 * k2 + lc));
              const uint32_t a0[4] = {widen_lo(w[0]), widen_lo(w[1]), widen_hi(w[0]), widen_hi(w[1])};
              const uint32_t a1[4] = {widen_lo(w[2]), widen_lo(w[3]), widen_hi(w[2]), widen_hi(w[3])};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(x[mt][nt], a0, q[2 * k2][nt][0], q[2 * k2][nt][1]);
                mma16816<false>(x[mt][nt], a1, q[2 * k2 + 1][nt][0], q[2 * k2 + 1][nt][1]);
              }
            }
          } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              uint32_t w[4];
              ldsm4(w, chunk(kb, mt * 16 + lr, 2 * ks + lc));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<C::kBf16>(x[mt][nt], w, q[ks][nt][0], q[ks][nt][1]);
            }
          }
        }
        // ---- scores in log2 units; what is not live is -inf
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = mt * 16 + i * 8 + row;
            const bool ok = (mask >> r) & 1;
            float ks = 1.f;
            if constexpr (C::kFp8) ks = scales[r];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float& y = x[mt][nt][2 * i + j];
                if constexpr (C::kFp8) y *= ks;
                y = ok ? y * factor[nt][j] : -INFINITY;
                top[nt][j] = fmaxf(top[nt][j], y);
              }
          }
        if (p.scores) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int col = nt * 8 + pair * 2 + j;
              if (col < cols) {
                float* dst = p.scores + (static_cast<int64_t>(b) * p.a.Hq + hq0 + col) * p.score_pitch + key0;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const int r = mt * 16 + i * 8 + row;
                    if (key0 + r < here.n) store_kept(dst + r, x[mt][nt][2 * i + j], keep);
                  }
              }
            }
        }
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) raise |= top[nt][j] > m[nt][j] + C::kAbove;
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float t = top[nt][j];
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
              t -= C::kBelow;
              if constexpr (C::kFp8) t = ceilf(t);  // whole, so that winv can follow
              t = fmaxf(t, m[nt][j]);
              float f = t == m[nt][j] ? 1.f : ex2(m[nt][j] - t);
              l[nt][j] *= f;
              if constexpr (C::kFp8) {
                // every product falls by 2^(t - m): winv takes that up, and the sums what it cannot
                const uint32_t to = (__float_as_uint(winv[nt][j]) >> 23) +
                                    (t == m[nt][j] ? 0 : static_cast<uint32_t>(fminf(t - m[nt][j], 400.f)));
                const uint32_t left_over = to - min(to, kWeightMost);
                winv[nt][j] = __uint_as_float(min(to, kWeightMost) << 23);
                f = left_over < 127 ? __uint_as_float((127 - left_over) << 23) : 0.f;
              }
              m[nt][j] = t;
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                o[dt][nt][j] *= f;
                o[dt][nt][2 + j] *= f;
              }
            }
        }
        if constexpr (C::kFp8) {
          // weights with their rows' V scales, and their maximum in each column
          float top_w[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) top_w[nt][0] = top_w[nt][1] = 0.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float vs = scales[C::kKeys + mt * 16 + i * 8 + row];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  float& y = x[mt][nt][2 * i + j];
                  const float e = ex2(y - finite_or_zero(m[nt][j]));
                  l[nt][j] += e;
                  y = e * vs;
                  top_w[nt][j] = fmaxf(top_w[nt][j], fabsf(y));
                }
            }
          bool over = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) over |= top_w[nt][j] * winv[nt][j] > kWeightTop;
          if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float t = top_w[nt][j];
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                if (!(t * winv[nt][j] > kWeightTop)) continue;
                // t into [2^10, 2^11); what was summed follows
                const uint32_t to = min(kWeightMost, 127 + 10 + 127 - (__float_as_uint(t) >> 23));
                const int down = static_cast<int>(to - (__float_as_uint(winv[nt][j]) >> 23));
                const float f = down > -127 ? __uint_as_float(static_cast<uint32_t>(127 + down) << 23) : 0.f;
                winv[nt][j] = __uint_as_float(to << 23);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                  o[dt][nt][j] *= f;
                  o[dt][nt][2 + j] *= f;
                }
              }
          }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t pb[NT][2], pl[NT][2];  // rounded softmax weights; what the rounding left, rounded
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float e0, e1;
              if constexpr (C::kFp8) {
                e0 = x[mt][nt][2 * i] * winv[nt][0];
                e1 = x[mt][nt][2 * i + 1] * winv[nt][1];
              } else {
                e0 = ex2(x[mt][nt][2 * i] - finite_or_zero(m[nt][0]));
                e1 = ex2(x[mt][nt][2 * i + 1] - finite_or_zero(m[nt][1]));
                l[nt][0] += e0;
                l[nt][1] += e1;
              }
              const uint32_t high = pack16<C::kBf16>(e0, e1);
              pb[nt][i] = transpose8(high);
              if constexpr (!C::kFp8)
                pl[nt][i] = transpose8(pack16<C::kBf16>(e0 - value16(high & 0xffffu, !C::kBf16),
                                                        e1 - value16(high >> 16, !C::kBf16)));
            }
          if constexpr (C::kFp8) {
#pragma unroll
            for (int d2 = 0; d2 < DT / 2; ++d2) {
              uint32_t w[4];
              ldsm4t(w, chunk(vb, mt * 16 + lr, 2 * d2 + lc));
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = __byte_perm(w[i], 0, 0x3120);
              const uint32_t a0[4] = {widen_lo(w[0]), widen_hi(w[0]), widen_lo(w[1]), widen_hi(w[1])};
              const uint32_t a1[4] = {widen_lo(w[2]), widen_hi(w[2]), widen_lo(w[3]), widen_hi(w[3])};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(o[2 * d2][nt], a0, pb[nt][0], pb[nt][1]);
                mma16816<false>(o[2 * d2 + 1][nt], a1, pb[nt][0], pb[nt][1]);
              }
            }
          } else {
            const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              uint32_t w[4];
              ldsm4t(w, chunk(vb, mt * 16 + vr, 2 * dt + vc));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<C::kBf16>(o[dt][nt], w, pb[nt][0], pb[nt][1]);
                mma16816<C::kBf16>(o[dt][nt], w, pl[nt][0], pl[nt][1]);
              }
            }
          }
        }
      }
      stage = stage == S - 1 ? 0 : stage + 1;
      --left;
      if (left > 0) here.next<C>(p);
    }

    // ---- the four warps' parts of this segment joined (in warp 0)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = l[nt][j];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        l[nt][j] = t;
        if (row == 0) {
          const int i = warp * NT * 8 + nt * 8 + pair * 2 + j;
          sm_m[i] = m[nt][j];
          sm_l[i] = t;
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = nt * 8 + pair * 2 + j;
        float top = sm_m[i], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_m[w * NT * 8 + i]);
        const float ref = finite_or_zero(top);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += sm_l[w * NT * 8 + i] * ex2(sm_m[w * NT * 8 + i] - ref);
        float f = ex2(m[nt][j] - ref);
        if constexpr (C::kFp8) f *= __uint_as_float((254u << 23) - __float_as_uint(winv[nt][j]));
        m[nt][j] = top;
        l[nt][j] = sum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          o[dt][nt][j] *= f;
          o[dt][nt][2 + j] *= f;
        }
      }
    // through the stage that each warp read last: its next load goes there, after the barriers
    const int idle_stage = stage == 0 ? S - 1 : stage - 1;
    const auto buffer = [&](int w) {
      return reinterpret_cast<float4*>(smem + w * C::kRing + idle_stage * C::kStage) + lane;
    };
    const auto put = [&] {
      float4* dst = buffer(warp);
#pragma unroll
      for (int i = 0; i < C::kFrags; ++i) {
        const float(&c)[4] = o[i / NT][i % NT];
        dst[i * 32] = make_float4(c[0], c[1], c[2], c[3]);
      }
    };
    const auto take = [&](int w) {
      const float4* src = buffer(w);
#pragma unroll
      for (int i = 0; i < C::kFrags; ++i) {
        float(&c)[4] = o[i / NT][i % NT];
        const float4 y = src[i * 32];
        c[0] += y.x;
        c[1] += y.y;
        c[2] += y.z;
        c[3] += y.w;
      }
    };
    if (warp >= 2) put();
    __syncthreads();
    if (warp < 2) take(warp + 2);
    if (warp == 1) put();
    __syncthreads();
    if (warp == 0) take(1);
    __syncthreads();
    if (warp == 0) {
      if (begins && ends) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = nt * 8 + pair * 2 + j;
            if (col >= cols) continue;
            const float inv = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];
            uint16_t* dst = p.a.out + b * p.a.o_seq + (hq0 + col) * p.a.o_head;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int half = 0; half < 2; ++half)
                dst[dim_of<C::kFp8>(dt, row, half)] = round16(o[dt][nt][2 * half + j] * inv, p.a.q_f16);
            if (row == 0) write_lse(p, b, hq0 + col, m[nt][j], l[nt][j]);
          }
      } else {
        const int slot = blockIdx.x * 2 + (first_segment ? 0 : 1);
#pragma unroll
        for (int i = 0; i < C::kFrags; ++i) {
          const float(&c)[4] = o[i / NT][i % NT];
          p.part_o[(static_cast<int64_t>(slot) * C::kFrags + i) * 32 + lane] = make_float4(c[0], c[1], c[2], c[3]);
        }
        if (row == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float* ml = p.part_ml + slot * 2 * NT * 8 + nt * 8 + pair * 2 + j;
              ml[0] = m[nt][j];
              ml[NT * 8] = l[nt][j];
            }
        }
      }
    }
    if (!(begins && ends)) {
      if (begins) {
        cut.begun = b * items + head * p.groups + g0 / (NT * 8);
        cut.begun_slot = first_segment ? 0 : 1;
      } else {
        cut.continued = b * items + head * p.groups + g0 / (NT * 8);
      }
    }
    first_segment = false;
  }
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = cut;
}

// Joins the partials of the item that CTA blockIdx.x of the main kernel began
// and others continued: CTA blockIdx.x + 1, + 2, ... in order.
template <int KV, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const Params p) {
  using C = Cfg<KV, D, NT>;
  constexpr int kE = C::kFrags * 32;  // float4 elements of a partial
  constexpr int kTeams = kJoinThreads > kE ? kJoinThreads / kE : 1;
  extern __shared__ float factors[];  // (parts, NT * 8)
  __shared__ float4 sums[kJoinThreads];
  __shared__ float sm_inv[NT * 8];
  __shared__ int count;
  launch_next();
  wait_previous();
  const Cut cut = p.cuts[blockIdx.x];
  if (cut.begun < 0) return;
  const int item = cut.begun, first_slot = blockIdx.x * 2 + cut.begun_slot;
  if (threadIdx.x == 0) count = p.grid - blockIdx.x;
  __syncthreads();
  for (int c = blockIdx.x + 1 + threadIdx.x; c < p.grid; c += kJoinThreads)
    if (p.cuts[c].continued != item) atomicMin(&count, c - static_cast<int>(blockIdx.x));
  __syncthreads();
  const int parts = count;
  const auto slot_of = [&](int i) { return i == 0 ? first_slot : static_cast<int>((blockIdx.x + i) * 2); };
  const int items = p.a.kv.heads * p.groups;
  const int b = item / items, head = item % items / p.groups, g0 = item % p.groups * NT * 8;
  const int cols = min(NT * 8, p.G - g0), hq0 = head * p.G + g0;
  // one warp per column: the maximum, the sum, every partial's factor
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < NT * 8) {
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_ml[slot_of(i) * 2 * NT * 8 + warp]);
#pragma unroll
    for (int s = 16; s > 0; s /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    const float ref = finite_or_zero(m);
    for (int i = lane; i < parts; i += 32) {
      const float* ml = p.part_ml + slot_of(i) * 2 * NT * 8 + warp;
      const float f = ex2(ml[0] - ref);
      factors[i * NT * 8 + warp] = f;
      l += ml[NT * 8] * f;
    }
#pragma unroll
    for (int s = 16; s > 0; s /= 2) l += __shfl_xor_sync(0xffffffffu, l, s);
    if (lane == 0) {
      sm_inv[warp] = l == 0.f ? 0.f : 1.f / l;
      if (warp < cols) write_lse(p, b, hq0 + warp, m, l);
    }
  }
  __syncthreads();
  const int team = threadIdx.x / kE;
  for (int e = threadIdx.x % kE; e < kE; e += kJoinThreads) {
    const int ln = e % 32, nt = e / 32 % NT, dt = e / 32 / NT;
    const int c0 = nt * 8 + (ln & 3) * 2;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = team; i < parts; i += kTeams) {
      const float4 y = p.part_o[static_cast<int64_t>(slot_of(i)) * kE + e];
      const float f0 = factors[i * NT * 8 + c0], f1 = factors[i * NT * 8 + c0 + 1];
      s.x += y.x * f0;
      s.y += y.y * f1;
      s.z += y.z * f0;
      s.w += y.w * f1;
    }
    if constexpr (kTeams > 1) {
      sums[threadIdx.x] = s;
      __syncthreads();
      if (team > 0) return;
#pragma unroll
      for (int i = 1; i < kTeams; ++i) {
        const float4 y = sums[threadIdx.x + i * kE];
        s.x += y.x;
        s.y += y.y;
        s.z += y.z;
        s.w += y.w;
      }
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = c0 + (i & 1);
      if (col < cols)
        p.a.out[b * p.a.o_seq + (hq0 + col) * p.a.o_head + dim_of<C::kFp8>(dt, ln >> 2, i >> 1)] =
            round16(v[i] * sm_inv[col], p.a.q_f16);
    }
  }
}

// Every key's weights, summed over the query heads of its KV head in order;
// four keys a thread.
__global__ void __launch_bounds__(256) decode_weights_kernel(const Params p) {
  wait_previous();
  const int h = blockIdx.y, b = blockIdx.z;
  const int n = table_length(p.a.t, p.a.kv.page_size, b, p.a.status);
  const int64_t row = static_cast<int64_t>(b) * p.a.Hq + h * p.G;
  const float* scores = p.scores + row * p.score_pitch;
  const float* lse2 = p.lse2 + row;
  float* dst = p.a.weights.w + b * p.a.weights.s_seq + h * p.a.weights.s_head;
  const bool whole = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
  const uint64_t policy = evict_first();
  for (int j = (blockIdx.x * 256 + threadIdx.x) * 4; j < n; j += gridDim.x * 1024) {
    float w[4] = {0.f, 0.f, 0.f, 0.f}, old[4];
    const bool four = whole && j + 4 <= n;
    if (four) {
      const float4 y = *reinterpret_cast<const float4*>(dst + j);
      old[0] = y.x;
      old[1] = y.y;
      old[2] = y.z;
      old[3] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = j + i < n ? dst[j + i] : 0.f;
    }
#pragma unroll 4
    for (int g = 0; g < p.G; ++g) {
      const float y = finite_or_zero(__ldcg(lse2 + g));
      // the rows of scores are whole 16-byte vectors; what lies past n is not used
      const float* src = scores + static_cast<int64_t>(g) * p.score_pitch + j;
      const float4 x = load_once(src, policy);
      if (threadIdx.x % 8 == 0) give_back_line(src);  // eight threads read a line
      w[0] += ex2(x.x - y);
      w[1] += ex2(x.y - y);
      w[2] += ex2(x.z - y);
      w[3] += ex2(x.w - y);
    }
    if (four) {
      *reinterpret_cast<float4*>(dst + j) = make_float4(old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < n) dst[j + i] = old[i] + w[i];
    }
  }
}

// Column blocks of 8 query heads that a group of G heads is given: two at most
// (a group of more than 16 heads takes several passes over its keys).
int column_blocks(int G) { return G > 8 ? 2 : 1; }

struct Workspace {
  size_t part_ml, cuts, lse2, scores, total;
  int pitch;
  Workspace(const PagedPool& kv, int B, int Hq, int table_pages, bool weights) {
    const size_t heads = static_cast<size_t>(B) * Hq;
    const int nt = column_blocks(Hq / kv.heads);
    const auto next = [this](size_t bytes) {
      const size_t at = total;
      total += (bytes + 127) / 128 * 128;
      return at;
    };
    total = 0;
    pitch = (table_pages * kv.page_size + 31) / 32 * 32;
    next(static_cast<size_t>(kMaxCtas) * 2 * (kv.D / 16) * nt * 512);  // part_o, at 0
    part_ml = next(static_cast<size_t>(kMaxCtas) * 2 * 2 * nt * 8 * 4);
    cuts = next(kMaxCtas * sizeof(Cut));
    lse2 = next(weights ? heads * 4 : 0);
    scores = next(weights ? heads * pitch * 4 : 0);
  }
};

template <int KV, int D, int NT>
cudaError_t launch(Params p, cudaStream_t st) {
  using C = Cfg<KV, D, NT>;
  static std::atomic<int> known[kMaxDevices];  // CTAs an SM holds, once this device is set up
  const int dev = current_device();
  int per_sm = known[dev].load(std::memory_order_relaxed);
  if (per_sm == 0) {
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<KV, D, NT>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, decode_kernel<KV, D, NT>, kThreads, C::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(decode_join_kernel<KV, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMaxCtas * NT * 8 * 4);
    if (e != cudaSuccess) return e;
    if (per_sm < 1) per_sm = 1;
    known[dev].store(per_sm, std::memory_order_relaxed);
  }
  p.grid = sm_count(dev) * per_sm < kMaxCtas ? sm_count(dev) * per_sm : kMaxCtas;
  if (p.grid <= 0) return cudaErrorInvalidDevice;
  decode_kernel<KV, D, NT><<<p.grid, kThreads, C::kSmem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_after(decode_join_kernel<KV, D, NT>, dim3(p.grid), kJoinThreads,
                      static_cast<size_t>(p.grid) * NT * 8 * 4, st, p);
}

template <int KV, int D>
cudaError_t launch_nt(const Params& p, int nt, cudaStream_t st) {
  return nt == 1 ? launch<KV, D, 1>(p, st) : launch<KV, D, 2>(p, st);
}

template <int KV>
cudaError_t launch_d(const Params& p, int nt, cudaStream_t st) {
  switch (p.a.kv.D) {
    case 32: return launch_nt<KV, 32>(p, nt, st);
    case 64: return launch_nt<KV, 64>(p, nt, st);
    case 128: return launch_nt<KV, 128>(p, nt, st);
    case 256: return launch_nt<KV, 256>(p, nt, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

size_t paged_decode_workspace(const PagedPool& kv, int B, int Hq, int table_pages, bool weights) {
  return Workspace(kv, B, Hq, table_pages, weights).total;
}

cudaError_t launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t st) {
  const bool weights = a.weights.w != nullptr;
  const Workspace ws(a.kv, a.t.B, a.Hq, a.t.pages, weights);
  char* base = static_cast<char*>(a.workspace);
  Params p{};
  p.a = a;
  p.G = a.Hq / a.kv.heads;
  const int nt = column_blocks(p.G);
  p.groups = (p.G + nt * 8 - 1) / (nt * 8);
  p.shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a.kv.page_size == 1 << s) p.shift = s;
  const int size = a.kv.dtype == kKvE4m3 ? 1 : 2;
  const int64_t unit = pool_unit(a.kv);
  if (unit == 0) return cudaErrorInvalidValue;
  p.u_page = static_cast<uint32_t>(a.kv.s_page * size / unit);
  p.u_head = static_cast<uint32_t>(a.kv.s_head * size / unit);
  p.u_slot = static_cast<uint32_t>(a.kv.s_slot * size / unit);
  p.unit = static_cast<uint32_t>(unit);
  p.score_pitch = ws.pitch;
  p.part_o = reinterpret_cast<float4*>(base);
  p.part_ml = reinterpret_cast<float*>(base + ws.part_ml);
  p.cuts = reinterpret_cast<Cut*>(base + ws.cuts);
  p.lse2 = weights ? reinterpret_cast<float*>(base + ws.lse2) : nullptr;
  p.scores = weights ? reinterpret_cast<float*>(base + ws.scores) : nullptr;
  cudaError_t e = cudaErrorInvalidValue;
  switch (a.kv.dtype) {
    case kKvBf16: e = launch_d<kKvBf16>(p, nt, st); break;
    case kKvF16: e = launch_d<kKvF16>(p, nt, st); break;
    case kKvE4m3: e = launch_d<kKvE4m3>(p, nt, st); break;
  }
  const int cap = a.t.pages * a.kv.page_size;
  if (e != cudaSuccess || !weights || cap == 0) return e;
  // enough CTAs for the SMs, at most one per 1024 positions
  const int rows = a.kv.heads * a.t.B, most = (cap + 1023) / 1024;
  const int want = (16 * sm_count(current_device()) + rows - 1) / rows;
  const int ctas = want < most ? want : most;
  if (static_cast<int64_t>(ctas) * 1024 > 0x7FFFFFFF - kMaxPositions) return cudaErrorInvalidValue;
  return launch_after(decode_weights_kernel, dim3(ctas, a.kv.heads, a.t.B), 256, 0, st, p);
}

}  // namespace rp
