// Log probability of given tokens, entropy, and the top alternatives of every
// row of logits.
//
// With m = max_v x_v, l = sum_v e^(x_v - m) and lse = m + log l:
//   logprob = (x_token - m) - log l        (not x_token - lse, which cancels
//                                           where |m| is large)
//   entropy = log l - (sum_v e^(x_v - m) (x_v - m)) / l
//   top     = the `top` largest x_v, ties to the lowest index.
// A row whose every logit is -inf has entropy 0 and log probabilities -inf;
// a NaN or +inf in a row makes its sums NaN.
//
// One pass over the logits, bound by HBM (and, for 16-bit logits, not far from
// the exp rate: one MUFU operation an element).  A thread keeps a reference
// value, moved only when a value exceeds it by 6.9 (2^10 in e^x), and sums e^(x - ref) and
// its product with x - ref in fp32; the maximum is not needed exactly.
// Alternatives cost the pass nothing but a running maximum: each thread leaves
// the maxima of its segments (32 to a few hundred values) in shared memory.
// Afterwards the k-th largest of 32 to 128 group maxima is a lower bound of the
// k-th largest value, and the few segments that reach it are read again (from
// L2).  A thread brings its own vectors in through a ring of its own (16-byte
// cp.async, two batches ahead), which needs no barrier and no registers; a CTA
// that has another row to do starts it there before it selects the last one's
// alternatives.
// Few rows are split over a cluster of CTAs, joined through distributed shared
// memory: one launch, no workspace.  Measured (replayed in a graph): 4095 x 100003
// fp32, 20 alternatives 304 us (5.4 TB/s; none: 262), 512 x 32000 bf16, 8
// alternatives 14.8 us, one row of 32000 over eight CTAs 9.3 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "internal.h"
#include "paged.h"
#include "ptx.cuh"

namespace rp {
namespace {

namespace cg = cooperative_groups;

constexpr int kT = 128;              // threads of a CTA
constexpr int kU = 4;                // 16-byte vectors of a thread's batch
constexpr int kStages = 3;           // batches of a thread in shared memory
constexpr int kRing = kStages * kU * kT * 16;  // bytes: 24 KB, five CTAs an SM
constexpr int kResident = 5;
constexpr int kSegments = 16;        // segments of a thread, at most
constexpr int kCandidates = 512;     // values kept for the selection
constexpr int kLook = 12;            // values of a thread in flight when segments are read again
constexpr int kManyHits = 256;       // more segments than this reach a bound only by ties
constexpr int kMaxCluster = 8;
static_assert(kMaxTop <= kT && kMaxCluster * kMaxTop <= kCandidates, "");
static_assert(kSegments * kT * 2 <= kMaxCluster * kMaxTop * 8, "the list of segments fits the merged keys");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kHeadroom = 6.9f;    // the reference may lie 2^10 below a value

// Order of values as one integer: NaN above +inf, -0 equal to 0; and back.
__device__ __forceinline__ uint32_t value_key(float x) {
  uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
// Alternatives in order: larger value first, then lower index.
__device__ __forceinline__ uint64_t rank_key(float x, int i) {
  return (static_cast<uint64_t>(value_key(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Element types: DT is an rp_dtype.
template <int DT>
struct Type {
  static constexpr int kVec = DT == 2 ? 4 : 8;  // elements of a 16-byte vector
  static constexpr int kSize = 16 / kVec;
  static constexpr uint32_t kNegInf = DT == 2 ? 0xFF800000u : DT == 1 ? 0xFC00FC00u : 0xFF80FF80u;
  __device__ static __forceinline__ float at(const void* p, int64_t i) {
    if constexpr (DT == 2) return __ldg(static_cast<const float*>(p) + i);
    const uint16_t u = __ldg(static_cast<const uint16_t*>(p) + i);
    return DT == 1 ? __half2float(__ushort_as_half(u)) : __uint_as_float(static_cast<uint32_t>(u) << 16);
  }
  // The two values of word w of a 16-bit vector.
  __device__ static __forceinline__ float2 pair(uint32_t w) {
    if constexpr (DT == 1) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  // Larger of two words' values (element-wise when 16-bit); NaN wins.
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t y;
    if constexpr (DT == 0) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else if constexpr (DT == 1) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else y = __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    return y;
  }
  __device__ static __forceinline__ float value(uint32_t w) {
    if constexpr (DT == 2) return __uint_as_float(w);
    const float2 v = pair(w);
    return max_nan(v.x, v.y);
  }
};

// A vector with elements missing, -inf there: elements e0, e0 + 1, ... of a row
// of V.  (Not inlined: the pass has it four times, for two vectors a row.)
template <int DT>
__device__ __noinline__ uint4 edge_vector(const char* row, int e0, int V) {
  using E = Type<DT>;
  uint32_t w[4] = {E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
#pragma unroll
  for (int i = 0; i < E::kVec; ++i) {
    const int e = e0 + i;
    if (e < 0 || e >= V) continue;
    if constexpr (DT == 2) {
      w[i] = __ldg(reinterpret_cast<const uint32_t*>(row) + e);
    } else {
      const uint32_t u = __ldg(reinterpret_cast<const uint16_t*>(row) + e);
      w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | (u << 16) : (w[i / 2] & 0xffff0000u) | u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums over a set of values relative to ref: l = sum e^(x - ref), s = sum
// e^(x - ref) log2(e) (x - ref).
struct Sums {
  float ref, l, s;
  // The same sums relative to `to` (not below ref's rounding of them).
  __device__ __forceinline__ void move(float to) {
    if (l == 0.f) {
      s = 0.f;
    } else {
      const float y = ((ref == -INFINITY ? 0.f : ref) - to) * kLog2e, f = ex2(y);
      s = f * (s + l * fmaxf(y, -1000.f));
      l *= f;
    }
    ref = to;
  }
};
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  const float to = fmaxf(a.ref, b.ref), ref = to == -INFINITY ? 0.f : to;
  a.move(ref);
  b.move(ref);
  return Sums{to, a.l + b.l, a.s + b.s};
}

struct Shared {
  Sums warp_sums[kT / 32];
  Sums sums;                        // of this CTA
  uint4 groups[kT / 4];             // keys of the groups' maxima
  uint64_t best[kMaxTop];           // this CTA's alternatives
  uint64_t merged[kMaxCluster * kMaxTop];
  int votes[kT / 32];
  int hits;
  int count, picked;
  uint32_t bound;
};

// The `k` largest of n different keys, in order, to out[0..k) (n >= k), by
// counting the larger ones of each.  All threads of the CTA.
__device__ __forceinline__ void select_top(const uint64_t* keys, int n, int k, uint64_t* out) {
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += kT) {
    const uint64_t key = keys[j];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += keys[i] > key;
    if (rank < k) out[rank] = key;
  }
  __syncthreads();
}

// A CTA's part of a row, as vectors that start at 16-byte boundaries: vector v
// holds elements v * kVec - shift + i, of which the first and last may lack
// some; [inner0, inner1) are whole, [v0, v1) the part's.
struct Part {
  const char* row;
  const uint4* base;
  int shift, v0, v1, inner0, inner1;
};

// One row per cluster at a time; the CTAs of a cluster take equal parts of it.
template <int DT>
__global__ void __launch_bounds__(kT, kResident) score_kernel(const ScoreArgs a, int per_segment) {
  using E = Type<DT>;
  constexpr int kVec = E::kVec;
  extern __shared__ __align__(16) uint8_t dynamic[];  // the ring; with alternatives, candidates and segment maxima
  __shared__ Shared sh;
  uint64_t* cand = reinterpret_cast<uint64_t*>(dynamic + kRing);
  float* segs = reinterpret_cast<float*>(cand + kCandidates);
  uint16_t* hit_list = reinterpret_cast<uint16_t*>(sh.merged);  // segments that reach the bound
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int V = a.vocab, top = a.top, rows_at_once = gridDim.x / parts;
  const auto part_of = [&](int r) {
    Part p;
    p.row = static_cast<const char*>(a.logits) + r * a.stride * E::kSize;
    p.shift = static_cast<int>(reinterpret_cast<uintptr_t>(p.row) & 15) / E::kSize;
    p.base = reinterpret_cast<const uint4*>(p.row - p.shift * E::kSize);
    const int vectors = (V + p.shift + kVec - 1) / kVec;
    p.v0 = static_cast<int>(static_cast<int64_t>(vectors) * part / parts);
    p.v1 = static_cast<int>(static_cast<int64_t>(vectors) * (part + 1) / parts);
    p.inner0 = p.shift ? 1 : 0;
    p.inner1 = (V + p.shift) / kVec;
    return p;
  };
  uint4* ring = reinterpret_cast<uint4*>(dynamic) + t;  // (stage, vector) at ring[(stage * kU + u) * kT]
  const auto fill = [&](const Part& p, int stage, int v) {  // the batch that starts with vector v
#pragma unroll
    for (int u = 0; u < kU && v < p.v1; ++u) {
      uint4* dst = ring + (stage * kU + u) * kT;
      const int w = v + u * kT;
      if (w >= p.inner0 && w < min(p.inner1, p.v1))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(p.base + w) : "memory");
      else
        *dst = w < p.v1 ? edge_vector<DT>(p.row, w * kVec - p.shift, V)
                        : make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the first batches of a part, to be read from `stage` on
  const auto start = [&](const Part& p, int stage) {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fill(p, (stage + i) % kStages, p.v0 + t + i * kU * kT);
  };
  int stage = 0;
  Part next = part_of(blockIdx.x / parts);
  start(next, stage);
  for (int r = blockIdx.x / parts; r < a.rows; r += rows_at_once) {
    const Part p = next;

    // thread 0 has the token's logit long before its sums
    int64_t token = -1;
    float token_logit = 0.f;
    if (part == 0 && t == 0) {
      token = a.tokens[r];
      if (token >= 0 && token < V) token_logit = E::at(p.row, token);
    }

    // ---- the pass
    Sums mine{-INFINITY, 0.f, 0.f};
    float seg = -INFINITY, best = -INFINITY;
    int in_seg = 0, n_seg = 0;
    uint64_t l2 = 0, s2 = 0;
    for (int v = p.v0 + t; v < p.v1; v += kU * kT) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      uint4 x[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) x[u] = ring[(stage * kU + u) * kT];
      fill(p, stage == 0 ? kStages - 1 : stage - 1, v + (kStages - 1) * kU * kT);
      stage = stage == kStages - 1 ? 0 : stage + 1;
      uint32_t m = x[0].x;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        m = E::larger(m, E::larger(x[u].x, x[u].y));
        m = E::larger(m, E::larger(x[u].z, x[u].w));
      }
      const float big = E::value(m);
      if (big > mine.ref + kHeadroom) {
        float x0, x1;
        unpack_f32x2(l2, x0, x1);
        mine.l = x0 + x1;
        unpack_f32x2(s2, x0, x1);
        mine.s = x0 + x1;
        mine.move(big);
        l2 = pack_f32x2(mine.l, 0.f);
        s2 = pack_f32x2(mine.s, 0.f);
      }
      seg = max_nan(seg, big);
      if (top > 0 && ++in_seg == per_segment) {
        segs[n_seg++ * kT + t] = seg;
        best = max_nan(best, seg);
        seg = -INFINITY;
        in_seg = 0;
      }
      const float ref = mine.ref == -INFINITY ? 0.f : mine.ref;
      const uint64_t nref = pack_f32x2(-ref, -ref), scale = pack_f32x2(kLog2e, kLog2e);
      const auto two = [&](float x0, float x1) {
        const uint64_t y = fmul2(fadd2(pack_f32x2(x0, x1), nref), scale);
        float y0, y1;
        unpack_f32x2(y, y0, y1);
        const uint64_t e = pack_f32x2(ex2(y0), ex2(y1));
        l2 = fadd2(l2, e);
        // e is 0 where the clamp acts (-inf logits)
        s2 = ffma2(e, pack_f32x2(fmaxf(y0, -1000.f), fmaxf(y1, -1000.f)), s2);
      };
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
        if constexpr (DT == 2) {
          two(__uint_as_float(w[0]), __uint_as_float(w[1]));
          two(__uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = E::pair(w[i]);
            two(f.x, f.y);
          }
        }
      }
    }
    if (r + rows_at_once < a.rows) {
      next = part_of(r + rows_at_once);
      start(next, stage);
    }
    {
      float x0, x1;
      unpack_f32x2(l2, x0, x1);
      mine.l = x0 + x1;
      unpack_f32x2(s2, x0, x1);
      mine.s = x0 + x1;
    }
    {
      float to = mine.ref;
#pragma unroll
      for (int s = 16; s > 0; s /= 2) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, s));
      mine.move(to == -INFINITY ? 0.f : to);
      mine.ref = to;
#pragma unroll
      for (int s = 16; s > 0; s /= 2) {
        mine.l += __shfl_xor_sync(0xffffffffu, mine.l, s);
        mine.s += __shfl_xor_sync(0xffffffffu, mine.s, s);
      }
    }
    if (lane == 0) sh.warp_sums[warp] = mine;

    // ---- this part's alternatives
    const int have = min(V, p.v1 * kVec - p.shift) - max(0, p.v0 * kVec - p.shift);  // its elements
    const int k = min(top, max(have, 0));
    if (k > 0) {
      if (in_seg > 0) {
        segs[n_seg++ * kT + t] = seg;
        best = max_nan(best, seg);
      }
      // the k-th largest of the maxima of 2 k or more groups of lanes (32, 64 or 128 groups)
      const int lanes = k <= 16 ? kT / 32 : k <= 32 ? kT / 64 : 1;  // of a group
      float g = best;
      for (int s = 1; s < lanes; s *= 2) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, s));
      const uint32_t group_key = value_key(g);
      if (t % lanes == 0) reinterpret_cast<uint32_t*>(sh.groups)[t / lanes] = group_key;
      if (t == 0) {
        sh.count = 0;
        sh.hits = 0;
        sh.bound = 0;
      }
      __syncthreads();
      if (t < kT / lanes) {
        const uint32_t key = reinterpret_cast<const uint32_t*>(sh.groups)[t];
        int above = 0;
#pragma unroll 4
        for (int i = 0; i < kT / lanes / 4; ++i) {
          const uint4 o = sh.groups[i];
          above += (o.x > key || (o.x == key && 4 * i < t)) + (o.y > key || (o.y == key && 4 * i + 1 < t)) +
                   (o.z > key || (o.z == key && 4 * i + 2 < t)) + (o.w > key || (o.w == key && 4 * i + 3 < t));
        }
        if (above == k - 1) sh.bound = key;
      }
      __syncthreads();
      // candidates: every value at or above the bound; `strict`: above it.  The
      // segments that reach it are listed first; then their elements are read again.
      // (Most segments at the bound are most of the row at one value, such as
      // logits masked to -inf: too many without a look.)
      const auto collect = [&](uint32_t bound, bool strict) {
        for (int i = 0; i < n_seg; ++i) {
          const uint32_t sk = value_key(segs[i * kT + t]);
          if (strict ? sk > bound : sk >= bound) hit_list[atomicAdd(&sh.hits, 1)] = static_cast<uint16_t>(i * kT + t);
        }
        __syncthreads();
        const int hits = sh.hits, each = per_segment * kU * kVec;
        if (!strict && hits > kManyHits && have > kCandidates) return kCandidates + 1;
        // (kLook loads of a thread in flight: the row may have left L2)
        for (int i = t; i < hits * each; i += kLook * kT) {
          float y[kLook];
          int at[kLook];
#pragma unroll
          for (int u = 0; u < kLook; ++u) {
            const int q = i + u * kT, hit = hit_list[min(q / each, hits - 1)], j = q % each;
            const int v = p.v0 + hit % kT + (hit / kT * per_segment * kU + j / kVec) * kT;
            at[u] = q < hits * each && v < p.v1 ? v * kVec - p.shift + j % kVec : -1;
            if (at[u] >= V) at[u] = -1;
            y[u] = at[u] >= 0 ? E::at(p.row, at[u]) : 0.f;
          }
#pragma unroll
          for (int u = 0; u < kLook; ++u) {
            const uint32_t key = value_key(y[u]);
            if (at[u] < 0 || (strict ? key <= bound : key < bound)) continue;
            const int to = atomicAdd(&sh.count, 1);
            if (to < kCandidates) cand[to] = rank_key(y[u], at[u]);
          }
        }
        __syncthreads();
        return sh.count;
      };
      uint32_t bound = sh.bound;
      int n = collect(bound, false);
      __syncthreads();
      // Too many: the values above the bound alone.  Are these too many as well,
      // the k-th largest of those at hand is a higher bound.
      while (n > kCandidates) {
        if (t == 0) sh.count = sh.hits = 0;
        __syncthreads();
        n = collect(bound, true);
        __syncthreads();
        if (n > kCandidates) {
          select_top(cand, kCandidates, k, sh.best);
          bound = static_cast<uint32_t>(sh.best[k - 1] >> 32);
          if (t == 0) sh.count = sh.hits = 0;
          __syncthreads();
          n = collect(bound, false);
          __syncthreads();
        } else if (n < k) {
          // the lowest indices among the values equal to the bound
          const int e0 = max(0, p.v0 * kVec - p.shift), e1 = min(V, p.v1 * kVec - p.shift);
          int need = k - n;
          for (int e = e0; e < e1 && need > 0; e += kT) {
            const bool tie = e + t < e1 && value_key(E::at(p.row, e + t)) == bound;
            const uint32_t votes = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) sh.votes[warp] = __popc(votes);
            __syncthreads();
            int before = __popc(votes & ((1u << lane) - 1)), all = 0;
            for (int w = 0; w < kT / 32; ++w) {
              if (w < warp) before += sh.votes[w];
              all += sh.votes[w];
            }
            if (tie && before < need) cand[n + before] = rank_key(key_value(bound), e + t);
            n += min(all, need);
            need -= min(all, need);
            __syncthreads();
          }
        }
      }
      select_top(cand, n, k, sh.best);
    }
    __syncthreads();
    if (t == 0) {
      Sums all = sh.warp_sums[0];
      for (int w = 1; w < kT / 32; ++w) all = joined(all, sh.warp_sums[w]);
      sh.sums = all;
      sh.picked = k;
    }

    // ---- the parts joined by the cluster's first CTA
    if (parts > 1) {
      cluster.sync();
      if (part == 0 && top > 0) {
        int n = 0;
        for (int i = 0; i < parts; ++i) {
          const Shared* other = cluster.map_shared_rank(&sh, i);
          const int m = other->picked;
          for (int j = t; j < m; j += kT) sh.merged[n + j] = other->best[j];
          n += m;
        }
        __syncthreads();
        select_top(sh.merged, n, top, sh.best);
      }
    } else {
      __syncthreads();
    }
    if (part == 0) {
      Sums all = sh.sums;
      for (int i = 1; i < parts; ++i) all = joined(all, cluster.map_shared_rank(&sh, i)->sums);
      const bool nothing = all.l == 0.f;  // every logit -inf
      const float ref = all.ref == -INFINITY ? 0.f : all.ref, logl = logf(all.l);
      if (t == 0) {
        float lp = 0.f;
        if (token >= V) {
          atomicCAS(a.status, 0, kStatusBadToken);
          lp = __int_as_float(0x7fc00000);
        } else if (token >= 0) {
          lp = nothing ? -INFINITY : (token_logit - ref) - logl;
        }
        a.logprobs[r] = lp;
        a.entropy[r] = nothing ? 0.f : logl - kLn2 * (all.s / all.l);
      }
      for (int i = t; i < top; i += kT) {
        const uint64_t key = sh.best[i];
        a.top_ids[static_cast<int64_t>(r) * top + i] = 0xffffffffu - static_cast<uint32_t>(key);
        a.top_logprobs[static_cast<int64_t>(r) * top + i] =
            nothing ? -INFINITY : (key_value(static_cast<uint32_t>(key >> 32)) - ref) - logl;
      }
    }
    if (parts > 1) cluster.sync();  // the others' shared memory is read until here
    else __syncthreads();           // as this CTA's own is
  }
}

template <int DT>
cudaError_t launch(const ScoreArgs& a, cudaStream_t st) {
  // CTAs of a row: while the GPU holds all of them at once and each has two vectors a thread.
  constexpr int kVec = Type<DT>::kVec;
  const int sms = sm_count(current_device());
  if (sms <= 0) return cudaErrorInvalidDevice;
  const int64_t vectors = static_cast<int64_t>(a.vocab) / kVec + 2;
  int parts = 1;
  while (parts < kMaxCluster && static_cast<int64_t>(a.rows) * parts * 2 <= sms * kResident &&
         vectors / (parts * 2) >= 2 * kT)
    parts *= 2;
  const int64_t batches = (vectors / parts + 1 + kU * kT - 1) / (kU * kT);  // of a thread
  const int per_segment = static_cast<int>((batches + kSegments - 1) / kSegments);
  const int64_t segments = (batches + per_segment - 1) / per_segment;
  const size_t smem = kRing + (a.top > 0 ? kCandidates * 8 + static_cast<size_t>(segments) * kT * 4 : 0);
  const int rows = a.rows < sms * kResident ? a.rows : sms * kResident;  // at once
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * parts);
  cfg.blockDim = dim3(kT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, score_kernel<DT>, a, per_segment);
}

}  // namespace

cudaError_t launch_token_logprobs(const ScoreArgs& a, cudaStream_t st) {
  return a.dtype == 2 ? launch<2>(a, st) : a.dtype == 1 ? launch<1>(a, st) : launch<0>(a, st);
}

}  // namespace rp
