// Log probability of given tokens, entropy, and the top alternatives of every
// row of logits.
//
// With m = max_v x_v, l = sum_v e^(x_v - m) and lse = m + log l:
//   logprob = x_token - lse
//   entropy = log l - (sum_v e^(x_v - m) (x_v - m)) / l
//   top     = the `top` largest x_v - lse, ties to the lowest index.
// A row whose every logit is -inf has entropy 0 and log probabilities -inf;
// a NaN or +inf in a row makes its sums NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "paged.h"

namespace rp {
namespace {

constexpr int kScoreThreads = 512;

__device__ __forceinline__ float logit(const void* row, int64_t i, int dtype) {
  if (dtype == 2) return static_cast<const float*>(row)[i];
  const uint16_t u = static_cast<const uint16_t*>(row)[i];
  return dtype == 1 ? __half2float(__ushort_as_half(u)) : __uint_as_float(static_cast<uint32_t>(u) << 16);
}

// Order of alternatives as one integer: larger value first, then lower index.
// NaN is above +inf, -0 equals 0.
__device__ __forceinline__ uint64_t rank_key(float x, int i) {
  uint32_t u = __float_as_uint(x);
  if (x != x) u = 0xffffffffu;
  else if (u == 0x80000000u) u = 0x80000000u;
  else u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

template <typename T, typename F>
__device__ T block_reduce(T x, T* buf, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 16; s > 0; s /= 2) x = f(x, __shfl_xor_sync(0xffffffffu, x, s));
  __syncthreads();
  if (lane == 0) buf[warp] = x;
  __syncthreads();
  x = buf[0];
  for (int w = 1; w < kScoreThreads / 32; ++w) x = f(x, buf[w]);
  return x;
}

// One CTA a row: maximum, then the sums, then one pass per alternative.
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const ScoreArgs a) {
  __shared__ float fbuf[kScoreThreads / 32];
  __shared__ uint64_t kbuf[kScoreThreads / 32];
  const int r = blockIdx.x, size = a.dtype == 2 ? 4 : 2;
  const void* row = static_cast<const char*>(a.logits) + r * a.stride * size;
  const auto fmax2 = [](float x, float y) { return (x != x || x > y) ? x : y; };
  const auto add = [](float x, float y) { return x + y; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) m = fmax2(logit(row, i, a.dtype), m);
  m = block_reduce(m, fbuf, fmax2);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, s = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float d = logit(row, i, a.dtype) - ref, e = expf(d);
    l += e;
    if (e != 0.f) s += e * d;
  }
  l = block_reduce(l, fbuf, add);
  s = block_reduce(s, fbuf, add);
  const float logl = logf(l);
  if (threadIdx.x == 0) {
    const int64_t t = a.tokens[r];
    float lp = 0.f;
    if (t >= a.vocab) {
      atomicCAS(a.status, 0, kStatusBadToken);
      lp = __int_as_float(0x7fc00000);
    } else if (t >= 0) {
      // (x - m) - log l, not x - lse: the latter cancels where |m| is large
      lp = m == -INFINITY ? -INFINITY : (logit(row, t, a.dtype) - ref) - logl;
    }
    a.logprobs[r] = lp;
    a.entropy[r] = m == -INFINITY ? 0.f : logl - s / l;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
      const uint64_t key = rank_key(logit(row, i, a.dtype), i);
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, kbuf, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    last = best;
    if (threadIdx.x == 0) {
      const int64_t i = 0xffffffffu - static_cast<uint32_t>(best);
      a.top_ids[static_cast<int64_t>(r) * a.top + k] = i;
      a.top_logprobs[static_cast<int64_t>(r) * a.top + k] =
          m == -INFINITY ? -INFINITY : (logit(row, i, a.dtype) - ref) - logl;
    }
  }
}

}  // namespace

cudaError_t launch_token_logprobs(const ScoreArgs& a, cudaStream_t st) {
  score_kernel<<<a.rows, kScoreThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace rp
