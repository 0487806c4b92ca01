// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b of length n, KV head h and each of the G = Hq / Hkv query
// heads g that share it:
//   s_gj = scale * q_g . k_j,  m_g = max_j s_gj,  l_g = sum_j 2^(s_gj - m_g)
//   out_g = sum_j 2^(s_gj - m_g) v_j / l_g,  lse_g = ln 2 * (m_g + log2 l_g)
// (s in log2 units), and on request w[b, h, j] += sum_g 2^(s_gj - m_g) / l_g.
// A sequence without tokens gives out = 0 and lse = -inf.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "internal.h"
#include "paged.h"

namespace rp {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSplits = 16;

__device__ __forceinline__ float value16(uint16_t u, bool f16) {
  return f16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(static_cast<uint32_t>(u) << 16);
}
__device__ __forceinline__ uint16_t round16(float x, bool f16) {
  return f16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
__device__ __forceinline__ float value_kv(const uint8_t* base, int64_t i, int dtype) {
  if (dtype == kKvE4m3)
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(base[i], __NV_E4M3)));
  return value16(reinterpret_cast<const uint16_t*>(base)[i], dtype == kKvF16);
}

// One warp per (sequence, query head, split): keys one after another, each
// lane D / 32 dimensions.
template <int D>
__global__ void decode_kernel(const PagedDecodeArgs a, float* part, float* scores, int cap) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x, split = blockIdx.x, hq = blockIdx.y, b = blockIdx.z;
  const int G = a.Hq / a.kv.heads, h = hq / G;
  const int n = table_length(a.t, a.kv.page_size, b, a.status);
  const int per = (n + kSplits - 1) / kSplits;
  const int j0 = split * per, j1 = min(n, j0 + per);
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = value16(a.q[b * a.q_seq + hq * a.q_head + e * 32 + lane], a.q_f16);
    o[e] = 0.f;
  }
  const int32_t* row = a.t.table + b * a.t.stride;
  for (int j = j0; j < j1; ++j) {
    const int64_t off = row_offset(a.kv, row, j, h, a.status);
    float x = -INFINITY, vs = 1.f;
    if (off >= 0) {
      x = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) x += q[e] * value_kv(a.kv.k, off + e * 32 + lane, a.kv.dtype);
#pragma unroll
      for (int s = 16; s > 0; s /= 2) x += __shfl_xor_sync(0xffffffffu, x, s);
      x *= a.scale_log2;
      if (a.kv.dtype == kKvE4m3) {
        const int64_t i = scale_index(a.kv, row, j, h);
        x *= a.kv.ks[i];
        vs = a.kv.vs[i];
      }
    }
    if (scores && lane == 0) scores[(static_cast<int64_t>(b) * a.Hq + hq) * cap + j] = x;
    const float m1 = (x > m) ? x : m;
    const float ref = m1 == -INFINITY ? 0.f : m1;
    const float keep = exp2f(m - ref), p = exp2f(x - ref);
    m = m1;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] *= keep;
      if (off >= 0) o[e] += p * vs * value_kv(a.kv.v, off + e * 32 + lane, a.kv.dtype);
    }
  }
  float* out = part + ((static_cast<int64_t>(b) * a.Hq + hq) * kSplits + split) * (D + 2);
  if (lane == 0) {
    out[0] = m;
    out[1] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[2 + e * 32 + lane] = o[e];
}

// The splits of one (sequence, query head) joined; one thread per dimension.
__global__ void decode_join_kernel(const PagedDecodeArgs a, const float* part, float* lse2, int D) {
  const int hq = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float* in = part + (static_cast<int64_t>(b) * a.Hq + hq) * kSplits * (D + 2);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s = 0; s < kSplits; ++s) m = fmaxf(m, in[s * (D + 2)]);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < kSplits; ++s) {
    const float f = exp2f(in[s * (D + 2)] - ref);
    l += in[s * (D + 2) + 1] * f;
    o += in[s * (D + 2) + 2 + d] * f;
  }
  a.out[b * a.o_seq + hq * a.o_head + d] = round16(l == 0.f ? 0.f : o / l, a.q_f16);
  if (d == 0) {
    lse2[b * a.Hq + hq] = m + log2f(l);
    if (a.lse) a.lse[b * a.Hq + hq] = kLn2 * (m + log2f(l));
  }
}

// Every key's weights, summed over the query heads of its KV head.
__global__ void decode_weights_kernel(const PagedDecodeArgs a, const float* scores, const float* lse2,
                                      int cap) {
  const int j = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (j >= table_length(a.t, a.kv.page_size, b, a.status)) return;
  const int G = a.Hq / a.kv.heads;
  float w = 0.f;
  for (int g = 0; g < G; ++g) {
    const int64_t hq = static_cast<int64_t>(b) * a.Hq + h * G + g;
    const float x = scores[hq * cap + j], y = lse2[hq];
    w += y == -INFINITY ? 0.f : exp2f(x - y);
  }
  a.weights.w[b * a.weights.s_seq + h * a.weights.s_head + j] += w;
}

struct Workspace {
  size_t part, lse2, scores, total;
  Workspace(const PagedPool& kv, int B, int Hq, int table_pages, bool weights) {
    const size_t heads = static_cast<size_t>(B) * Hq;
    part = 0;
    lse2 = heads * kSplits * (kv.D + 2) * 4;
    scores = lse2 + heads * 4;
    total = scores + (weights ? heads * table_pages * kv.page_size * 4 : 0);
  }
};

}  // namespace

size_t paged_decode_workspace(const PagedPool& kv, int B, int Hq, int table_pages, bool weights) {
  return Workspace(kv, B, Hq, table_pages, weights).total;
}

cudaError_t launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t st) {
  const Workspace ws(a.kv, a.t.B, a.Hq, a.t.pages, a.weights.w != nullptr);
  char* base = static_cast<char*>(a.workspace);
  float* part = reinterpret_cast<float*>(base + ws.part);
  float* lse2 = reinterpret_cast<float*>(base + ws.lse2);
  float* scores = a.weights.w ? reinterpret_cast<float*>(base + ws.scores) : nullptr;
  const int cap = a.t.pages * a.kv.page_size;
  const dim3 grid(kSplits, a.Hq, a.t.B);
  switch (a.kv.D) {
    case 32: decode_kernel<32><<<grid, 32, 0, st>>>(a, part, scores, cap); break;
    case 64: decode_kernel<64><<<grid, 32, 0, st>>>(a, part, scores, cap); break;
    case 128: decode_kernel<128><<<grid, 32, 0, st>>>(a, part, scores, cap); break;
    case 256: decode_kernel<256><<<grid, 32, 0, st>>>(a, part, scores, cap); break;
    default: return cudaErrorInvalidValue;
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  decode_join_kernel<<<dim3(a.Hq, a.t.B), a.kv.D, 0, st>>>(a, part, lse2, a.kv.D);
  e = cudaGetLastError();
  if (e != cudaSuccess || !scores || cap == 0) return e;
  decode_weights_kernel<<<dim3((cap + 255) / 256, a.kv.heads, a.t.B), 256, 0, st>>>(a, scores, lse2, cap);
  return cudaGetLastError();
}

}  // namespace rp
