// RMS norm of every query and key head with the position rotation in the same pass,
// and its gradient.
//
// For one row x (a head of one token, hd values), r = (mean(x^2) + eps)^-1/2 and the
// rotation R of the pairs (i, i + hd/2) by the token's angles (the reference's RoPE,
// shaders/ops_mha.metal:14-29):
//   forward   y = R (gamma * x r)
//   backward  dz = R^T dy, dgamma = sum over rows of dz * x r,
//             u = dz gamma, dx = r (u - x r mean(u * x r))
// Without gamma the row is only rotated (y = R x, dx = R^T dy); without a table it is
// only normalised. Everything between the loads and the stores is FP32; BF16 outputs
// are rounded once. No reference counterpart for the norm (its MHA has none).
#include "common.cuh"
#include "kernels.h"

#include <algorithm>

namespace wv {
namespace {

constexpr int kWarpsPerCta = 8;
constexpr int kMaxPairs = kQkNormMaxHeadDim / 2 / 32;  // pairs of a row per lane

template <class T> WV_DEV float ld_f(const T* p);
template <> WV_DEV float ld_f<float>(const float* p) { return *p; }
template <> WV_DEV float ld_f<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
WV_DEV void st_f(float* p, float v) { *p = v; }
WV_DEV void st_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

WV_DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Table row of a token, or null when it is not rotated. A position outside the table
// is recorded in the error word and leaves the row unrotated.
WV_DEV const float2* angles(const QkNormArgs& a, int64_t t, int half) {
  if (!a.rope) return nullptr;
  const int pos = a.positions ? a.positions[t] : (int)(a.pos_mod > 0 ? t % a.pos_mod : t);
  if (pos < 0 || pos >= a.max_pos) {
    if (a.err) atomicCAS(a.err, 0u, kErrRopePos);
    return nullptr;
  }
  return a.rope + (size_t)pos * half;
}

// One warp per row, lane l on pairs l, l + 32, ...: any even head_dim up to
// kQkNormMaxHeadDim and any row stride or alignment.
template <class T>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_rows_kernel(const QkNormArgs a) {
  pdl_wait();
  pdl_trigger();
  const int half = a.head_dim / 2, lane = (int)lane_id();
  const int per = a.heads + a.kv_heads;
  const int64_t rows = a.tokens * per;
  for (int64_t row = (int64_t)blockIdx.x * kWarpsPerCta + warp_id(); row < rows;
       row += (int64_t)gridDim.x * kWarpsPerCta) {
    const int64_t t = row / per;
    const int h = (int)(row % per);
    const bool key = h >= a.heads;
    const size_t in = key ? (size_t)t * a.ldk + (size_t)(h - a.heads) * a.head_dim : (size_t)t * a.ldq + (size_t)h * a.head_dim;
    const size_t to = key ? (size_t)t * a.ldko + (size_t)(h - a.heads) * a.head_dim : (size_t)t * a.ldqo + (size_t)h * a.head_dim;
    const T* x = static_cast<const T*>(key ? a.k : a.q) + in;
    T* y = static_cast<T*>(key ? a.k_out : a.q_out) + to;
    const float* gamma = key ? a.k_gamma : a.q_gamma;
    float xa[kMaxPairs], xb[kMaxPairs], ss = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxPairs; ++j) {
      const int i = lane + 32 * j;
      xa[j] = i < half ? ld_f<T>(x + i) : 0.f;
      xb[j] = i < half ? ld_f<T>(x + half + i) : 0.f;
      ss += xa[j] * xa[j] + xb[j] * xb[j];
    }
    const float r = gamma ? rsqrtf(warp_sum(ss) / (float)a.head_dim + a.eps) : 1.f;
    const float2* cs = angles(a, t, half);
#pragma unroll
    for (int j = 0; j < kMaxPairs; ++j) {
      const int i = lane + 32 * j;
      if (i >= half) continue;
      const float za = gamma ? xa[j] * r * gamma[i] : xa[j], zb = gamma ? xb[j] * r * gamma[half + i] : xb[j];
      const float2 c = cs ? cs[i] : make_float2(1.f, 0.f);
      st_f(y + i, za * c.x - zb * c.y);
      st_f(y + half + i, za * c.y + zb * c.x);
    }
  }
}

// Backward with the same mapping. CTAs below a.part_q take query rows, the others key
// rows; each sums its rows' gamma gradients in registers, then over its warps, into
// its own row of `partial`, which dgamma_kernel adds up in row order: no atomics, the
// same result every time.
template <class T>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_rows_bwd_kernel(const QkNormArgs a) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float acc[];  // [warps][head_dim]
  const int half = a.head_dim / 2, lane = (int)lane_id(), warp = (int)warp_id();
  const bool key = (int)blockIdx.x >= a.part_q;
  const int per = key ? a.kv_heads : a.heads;
  const int64_t rows = a.tokens * per, ctas = key ? gridDim.x - a.part_q : a.part_q;
  const float* gamma = key ? a.k_gamma : a.q_gamma;
  float ga[kMaxPairs] = {}, gb[kMaxPairs] = {};
  for (int64_t row = (int64_t)(blockIdx.x - (key ? a.part_q : 0)) * kWarpsPerCta + warp; row < rows;
       row += ctas * kWarpsPerCta) {
    const int64_t t = row / per;
    const size_t h = (size_t)(row % per) * a.head_dim;
    const T* x = static_cast<const T*>(key ? a.k : a.q) + (size_t)t * (key ? a.ldk : a.ldq) + h;
    const T* dy = static_cast<const T*>(key ? a.dk_out : a.dq_out) + (size_t)t * (key ? a.lddko : a.lddqo) + h;
    T* dx = static_cast<T*>(key ? a.k_out : a.q_out) + (size_t)t * (key ? a.ldko : a.ldqo) + h;
    const float2* cs = angles(a, t, half);
    float xa[kMaxPairs], xb[kMaxPairs], za[kMaxPairs], zb[kMaxPairs], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxPairs; ++j) {
      const int i = lane + 32 * j;
      xa[j] = xb[j] = za[j] = zb[j] = 0.f;
      if (i >= half) continue;
      const float2 c = cs ? cs[i] : make_float2(1.f, 0.f);
      const float da = ld_f<T>(dy + i), db = ld_f<T>(dy + half + i);
      za[j] = da * c.x + db * c.y;
      zb[j] = db * c.x - da * c.y;
      if (!gamma) continue;
      xa[j] = ld_f<T>(x + i);
      xb[j] = ld_f<T>(x + half + i);
      ss += xa[j] * xa[j] + xb[j] * xb[j];
    }
    float r = 1.f;
    if (gamma) {
      r = rsqrtf(warp_sum(ss) / (float)a.head_dim + a.eps);
#pragma unroll
      for (int j = 0; j < kMaxPairs; ++j) {
        const int i = lane + 32 * j;
        if (i >= half) continue;
        xa[j] *= r;
        xb[j] *= r;
        ga[j] += za[j] * xa[j];
        gb[j] += zb[j] * xb[j];
        za[j] *= gamma[i];
        zb[j] *= gamma[half + i];
        dot += za[j] * xa[j] + zb[j] * xb[j];
      }
      dot = warp_sum(dot) / (float)a.head_dim;
    }
#pragma unroll
    for (int j = 0; j < kMaxPairs; ++j) {
      const int i = lane + 32 * j;
      if (i >= half) continue;
      st_f(dx + i, r * (za[j] - xa[j] * dot));
      st_f(dx + half + i, r * (zb[j] - xb[j] * dot));
    }
  }
#pragma unroll
  for (int j = 0; j < kMaxPairs; ++j) {
    const int i = lane + 32 * j;
    if (i < half) {
      acc[warp * a.head_dim + i] = ga[j];
      acc[warp * a.head_dim + half + i] = gb[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.head_dim; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kWarpsPerCta; ++w) s += acc[w * a.head_dim + i];
    a.partial[(size_t)blockIdx.x * a.head_dim + i] = s;
  }
}

// dgamma[q or k][i] = sum of the partial rows in row order.
__global__ void dgamma_kernel(const float* partial, int part_q, int parts, int hd, float* dq_gamma, float* dk_gamma) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= hd) return;
  float* out = blockIdx.y ? dk_gamma : dq_gamma;
  if (!out) return;
  float s = 0.f;
  for (int p = blockIdx.y ? part_q : 0; p < (blockIdx.y ? parts : part_q); ++p) s += partial[(size_t)p * hd + i];
  out[i] = s;
}

}  // namespace

size_t qk_norm_workspace_bytes(int head_dim) { return (size_t)kQkNormParts * head_dim * sizeof(float); }

cudaError_t qk_norm_forward(const QkNormArgs& a, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  if (rows == 0) return cudaSuccess;
  const int grid = (int)std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, (int64_t)a.sm_count * 64);
  return a.is_bf16 ? launch_pdl(qk_norm_rows_kernel<__nv_bfloat16>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a)
                   : launch_pdl(qk_norm_rows_kernel<float>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a);
}

cudaError_t qk_norm_backward(const QkNormArgs& in, cudaStream_t s) {
  QkNormArgs a = in;
  // CTAs in proportion to the rows of queries and keys, at least one for each
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  const int parts = (int)std::max<int64_t>(2, std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, kQkNormParts));
  a.part_q = std::min(parts - 1, std::max(1, (int)((int64_t)parts * a.heads / std::max(1, a.heads + a.kv_heads))));
  const size_t smem = (size_t)kWarpsPerCta * a.head_dim * sizeof(float);
  cudaError_t e = a.is_bf16 ? launch_pdl(qk_norm_rows_bwd_kernel<__nv_bfloat16>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a)
                            : launch_pdl(qk_norm_rows_bwd_kernel<float>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a);
  if (e != cudaSuccess || (!a.dq_gamma && !a.dk_gamma)) return e;
  return launch_pdl(dgamma_kernel, dim3((a.head_dim + 127) / 128, 2), dim3(128), 0, s, (const float*)a.partial, a.part_q,
                    parts, a.head_dim, a.dq_gamma, a.dk_gamma);
}

}  // namespace wv
