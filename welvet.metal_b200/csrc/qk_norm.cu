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

// A CTA's sums of the gamma gradients into its two rows of `partial` (queries, keys):
// acc [warps][2][head_dim] is added up in warp order.
WV_DEV void write_partial(const QkNormArgs& a, const float* acc) {
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.head_dim; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kWarpsPerCta; ++w) s += acc[w * 2 * a.head_dim + i];
    a.partial[(size_t)blockIdx.x * 2 * a.head_dim + i] = s;
  }
}

// Backward with the same mapping. The gamma gradients are summed in registers over a
// warp's rows, over the CTA's warps in shared memory, and over the CTAs by
// dgamma_kernel, each time in a fixed order: no atomics, the same bits every time.
template <class T>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_rows_bwd_kernel(const QkNormArgs a) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float acc[];  // [warps][2][head_dim]
  const int half = a.head_dim / 2, lane = (int)lane_id(), warp = (int)warp_id();
  const int per = a.heads + a.kv_heads;
  const int64_t rows = a.tokens * per;
  float ga[2][kMaxPairs] = {}, gb[2][kMaxPairs] = {};
  for (int64_t row = (int64_t)blockIdx.x * kWarpsPerCta + warp; row < rows; row += (int64_t)gridDim.x * kWarpsPerCta) {
    const int64_t t = row / per;
    const int hh = (int)(row % per);
    const bool key = hh >= a.heads;
    const size_t h = (size_t)(key ? hh - a.heads : hh) * a.head_dim;
    const T* x = static_cast<const T*>(key ? a.k : a.q) + (size_t)t * (key ? a.ldk : a.ldq) + h;
    const T* dy = static_cast<const T*>(key ? a.dk_out : a.dq_out) + (size_t)t * (key ? a.lddko : a.lddqo) + h;
    T* dx = static_cast<T*>(key ? a.k_out : a.q_out) + (size_t)t * (key ? a.ldko : a.ldqo) + h;
    const float* gamma = key ? a.k_gamma : a.q_gamma;
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
        const float pa = za[j] * xa[j], pb = zb[j] * xb[j];
        ga[0][j] += key ? 0.f : pa;
        gb[0][j] += key ? 0.f : pb;
        ga[1][j] += key ? pa : 0.f;
        gb[1][j] += key ? pb : 0.f;
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
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int j = 0; j < kMaxPairs; ++j) {
      const int i = lane + 32 * j;
      if (i < half) {
        acc[(warp * 2 + side) * a.head_dim + i] = ga[side][j];
        acc[(warp * 2 + side) * a.head_dim + half + i] = gb[side][j];
      }
    }
  write_partial(a, acc);
}

// dgamma = sum of the CTAs' partial rows: 32 columns a CTA, 32 threads on a column take
// every 32nd row, then add up in row order.
__global__ void __launch_bounds__(1024) dgamma_kernel(const float* partial, int parts, int hd, float* dq_gamma, float* dk_gamma) {
  __shared__ float sum[32][33];
  pdl_wait();
  pdl_trigger();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, i = blockIdx.x * 32 + x;
  float s = 0.f;
  if (i < 2 * hd)
    for (int p = y; p < parts; p += 32) s += partial[(size_t)p * 2 * hd + i];
  sum[y][x] = s;
  __syncthreads();
  if (y == 0 && i < 2 * hd) {
    for (int k = 1; k < 32; ++k) s += sum[k][x];
    float* out = i < hd ? dq_gamma : dk_gamma;
    if (out) out[i % hd] = s;
  }
}

// ------------------------------------------------------------ 16-byte rows
// head_dim 64, 128, 256 with rows aligned to 16 bytes: VEC pairs of a row per lane (16
// bytes of each half), so a row takes hd / 2 / VEC lanes and a warp RPW rows at once;
// the partners of a rotation sit in one lane, and a warp keeps the angles and gammas of
// its token in registers over all heads of its share. Bound by HBM: the loads of two
// row groups are in flight before the first is used.
template <class T, int HD> struct VT {
  static constexpr int VEC = 16 / (int)sizeof(T), LPR = HD / 2 / VEC, RPW = 32 / LPR;
};
template <class T, int HD> WV_DEV float row_sum(float v) {
#pragma unroll
  for (int o = VT<T, HD>::LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
WV_DEV void unpack(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
WV_DEV void unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x);
  f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z);
  f[3] = __uint_as_float(u.w);
}
WV_DEV uint4 pack(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
WV_DEV uint4 pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <int N> WV_DEV void load_f(const float* p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    f[i] = v.x;
    f[i + 1] = v.y;
    f[i + 2] = v.z;
    f[i + 3] = v.w;
  }
}

// A warp's share of one token: groups [g0, g1) of RPW heads, the query groups first.
// BWD: dx and the gamma gradients instead of y.
template <class T, int HD, bool BWD>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_vec_kernel(const QkNormArgs a, int slices) {
  using V = VT<T, HD>;
  constexpr int VEC = V::VEC;
  extern __shared__ float acc[];
  pdl_wait();
  pdl_trigger();
  const int lane = (int)lane_id(), warp = (int)warp_id();
  const int sub = lane / V::LPR, at = (lane % V::LPR) * VEC;  // row of the group, first pair
  const int gq = (a.heads + V::RPW - 1) / V::RPW, groups = gq + (a.kv_heads + V::RPW - 1) / V::RPW;
  const int per = (groups + slices - 1) / slices;
  const uint32_t units = (uint32_t)a.tokens * (uint32_t)slices;
  float dg[BWD ? 2 : 1][2][VEC];  // [queries, keys][half]
#pragma unroll
  for (int i = 0; i < (BWD ? 2 : 1) * 2 * VEC; ++i) (&dg[0][0][0])[i] = 0.f;

  for (uint32_t unit = blockIdx.x * kWarpsPerCta + warp; unit < units; unit += gridDim.x * kWarpsPerCta) {
    const int64_t t = unit / (uint32_t)slices;
    const int g0 = (int)(unit % (uint32_t)slices) * per, g1 = min(groups, g0 + per);
    float cs[2 * VEC];
    const float2* tab = angles(a, t, HD / 2);
    if (tab) {
      load_f(reinterpret_cast<const float*>(tab + at), cs);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        cs[2 * i] = 1.f;
        cs[2 * i + 1] = 0.f;
      }
    }
    auto side = [&](int key, const void* xp, int64_t ldx, const void* dyp, int64_t lddy, void* yp, int64_t ldy,
                    const float* gamma, int heads, int from, int to) {
      if (from >= to) return;
      const T* x = static_cast<const T*>(xp) + t * ldx + at;
      const T* dy = BWD ? static_cast<const T*>(dyp) + t * lddy + at : nullptr;
      T* y = static_cast<T*>(yp) + t * ldy + at;
      float w[2][VEC];
      if (gamma) {
        load_f(gamma + at, w[0]);
        load_f(gamma + HD / 2 + at, w[1]);
      }
      constexpr int U = 2;  // row groups in flight
      for (int g = from; g < to; g += U) {
        uint4 in[U][2], up[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = (g + u) * V::RPW + sub;
          const bool on = g + u < to && h < heads;
          in[u][0] = in[u][1] = up[u][0] = up[u][1] = make_uint4(0u, 0u, 0u, 0u);
          if (on && (!BWD || gamma)) {
            in[u][0] = *reinterpret_cast<const uint4*>(x + (size_t)h * HD);
            in[u][1] = *reinterpret_cast<const uint4*>(x + (size_t)h * HD + HD / 2);
          }
          if (BWD && on) {
            up[u][0] = *reinterpret_cast<const uint4*>(dy + (size_t)h * HD);
            up[u][1] = *reinterpret_cast<const uint4*>(dy + (size_t)h * HD + HD / 2);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = (g + u) * V::RPW + sub;
          float xa[VEC], xb[VEC], ya[VEC], yb[VEC], r = 1.f;
          unpack(in[u][0], xa);
          unpack(in[u][1], xb);
          if (gamma) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
            r = rsqrtf(row_sum<T, HD>(ss) * (1.f / HD) + a.eps);
          }
          if (!BWD) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float za = gamma ? xa[i] * r * w[0][i] : xa[i], zb = gamma ? xb[i] * r * w[1][i] : xb[i];
              ya[i] = za * cs[2 * i] - zb * cs[2 * i + 1];
              yb[i] = za * cs[2 * i + 1] + zb * cs[2 * i];
            }
          } else {
            float da[VEC], db[VEC], dot = 0.f;
            unpack(up[u][0], da);
            unpack(up[u][1], db);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              float za = da[i] * cs[2 * i] + db[i] * cs[2 * i + 1], zb = db[i] * cs[2 * i] - da[i] * cs[2 * i + 1];
              if (gamma) {
                xa[i] *= r;
                xb[i] *= r;
                dg[BWD ? key : 0][0][i] += za * xa[i];
                dg[BWD ? key : 0][1][i] += zb * xb[i];
                za *= w[0][i];
                zb *= w[1][i];
                dot += za * xa[i] + zb * xb[i];
              }
              da[i] = za;
              db[i] = zb;
            }
            if (gamma) dot = row_sum<T, HD>(dot) * (1.f / HD);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              ya[i] = gamma ? r * (da[i] - xa[i] * dot) : da[i];
              yb[i] = gamma ? r * (db[i] - xb[i] * dot) : db[i];
            }
          }
          if (g + u < to && h < heads) {
            *reinterpret_cast<uint4*>(y + (size_t)h * HD) = pack(ya);
            *reinterpret_cast<uint4*>(y + (size_t)h * HD + HD / 2) = pack(yb);
          }
        }
      }
    };
    side(0, a.q, a.ldq, a.dq_out, a.lddqo, a.q_out, a.ldqo, a.q_gamma, a.heads, min(g0, gq), min(g1, gq));
    side(1, a.k, a.ldk, a.dk_out, a.lddko, a.k_out, a.ldko, a.k_gamma, a.kv_heads, max(g0, gq) - gq, max(g1, gq) - gq);
  }
  if constexpr (BWD) {
#pragma unroll
    for (int key = 0; key < 2; ++key)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float v = dg[key][hf][i];
#pragma unroll
          for (int o = 16; o >= V::LPR; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if (sub == 0) acc[(warp * 2 + key) * HD + hf * (HD / 2) + at + i] = v;
        }
    write_partial(a, acc);
  }
}

// Rows that the 16-byte kernel can take.
bool vec_ok(const QkNormArgs& a, bool bwd) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
  const int es = a.is_bf16 ? 2 : 4;
  const auto fits = [&](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0; };
  const auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  if (low(a.q_gamma) || low(a.k_gamma) || low(a.rope)) return false;
  if (a.heads && (!fits(a.q, a.ldq) || !fits(a.q_out, a.ldqo) || (bwd && !fits(a.dq_out, a.lddqo)))) return false;
  if (a.kv_heads && (!fits(a.k, a.ldk) || !fits(a.k_out, a.ldko) || (bwd && !fits(a.dk_out, a.lddko)))) return false;
  return true;
}

// A token is one warp's work, or shared by several while tokens alone leave the SMs
// without kWarpsPerSm warps each.
constexpr int kWarpsPerSm = 32;
template <class T, int HD, bool BWD> cudaError_t launch_vec(const QkNormArgs& a, int max_grid, cudaStream_t s, int* grid_out) {
  using V = VT<T, HD>;
  const int groups = (a.heads + V::RPW - 1) / V::RPW + (a.kv_heads + V::RPW - 1) / V::RPW;
  const int64_t want = (int64_t)a.sm_count * kWarpsPerSm;
  const int slices = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (want + a.tokens - 1) / std::max<int64_t>(1, a.tokens)));
  const int64_t ctas = (a.tokens * slices + kWarpsPerCta - 1) / kWarpsPerCta;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(ctas, max_grid));
  *grid_out = grid;
  return launch_pdl(qk_norm_vec_kernel<T, HD, BWD>, dim3(grid), dim3(kWarpsPerCta * 32),
                    BWD ? (size_t)kWarpsPerCta * 2 * HD * sizeof(float) : 0, s, a, slices);
}
template <bool BWD> cudaError_t launch_vec_any(const QkNormArgs& a, int max_grid, cudaStream_t s, int* grid) {
  switch (a.head_dim) {
  case 64: return a.is_bf16 ? launch_vec<__nv_bfloat16, 64, BWD>(a, max_grid, s, grid) : launch_vec<float, 64, BWD>(a, max_grid, s, grid);
  case 128: return a.is_bf16 ? launch_vec<__nv_bfloat16, 128, BWD>(a, max_grid, s, grid) : launch_vec<float, 128, BWD>(a, max_grid, s, grid);
  default: return a.is_bf16 ? launch_vec<__nv_bfloat16, 256, BWD>(a, max_grid, s, grid) : launch_vec<float, 256, BWD>(a, max_grid, s, grid);
  }
}

}  // namespace

size_t qk_norm_workspace_bytes(int head_dim) { return (size_t)kQkNormParts * 2 * head_dim * sizeof(float); }

cudaError_t qk_norm_forward(const QkNormArgs& a, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  if (rows == 0) return cudaSuccess;
  int grid = 0;
  if (vec_ok(a, false)) return launch_vec_any<false>(a, 1 << 30, s, &grid);
  grid = (int)std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, (int64_t)a.sm_count * 64);
  return a.is_bf16 ? launch_pdl(qk_norm_rows_kernel<__nv_bfloat16>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a)
                   : launch_pdl(qk_norm_rows_kernel<float>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a);
}

cudaError_t qk_norm_backward(const QkNormArgs& a, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  int parts = 0;
  cudaError_t e;
  if (vec_ok(a, true)) {
    e = launch_vec_any<true>(a, kQkNormParts, s, &parts);
  } else {
    parts = (int)std::max<int64_t>(1, std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, kQkNormParts));
    const size_t smem = (size_t)kWarpsPerCta * 2 * a.head_dim * sizeof(float);
    e = a.is_bf16 ? launch_pdl(qk_norm_rows_bwd_kernel<__nv_bfloat16>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a)
                  : launch_pdl(qk_norm_rows_bwd_kernel<float>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a);
  }
  if (e != cudaSuccess || (!a.dq_gamma && !a.dk_gamma)) return e;
  return launch_pdl(dgamma_kernel, dim3((2 * a.head_dim + 31) / 32), dim3(1024), 0, s, (const float*)a.partial, parts,
                    a.head_dim, a.dq_gamma, a.dk_gamma);
}

}  // namespace wv
