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
// kQkNormMaxHeadDim and any row stride or alignment. Bound by the issue of its narrow
// accesses: 446 us for 16384 tokens x 64 heads of 128, BF16 (92 with aligned rows).
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

// A CTA's sum of its side's gamma gradient into its row of `partial`: acc
// [warps][head_dim] is added up in warp order.
WV_DEV void write_partial(const QkNormArgs& a, const float* acc) {
  __syncthreads();
  for (int i = threadIdx.x; i < a.head_dim; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kWarpsPerCta; ++w) s += acc[w * a.head_dim + i];
    a.partial[(size_t)blockIdx.x * a.head_dim + i] = s;
  }
}

// Backward with the same mapping. The first part_q CTAs take the query rows, the others
// the key rows. The gamma gradients are summed in registers over a warp's rows, over
// the CTA's warps in shared memory, and over the CTAs by dgamma_kernel, each time in a
// fixed order: no atomics, the same bits every time. 588 us for 16384 x 40 heads of 128
// (104 with aligned rows).
template <class T>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_rows_bwd_kernel(const QkNormArgs a, int part_q) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float acc[];  // [warps][head_dim]
  const int half = a.head_dim / 2, lane = (int)lane_id(), warp = (int)warp_id();
  const bool key = (int)blockIdx.x >= part_q;
  const int per = key ? a.kv_heads : a.heads;
  const int64_t rows = a.tokens * per, ctas = key ? gridDim.x - part_q : part_q;
  const float* gamma = key ? a.k_gamma : a.q_gamma;
  float ga[kMaxPairs] = {}, gb[kMaxPairs] = {};
  for (int64_t row = (int64_t)(blockIdx.x - (key ? part_q : 0)) * kWarpsPerCta + warp; row < rows;
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
  write_partial(a, acc);
}

// dgamma = sum of the CTAs' partial rows (the first part_q belong to the queries): 32
// columns a CTA, 32 threads on a column take every 32nd row, then add up in row order.
__global__ void __launch_bounds__(1024) dgamma_kernel(const float* partial, int part_q, int parts, int hd, float* dq_gamma,
                                                      float* dk_gamma) {
  __shared__ float sum[32][33];
  pdl_wait();
  pdl_trigger();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, i = blockIdx.x * 32 + x;
  const int to = blockIdx.y ? parts : part_q;
  float s = 0.f;
  if (i < hd)
    for (int p = (blockIdx.y ? part_q : 0) + y; p < to; p += 32) s += partial[(size_t)p * hd + i];
  sum[y][x] = s;
  __syncthreads();
  if (y == 0 && i < hd) {
    for (int k = 1; k < 32; ++k) s += sum[k][x];
    float* out = blockIdx.y ? dk_gamma : dq_gamma;
    if (out) out[i] = s;
  }
}

// ------------------------------------------------------------ aligned rows
// head_dim 64, 128, 256 with rows aligned to 16 bytes: VEC pairs of a row per lane, so a
// row takes hd / 2 / VEC lanes and a warp RPW rows at once; the partners of a rotation
// sit in one lane, and a warp keeps the angles of its token and the gammas of its side
// in registers over all heads of its share. Bound by HBM: two groups of rows are
// requested before the first is used. Forward: 16 bytes a load (16384 tokens x 64 heads
// of 128, BF16: 92 us, 5.9 TB/s, 0.91 of the copy rate; x 40 heads, FP32: 108 us, 0.96;
// in a CUDA graph, 95 a call). Backward: four pairs a lane, since x, dy, gamma, its
// gradient and the angles of eight pairs take 161 registers, 8 warps an SM: 143 us for
// 16384 x 40 heads of 128, against 103 (108 a call; 5.0 TB/s, 0.76 of the copy rate). What
// keeps it there: a warp takes whole tokens over a fixed grid, so the busiest does 80 row
// groups of a mean of 69 here (48 of 35 for 8192 tokens), and its loads are the leading
// stall (5.3 warps an issue; shuffles 1.3), although rows fetched three pieces ahead into
// shared memory took 101 to 131 us. Even shares of row groups have not been tried.
template <class T, int HD, bool BWD> struct VT {
  static constexpr int VEC = BWD ? 4 : 16 / (int)sizeof(T), LPR = HD / 2 / VEC, RPW = 32 / LPR;
};
template <int LPR> WV_DEV float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int WORDS> struct Raw {  // WORDS 32-bit words, loaded and stored at once
  uint32_t w[WORDS];
};
template <int WORDS> WV_DEV void load_raw(Raw<WORDS>& r, const void* p) {
  if constexpr (WORDS == 4) {
    const uint4 v = *static_cast<const uint4*>(p);
    r.w[0] = v.x;
    r.w[1] = v.y;
    r.w[2] = v.z;
    r.w[3] = v.w;
  } else {
    const uint2 v = *static_cast<const uint2*>(p);
    r.w[0] = v.x;
    r.w[1] = v.y;
  }
}
template <int WORDS> WV_DEV void store_raw(void* p, const Raw<WORDS>& r) {
  if constexpr (WORDS == 4) *static_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else *static_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
}
template <class T, int VEC> WV_DEV void unpack(const Raw<VEC * sizeof(T) / 4>& r, float (&f)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    f[i] = sizeof(T) == 4 ? __uint_as_float(r.w[i]) : __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
}
template <class T, int VEC> WV_DEV Raw<VEC * sizeof(T) / 4> pack(const float (&f)[VEC]) {
  Raw<VEC * sizeof(T) / 4> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) r.w[i / 2] = pack_bf16x2(f[i], f[i + 1]);
  }
  return r;
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

// A warp's share of one token and side: groups of RPW heads. The first part_q CTAs take
// the queries, the others the keys; slices_q / slices_k warps share a token. BWD: dx and
// the gamma gradients instead of y.
template <class T, int HD, bool BWD>
__global__ void __launch_bounds__(kWarpsPerCta * 32, BWD ? 4 : 3)
    qk_norm_vec_kernel(const QkNormArgs a, int part_q, int slices_q, int slices_k) {
  using V = VT<T, HD, BWD>;
  constexpr int VEC = V::VEC, WORDS = VEC * (int)sizeof(T) / 4;
  extern __shared__ float acc[];
  pdl_wait();
  pdl_trigger();
  const int lane = (int)lane_id(), warp = (int)warp_id();
  const int sub = lane / V::LPR, at = (lane % V::LPR) * VEC;  // row of the group, first pair
  const bool key = (int)blockIdx.x >= part_q;
  const int heads = key ? a.kv_heads : a.heads;
  const uint32_t slices = key ? slices_k : slices_q, ctas = key ? gridDim.x - part_q : part_q;
  const int groups = (heads + V::RPW - 1) / V::RPW, per = (groups + (int)slices - 1) / (int)slices;
  const uint32_t units = heads ? (uint32_t)a.tokens * slices : 0u;
  const float* gamma = key ? a.k_gamma : a.q_gamma;
  const T* xp = static_cast<const T*>(key ? a.k : a.q) + at;
  const T* dyp = BWD ? static_cast<const T*>(key ? a.dk_out : a.dq_out) + at : nullptr;
  T* yp = static_cast<T*>(key ? a.k_out : a.q_out) + at;
  const int64_t ldx = key ? a.ldk : a.ldq, lddy = key ? a.lddko : a.lddqo, ldy = key ? a.ldko : a.ldqo;
  float w[2][VEC], dg[2][VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) w[0][i] = w[1][i] = dg[0][i] = dg[1][i] = 0.f;
  if (gamma) {
    load_f(gamma + at, w[0]);
    load_f(gamma + HD / 2 + at, w[1]);
  }

  for (uint32_t unit = (blockIdx.x - (key ? part_q : 0)) * kWarpsPerCta + warp; unit < units; unit += ctas * kWarpsPerCta) {
    const int64_t t = unit / slices;
    const int g0 = (int)(unit % slices) * per, g1 = min(groups, g0 + per);
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
    const T* x = xp + t * ldx;
    const T* dy = BWD ? dyp + t * lddy : nullptr;
    T* y = yp + t * ldy;
    constexpr int U = BWD && sizeof(T) == 4 ? 1 : 2;  // row groups in flight (FP32 backward: 27 us with 2, 22 with 1)
    for (int g = g0; g < g1; g += U) {
      Raw<WORDS> in[U][2], up[BWD ? U : 1][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (g + u) * V::RPW + sub;
        const bool on = g + u < g1 && h < heads;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          in[u][hf] = Raw<WORDS>{};
          if (on && (!BWD || gamma)) load_raw(in[u][hf], x + (size_t)h * HD + hf * (HD / 2));
          if constexpr (BWD) {
            up[u][hf] = Raw<WORDS>{};
            if (on) load_raw(up[u][hf], dy + (size_t)h * HD + hf * (HD / 2));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (g + u) * V::RPW + sub;
        float xa[VEC], xb[VEC], ya[VEC], yb[VEC], r = 1.f;
        unpack<T>(in[u][0], xa);
        unpack<T>(in[u][1], xb);
        if (gamma) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < VEC; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
          r = rsqrtf(row_sum<V::LPR>(ss) * (1.f / HD) + a.eps);
        }
        if constexpr (!BWD) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float za = gamma ? xa[i] * r * w[0][i] : xa[i], zb = gamma ? xb[i] * r * w[1][i] : xb[i];
            ya[i] = za * cs[2 * i] - zb * cs[2 * i + 1];
            yb[i] = za * cs[2 * i + 1] + zb * cs[2 * i];
          }
        } else {
          float da[VEC], db[VEC], dot = 0.f;
          unpack<T>(up[u][0], da);
          unpack<T>(up[u][1], db);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float za = da[i] * cs[2 * i] + db[i] * cs[2 * i + 1], zb = db[i] * cs[2 * i] - da[i] * cs[2 * i + 1];
            if (gamma) {
              xa[i] *= r;
              xb[i] *= r;
              dg[0][i] += za * xa[i];
              dg[1][i] += zb * xb[i];
              za *= w[0][i];
              zb *= w[1][i];
              dot += za * xa[i] + zb * xb[i];
            }
            da[i] = za;
            db[i] = zb;
          }
          if (gamma) dot = row_sum<V::LPR>(dot) * (1.f / HD);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            ya[i] = gamma ? r * (da[i] - xa[i] * dot) : da[i];
            yb[i] = gamma ? r * (db[i] - xb[i] * dot) : db[i];
          }
        }
        if (g + u < g1 && h < heads) {
          store_raw(y + (size_t)h * HD, pack<T>(ya));
          store_raw(y + (size_t)h * HD + HD / 2, pack<T>(yb));
        }
      }
    }
  }
  if constexpr (BWD) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float v = dg[hf][i];
#pragma unroll
        for (int o = 16; o >= V::LPR; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (sub == 0) acc[warp * HD + hf * (HD / 2) + at + i] = v;
      }
    write_partial(a, acc);
  }
}

// Rows that the vector kernel can take.
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

// CTAs of the queries among `ctas` in proportion to the rows, one at least for each side.
int queries_part(const QkNormArgs& a, int ctas) {
  return std::min(ctas - 1, std::max(1, (int)((int64_t)ctas * a.heads / (a.heads + a.kv_heads))));
}

// A token's side is one warp's work, or shared by several while tokens alone leave the
// SMs without kWarpsPerSm warps each.
constexpr int kWarpsPerSm = 32;
template <class T, int HD, bool BWD> cudaError_t launch_vec(const QkNormArgs& a, cudaStream_t s, int* parts, int* part_q) {
  using V = VT<T, HD, BWD>;
  const int gq = (a.heads + V::RPW - 1) / V::RPW, gk = (a.kv_heads + V::RPW - 1) / V::RPW;
  const int64_t tokens = std::max<int64_t>(1, a.tokens);
  const int64_t want = ((int64_t)a.sm_count * kWarpsPerSm + tokens - 1) / tokens;  // warps a token
  const auto share = [&](int g) { return (int)std::max<int64_t>(1, std::min<int64_t>(g, (want * g + gq + gk - 1) / (gq + gk))); };
  const int sq = share(gq), sk = share(gk);
  const auto ctas = [&](int heads, int slices) { return heads ? (tokens * slices + kWarpsPerCta - 1) / kWarpsPerCta : 1; };
  int64_t cq = ctas(a.heads, sq), ck = ctas(a.kv_heads, sk);
  if (cq + ck > kQkNormParts && BWD) {  // a partial row of the gamma gradients for each CTA
    cq = queries_part(a, kQkNormParts);
    ck = kQkNormParts - cq;
  }
  *part_q = (int)cq;
  *parts = (int)(cq + ck);
  return launch_pdl(qk_norm_vec_kernel<T, HD, BWD>, dim3((unsigned)*parts), dim3(kWarpsPerCta * 32),
                    BWD ? (size_t)kWarpsPerCta * HD * sizeof(float) : 0, s, a, *part_q, sq, sk);
}
template <bool BWD> cudaError_t launch_vec_any(const QkNormArgs& a, cudaStream_t s, int* parts, int* part_q) {
  const auto go = [&](auto t) {
    using T = decltype(t);
    switch (a.head_dim) {
    case 64: return launch_vec<T, 64, BWD>(a, s, parts, part_q);
    case 128: return launch_vec<T, 128, BWD>(a, s, parts, part_q);
    default: return launch_vec<T, 256, BWD>(a, s, parts, part_q);
    }
  };
  return a.is_bf16 ? go(__nv_bfloat16{}) : go(float{});
}

}  // namespace

size_t qk_norm_workspace_bytes(int head_dim) { return (size_t)kQkNormParts * head_dim * sizeof(float); }

cudaError_t qk_norm_forward(const QkNormArgs& a, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  if (rows == 0) return cudaSuccess;
  int parts = 0, part_q = 0;
  if (vec_ok(a, false)) return launch_vec_any<false>(a, s, &parts, &part_q);
  const int grid = (int)std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, (int64_t)a.sm_count * 64);
  return a.is_bf16 ? launch_pdl(qk_norm_rows_kernel<__nv_bfloat16>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a)
                   : launch_pdl(qk_norm_rows_kernel<float>, dim3(grid), dim3(kWarpsPerCta * 32), 0, s, a);
}

cudaError_t qk_norm_backward(const QkNormArgs& a, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.heads + a.kv_heads);
  int parts = 0, part_q = 0;
  cudaError_t e;
  if (vec_ok(a, true)) {
    e = launch_vec_any<true>(a, s, &parts, &part_q);
  } else {
    parts = (int)std::max<int64_t>(2, std::min<int64_t>((rows + kWarpsPerCta - 1) / kWarpsPerCta, kQkNormParts));
    part_q = queries_part(a, parts);
    const size_t smem = (size_t)kWarpsPerCta * a.head_dim * sizeof(float);
    e = a.is_bf16 ? launch_pdl(qk_norm_rows_bwd_kernel<__nv_bfloat16>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a, part_q)
                  : launch_pdl(qk_norm_rows_bwd_kernel<float>, dim3(parts), dim3(kWarpsPerCta * 32), smem, s, a, part_q);
  }
  if (e != cudaSuccess || (!a.dq_gamma && !a.dk_gamma)) return e;
  return launch_pdl(dgamma_kernel, dim3((a.head_dim + 31) / 32, 2), dim3(1024), 0, s, (const float*)a.partial, part_q, parts,
                    a.head_dim, a.dq_gamma, a.dk_gamma);
}

}  // namespace wv
