// The paged KV cache in E4M3: appending tokens, and attention over it for every shape
// the tensor-core kernel (kv8_attn.cu) does not take.
//
// Pools hold pages of 64 tokens, codes [page][kv_head][64][head_dim], and one scale
// for each block of 16 tokens, [page][kv_head][4]; a value is code * scale. A scale is
// the smallest power of two s >= 2^-64 with amax / s <= 448, so dividing by it and
// changing it later are exact as long as the code stays normal: a block that gains
// tokens with larger values takes the larger scale and its held codes are rewritten.
// (A scale that is not a power of two would round the held codes once more each time.)
// Per-token accuracy is that of E4M3, a relative 2^-4 for every value above 2^-13 of
// the block's largest (the scaled maximum lies above 224, the smallest normal code is
// 2^-6). A block that is given a value which is not finite gets a NaN
// scale and reads as NaN until it is begun anew; its codes stay finite, so that a
// masked token never reaches an output through 0 * NaN.
// ctx_len[b] counts the new tokens: those of sequence b are at positions
// [ctx_len - n_b, ctx_len), n_b = seq_lens ? seq_lens[b] : seq.
// No reference counterpart (it has no KV cache).
#include "kv8.cuh"

#include <algorithm>

namespace wv {
namespace {

WV_DEV float block_max(float v, float* tmp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();  // tmp may still be read by the previous call
  if (lane_id() == 0) tmp[warp_id()] = v;
  __syncthreads();
  v = tmp[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = fmaxf(v, tmp[w]);
  return v;
}

// ------------------------------------------------------------------- append
// One CTA per (block of a sequence, KV head, K or V): any even head_dim and stride.
// Rotated keys are computed twice (once for the maximum), with the products and the
// sum rounded one by one so that a key is the same code on every path. Bound by the issue
// of its two-byte accesses: 476 us for 4 x 4096 tokens of 32 heads of 128 (73 us below),
// 3.5 us for one token each of 64 sequences (2.8).
__global__ void __launch_bounds__(128) kv8_append_kernel(const Kv8AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float tmp[4];
  const int b = blockIdx.z, hd = a.c.head_dim, half = hd / 2;
  const bool is_v = (blockIdx.y & 1) != 0;
  const int kh = (int)(blockIdx.y >> 1);
  const int n = kv8_new(a.seq_lens, b, a.seq), ctx = a.c.ctx_len[b], start = ctx - n;
  const int first = max(start, 0);  // new tokens before position 0 do not exist
  const int blk = first / kKv8Block + (int)blockIdx.x;
  const int p0 = blk * kKv8Block, lo = max(first, p0), hi = min(ctx, p0 + kKv8Block);
  if (lo >= hi) return;
  const int page = kv8_page(a.c, b, blk / kKv8Subs, a.err);
  if (page < 0) return;
  const size_t ph = (size_t)page * a.c.kv_heads + kh;
  uint8_t* codes = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + (ph * kKv8Page + p0 % kKv8Page) * hd;
  float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + ph * kKv8Subs + blk % kKv8Subs;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_v ? a.v : a.k) + (size_t)kh * hd;
  const int ld = is_v ? a.ldv : a.ldk;

  auto pair = [&](int idx) -> float2 {  // values i and i + half of token lo + idx / half
    const int p = lo + idx / half, i = idx % half;
    const __nv_bfloat16* x = src + ((size_t)b * a.seq + (p - start)) * ld;
    const float u = __bfloat162float(x[i]), w = __bfloat162float(x[half + i]);
    if (is_v || !a.rope) return make_float2(u, w);
    if (p >= a.max_pos) {
      if (a.err) atomicCAS(a.err, 0u, kErrRopePos);
      return make_float2(u, w);
    }
    const float2 c = a.rope[(size_t)p * half + i];
    return make_float2(__fsub_rn(__fmul_rn(u, c.x), __fmul_rn(w, c.y)), __fadd_rn(__fmul_rn(u, c.y), __fmul_rn(w, c.x)));
  };
  float amax = 0.f;
  for (int idx = threadIdx.x; idx < (hi - lo) * half; idx += blockDim.x) {
    const float2 x = pair(idx);
    const float m = fmaxf(fabsf(x.x), fabsf(x.y));
    amax = fmaxf(amax, x.x - x.x == 0.f && x.y - x.y == 0.f ? m : INFINITY);  // NaN counts as infinite
  }
  amax = block_max(amax, tmp);
  const float s_old = lo > p0 ? *scale : 0.f;
  const bool poison = amax == INFINITY || s_old != s_old;
  const float s = poison ? __uint_as_float(0x7fc00000u) : fmaxf(kv8_scale(amax), s_old);
  for (int idx = threadIdx.x; idx < (hi - lo) * half; idx += blockDim.x) {
    const float2 x = poison ? make_float2(0.f, 0.f) : pair(idx);
    const uint32_t c = poison ? 0u : e4m3x2(x.x / s, x.y / s);
    uint8_t* row = codes + (size_t)(lo - p0 + idx / half) * hd + idx % half;
    row[0] = (uint8_t)c;
    row[half] = (uint8_t)(c >> 8);
  }
  if (lo > p0 && !poison && s != s_old)
    for (int i = threadIdx.x; i < (lo - p0) * hd; i += blockDim.x)
      codes[i] = (uint8_t)e4m3x2(e4m3_value(codes[i]) * s_old / s, 0.f);
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = s;
}

// The largest magnitude of three values, NaN if one is NaN.
WV_DEV float abs_max(float x, float y, float z) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// e4m3x2(lo f, hi f), both products in one instruction.
WV_DEV uint32_t e4m3x2_scaled(float lo, float hi, float f) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(lo), "+f"(hi) : "f"(f));
  return e4m3x2(lo, hi);
}

// head_dim 64 and 128, 16-byte aligned rows, codes and table: one warp per (block, KV
// head, K or V) holds the block's 16 rows in registers, 8 pairs of a row per lane (16
// bytes of each half, the partners of the rotation together), so the rows are read
// once and the maximum needs five shuffles. Bound by HBM for prompts (4 bytes read, 2
// written a value pair of K and V), by latency for single tokens.
// CTAs of 4 heads, 24 warps to an SM: 4 x 4096 tokens x 32 KV heads of 128 take 73 us
// (5.4 TB/s of 403 MB); 8 heads 80 us, 2 heads 107 us, 20 warps without the bound on
// registers 87 us; values without a rotation 64 us (all in a CUDA graph; a call on a
// stream takes 79 us).
constexpr int kAppendWarps = 4;
template <int HD>
__global__ void __launch_bounds__(kAppendWarps * 32, 6) kv8_append_vec_kernel(const Kv8AppendArgs a, int blocks) {
  constexpr int LPR = HD / 16, RPW = 32 / LPR, IT = kKv8Block / RPW;
  constexpr int F4 = HD / 4;  // 16-byte pieces of a row of the table, two pairs each
  __shared__ float4 tab[kKv8Block * F4];
  pdl_wait();
  pdl_trigger();
  const int lane = (int)lane_id(), sub = lane / LPR, at = (lane % LPR) * 8;
  const int groups = (a.c.kv_heads + (int)(blockDim.x >> 5) - 1) / (int)(blockDim.x >> 5);
  int unit = (int)blockIdx.x / groups;
  const int kh = ((int)blockIdx.x % groups) * (int)(blockDim.x >> 5) + (int)warp_id();
  const bool is_v = (unit & 1) != 0;
  unit >>= 1;
  const int b = unit / blocks;
  const int n = kv8_new(a.seq_lens, b, a.seq), ctx = a.c.ctx_len[b], start = ctx - n;
  const int first = max(start, 0), blk = first / kKv8Block + unit % blocks;
  const int p0 = blk * kKv8Block, lo = max(first, p0), hi = min(ctx, p0 + kKv8Block);
  if (lo >= hi) return;
  const int ld = is_v ? a.ldv : a.ldk;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_v ? a.v : a.k) + (size_t)kh * HD + at;
  uint4 raw[IT][2];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int p = p0 + it * RPW + sub;
    raw[it][0] = raw[it][1] = make_uint4(0u, 0u, 0u, 0u);
    if (p < lo || p >= hi || kh >= a.c.kv_heads) continue;
    const __nv_bfloat16* x = src + ((size_t)b * a.seq + (p - start)) * ld;
    raw[it][0] = *reinterpret_cast<const uint4*>(x);
    raw[it][1] = *reinterpret_cast<const uint4*>(x + HD / 2);
  }
  // A lane's eight pairs are four pieces of the table, 64 bytes apart between lanes: read
  // from global memory that is four times the wavefronts. The CTA's heads share the
  // block's rows of it in shared memory, pieces swapped so that no bank meets another.
  const bool rotate = !is_v && a.rope;
  if (rotate) {
    const float4* src4 = reinterpret_cast<const float4*>(a.rope);
    for (int i = (lo - p0) * F4 + (int)threadIdx.x; i < (hi - p0) * F4; i += (int)blockDim.x) {
      const int p = p0 + i / F4;
      if (p < a.max_pos)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&tab[i ^ ((i >> 3) & 3)])),
                     "l"(src4 + (size_t)p * F4 + i % F4)
                     : "memory");
      else if (a.err)
        atomicCAS(a.err, 0u, kErrRopePos);
    }
  }
  const int page = kv8_page(a.c, b, blk / kKv8Subs, a.err);
  if (rotate) asm volatile("cp.async.wait_all;" ::: "memory");
  if (page < 0) return;
  __syncthreads();
  if (kh >= a.c.kv_heads) return;
  const size_t ph = (size_t)page * a.c.kv_heads + kh;
  uint8_t* codes = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + (ph * kKv8Page + p0 % kKv8Page) * HD + at;
  float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + ph * kKv8Subs + blk % kKv8Subs;
  const float s_old = lo > p0 ? *scale : 0.f;

  float x[IT][2][8], amax = 0.f;  // the largest magnitude; NaN if one is
  if (!rotate) {                  // BF16 magnitudes order as integers, NaN above all
    uint32_t top = 0u;
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        top = __vmaxu2(__vmaxu2(__vmaxu2(top, raw[it][hf].x & 0x7fff7fffu), raw[it][hf].y & 0x7fff7fffu),
                       __vmaxu2(raw[it][hf].z & 0x7fff7fffu, raw[it][hf].w & 0x7fff7fffu));
    amax = __uint_as_float(max(top & 0xffff0000u, top << 16));
  }
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int p = p0 + it * RPW + sub;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint32_t w[4] = {raw[it][hf].x, raw[it][hf].y, raw[it][hf].z, raw[it][hf].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[it][hf][2 * i] = __uint_as_float(w[i] << 16);
        x[it][hf][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    if (rotate) {
      if (p >= lo && p < hi && p < a.max_pos) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int f = (it * RPW + sub) * F4 + at / 2 + i / 2;
          const float4 c = tab[f ^ ((f >> 3) & 3)];
          const float cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float u = x[it][0][i + e], w = x[it][1][i + e];
            x[it][0][i + e] = __fsub_rn(__fmul_rn(u, cs[2 * e]), __fmul_rn(w, cs[2 * e + 1]));
            x[it][1][i + e] = __fadd_rn(__fmul_rn(u, cs[2 * e + 1]), __fmul_rn(w, cs[2 * e]));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = abs_max(amax, x[it][0][i], x[it][1][i]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = abs_max(amax, __shfl_xor_sync(0xffffffffu, amax, o), 0.f);
  const bool poison = !(amax < INFINITY) || s_old != s_old;
  const float s = poison ? __uint_as_float(0x7fc00000u) : fmaxf(kv8_scale(amax), s_old);
  // s is a power of two between 2^-64 and 2^120 (or the caller's own larger scale):
  // multiplying by 1/s is dividing by s.
  const float inv = 1.f / s;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int r = it * RPW + sub, p = p0 + r;
    if (p < lo || p >= hi) continue;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint32_t c[4] = {};
      if (!poison) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = e4m3x2_scaled(x[it][hf][2 * i], x[it][hf][2 * i + 1], inv);
      }
      *reinterpret_cast<uint2*>(codes + (size_t)r * HD + hf * (HD / 2)) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
    }
  }
  if (lo > p0) {
    if (!poison && s != s_old) {  // the held codes move to the larger scale
      const float f = s_old * inv;
      for (int r = sub; r < lo - p0; r += RPW)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint2* q = reinterpret_cast<uint2*>(codes + (size_t)r * HD + hf * (HD / 2));
          const uint32_t w[2] = {q->x, q->y};
          uint32_t o[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 y = e4m3x2_value(w[i] & 0xffffu), z = e4m3x2_value(w[i] >> 16);
            o[i] = e4m3x2(y.x * f, y.y * f) | (e4m3x2(z.x * f, z.y * f) << 16);
          }
          *q = make_uint2(o[0], o[1]);
        }
    }
    __syncwarp();  // every lane has read the old scale
  }
  if (lane == 0) *scale = s;
}

// --------------------------------------------------------- attention, any shape
constexpr int kGenWarps = 4;

// One CTA per (query row, head): warp w takes the 32-key groups w, w + 4, ... of the
// row's keys, a lane per key for the scores and a lane per dimension for the values,
// with a running maximum and sum; the warps merge in shared memory, in warp order. Bound
// by instructions, and a KV head is read once for each of its query heads: 64 x 4096
// tokens, 32 heads over 8 of 64, take 1605 us (46 on the tensor cores).
template <bool ALIBI>
__global__ void __launch_bounds__(kGenWarps * 32) kv8_attn_rows_kernel(const Kv8AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int kDims = kKv8MaxHeadDim / 32;
  __shared__ float qs[kKv8MaxHeadDim];
  __shared__ float mw[kGenWarps], lw[kGenWarps], ow[kGenWarps][kKv8MaxHeadDim];
  const int hd = a.c.head_dim, warp = (int)warp_id(), lane = (int)lane_id();
  const int h = blockIdx.x % a.heads, t = blockIdx.x / a.heads, b = blockIdx.z;
  const int kh = h / (a.heads / a.c.kv_heads);
  const int n = kv8_new(a.seq_lens, b, a.seq), ctx = a.c.ctx_len[b];
  const int qpos = ctx - n + t;
  const size_t row = (size_t)b * a.seq + t;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + row * a.ldo + (size_t)h * hd;
  if (t >= n || qpos < 0) {  // no such token: a row that sees nothing
    for (int d = threadIdx.x; d < hd; d += blockDim.x) out[d] = __float2bfloat16_rn(0.f);
    return;
  }
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + row * a.ldq + (size_t)h * hd;
  for (int d = threadIdx.x; d < hd; d += blockDim.x) qs[d] = __bfloat162float(q[d]);
  __syncthreads();
  const int most = a.c.max_pages * kKv8Page;  // a length past the table is recorded and cut there
  if (qpos >= most && threadIdx.x == 0 && a.err) atomicCAS(a.err, 0u, kErrKvPage);
  const int k1 = min(qpos, most - 1) + 1, k0 = a.window > 0 ? max(0, qpos - a.window + 1) : 0;
  const float sl = a.scale * 1.4426950408889634f;
  const float slope = ALIBI ? exp2f(-(float)(a.head_base + h + 1) * 8.0f / (float)a.total_heads) * 1.4426950408889634f : 0.f;
  float m = -INFINITY, l = 0.f, o[kDims] = {};
  const int groups = (k1 + 31) / 32;
  for (int g = k0 / 32 + warp; g < groups; g += kGenWarps) {
    const int page = kv8_page(a.c, b, g * 32 / kKv8Page, a.err);
    if (page < 0) continue;
    const size_t ph = (size_t)page * a.c.kv_heads + kh;
    const int key = g * 32 + lane, slot = key % kKv8Page;
    const bool on = key >= k0 && key < k1;
    const uint8_t* kr = static_cast<const uint8_t*>(a.c.k) + (ph * kKv8Page + slot) * hd;
    float x = -INFINITY;
    if (on) {
      float s = 0.f;
      for (int d = 0; d < hd; ++d) s += qs[d] * e4m3_value(kr[d]);
      x = s * a.c.k_scale[ph * kKv8Subs + slot / kKv8Block] * sl;
      if (ALIBI) x -= slope * (float)(qpos - key);
    }
    float mx = x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    const float mnew = fmaxf(m, mx);
    const float corr = m == -INFINITY ? 0.f : exp2f(m - mnew);
    float p = on ? exp2f(x - mnew) : 0.f;
    l = l * corr + p;
#pragma unroll
    for (int j = 0; j < kDims; ++j) o[j] *= corr;
    m = mnew;
    p = on ? p * a.c.v_scale[ph * kKv8Subs + slot / kKv8Block] : 0.f;
    const uint8_t* vp = static_cast<const uint8_t*>(a.c.v) + (ph * kKv8Page + g * 32 % kKv8Page) * hd;
    for (int kk = 0; kk < 32; ++kk) {
      const float pk = __shfl_sync(0xffffffffu, p, kk);
      if (g * 32 + kk < k0 || g * 32 + kk >= k1) continue;  // rows there may hold anything
#pragma unroll
      for (int j = 0; j < kDims; ++j)
        if (lane + 32 * j < hd) o[j] += pk * e4m3_value(vp[(size_t)kk * hd + lane + 32 * j]);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (lane == 0) {
    mw[warp] = m;
    lw[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < kDims; ++j)
    if (lane + 32 * j < hd) ow[warp][lane + 32 * j] = o[j];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < kGenWarps; ++w) M = fmaxf(M, mw[w]);
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    float num = 0.f, den = 0.f;
    for (int w = 0; w < kGenWarps; ++w) {
      // a warp without a key has l = 0; one whose scores are all NaN has l = NaN
      const float f = mw[w] == -INFINITY ? 1.f : exp2f(mw[w] - M);
      num += f * ow[w][d];
      den += f * lw[w];
    }
    out[d] = __float2bfloat16_rn(den == 0.f ? 0.f : num / den);
  }
}

}  // namespace

cudaError_t kv8_append(const Kv8AppendArgs& a, cudaStream_t s) {
  // blocks that seq tokens can touch, wherever they begin
  const int blocks = (a.seq + kKv8Block - 2) / kKv8Block + 1;
  const auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; };
  const int warps = std::min(a.c.kv_heads, kAppendWarps);
  const int64_t ctas = (int64_t)blocks * 2 * a.batch * ((a.c.kv_heads + warps - 1) / warps);
  if ((a.c.head_dim == 64 || a.c.head_dim == 128) && a.ldk % 8 == 0 && a.ldv % 8 == 0 && !low(a.k) && !low(a.v) &&
      !low(a.c.k) && !low(a.c.v) && !low(a.rope) && ctas < (1ll << 31))
    return launch_pdl(a.c.head_dim == 64 ? kv8_append_vec_kernel<64> : kv8_append_vec_kernel<128>, dim3((unsigned)ctas),
                      dim3(warps * 32), 0, s, a, blocks);
  return launch_pdl(kv8_append_kernel, dim3(blocks, 2 * a.c.kv_heads, a.batch), dim3(128), 0, s, a);
}

cudaError_t kv8_attention(const Kv8AttnArgs& a, cudaStream_t s) {
  if (kv8_attention_tc_supported(a)) return kv8_attention_tc(a, s);
  const dim3 grid((unsigned)a.seq * a.heads, 1, a.batch);
  return a.alibi ? launch_pdl(kv8_attn_rows_kernel<true>, grid, dim3(kGenWarps * 32), 0, s, a)
                 : launch_pdl(kv8_attn_rows_kernel<false>, grid, dim3(kGenWarps * 32), 0, s, a);
}

}  // namespace wv
