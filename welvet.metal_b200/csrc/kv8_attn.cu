// Attention over the paged E4M3 KV cache on the 5th-generation tensor cores: head_dim
// 64 and 128, from one new token per sequence to prompt chunks.
//
// The codes are never widened. With the keys as the 128-row operand, both products run
// as FP8 UMMAs on the tiles as TMA brings them from the pages:
//   S^T [128 keys, columns] = K [128 keys, hd] (A, E4M3, K-major) * Q^T
//   O^T [hd, columns]      += V^T (A, E4M3, MN-major: the same [key][hd] bytes) * P^T
// A column is one (new token, query head of the KV group); RT of them share a CTA's
// pass over the keys, so a decode step needs a 16-column MMA and no padding of queries
// to 128 rows, and a thread of the softmax holds one key of every column: no work is
// spent on absent queries, and no row reductions across lanes are needed per tile.
// What the small operands lose in 8 bits is kept in more of them:
//   * a query row, scaled by a power of two so that its largest value lies in (224, 448],
//     is a sum of two E4M3 codes: a BF16 query has 8 bits, the codes 4 each, and only the
//     smallest step of a code, 2^-9, cuts. Off by at most 2^-10, which is 2^-17 of the
//     row's largest value;
//   * a probability, rounded to FP16, is hi + lo/8 + lo2/64 in E5M2 codes (3 significant
//     bits each, rounded to nearest in turn): a relative 2^-9 down to 2^-19 of the
//     largest, and 2^-28 of the largest below that, so that long tails of small
//     probabilities still add up. E4M3 codes would be finer but end at 2^-14. The row's
//     sum takes the probabilities before this rounding, so a row that one key rules is off
//     by up to 2^-9 as a whole, less than half a place of its BF16 output.
// The codes of one sum are columns side by side (2 RT of S, 3 RT of O), added when
// read: a 128-row MMA of 32 bytes takes about 60 cycles for any N up to 128, so one
// wide MMA is cheaper than several narrow ones into the same columns.
// Scores and sums are FP32 (TMEM accumulators, registers).
//
// Softmax in the log2 domain with the value scale folded in: z = s kscale qscale
// scale log2e + log2(vscale), p = 2^(z - ref), O += p * code, l += p / vscale (FP32: the
// scales of a row's blocks may lie 2^100 apart). ref is a column's running maximum of z,
// raised only when it is exceeded by more than 2^10 (E5M2 has the room), so that after the
// first tile one vote and no maximum is the rule; when it moves, O and l are rescaled.
// (Room of 2^3 and remainders that need no factor of 8 are 16 instructions fewer but move
// references more often: 625 us against 574, at the time, for the prompt piece below.)
//
// Roles: softmax warpgroups (thread = TMEM lane = key; each takes CPW of the columns), a
// TMA warp (pages of codes and their four scales into rings of 128-key tiles), an MMA
// warp (S_0, S_1, then PV_i with S_{i+2}; S and P double-buffered). Keys and values have
// rings of their own: a key tile is free as soon as its S is done, two tiles before its
// values are, so equal rings leave each three tiles of time to load (one ring of both
// left a load one tile: 1.1 against 0.6 k cycles a tile).
// A long context is split over a cluster of up to 16 CTAs whose partial (ref, l, O)
// are joined through distributed shared memory in rank order: no workspace, no second
// launch, the same bits every time. An unsplit one goes from TMEM to the output.
//
// Measured, in a CUDA graph (calls on a stream take 3 to 4 % more). 32 sequences of 8192 tokens, 32 KV heads of 128: 305-320 us, 6.7-7.0 TB/s of
// codes and scales; 64 of 4096, 8 KV heads of 64 for 32 heads: 46 us, 5.3 TB/s; 5 tokens
// each for 8 sequences in a window of 8192, 8 KV heads of 128: 34-38 us, 3.6-4 TB/s (6.3
// in the loop, the rest is the first tile's chain of lengths, page ids, copies, MMA and
// softmax, and the joining); 2048 tokens over 10001, 32 heads of 128: 555 us, 543
// TFLOP/s. The first three are bound by HBM; the last by the issue of the softmax in this
// layout, about 300 instructions a warp and tile of 16 columns (the tensor pipe is 30 %
// busy). The layout is for few query rows; a prompt piece has thousands a KV head, and
// query rows as the 128-row operand over tiles widened to BF16 have not been tried.
// Masked keys and rows past the context: their p is set to 0 and their V rows cleared
// (a byte never written may be a NaN code); NaN scales reach only columns that see them.
#include "attn_common.cuh"
#include "kv8.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

namespace wv {
namespace {

constexpr int kKeys = 128;          // keys of a tile: two pages
constexpr float kBias = 5.f;        // log2 of p at the reference
constexpr float kSlack = 10.f;      // z may exceed the reference by this much (p <= 2^15)
constexpr float kNoRef = 1e30f;     // bias - ref of a column that has seen no key, when joining
constexpr int kMaxCluster = 16;

// Column groups of a tile: softmax warps hide the latency of each other's chains (TMEM
// load, exponentials, conversions, stores) while registers last. 16 columns a thread: 574
// us for the prompt piece above and 34 for the verification step, with 32: 599 and 39.
// (Two sets of warpgroups on alternate tiles, each with an O of its own, took the same
// times as one.)
template <int HD, int RT> struct KT {
  static constexpr int NCG = RT == 64 ? 4 : RT == 32 ? 2 : 1;
  static constexpr int CPW = RT / NCG;              // columns of a warpgroup
  static constexpr int SOFT_WARPS = NCG * 4;
  static constexpr int THREADS = SOFT_WARPS * 32 + 64;
  static constexpr int TILE = kKeys * HD;           // bytes of a K or V tile
  static constexpr int NS = 2 * RT;                 // query rows: hi | lo
  // Columns of S: hi | lo, from one MMA, added in registers; with 64 columns hi + lo, from
  // two MMAs into one accumulator (there the softmax bounds, not the MMAs).
  static constexpr bool SUM = RT == 64;
  static constexpr int SC = SUM ? RT : NS;
  static constexpr int NO = RT == 8 ? 32 : 3 * RT;  // columns of O and P: three terms
  static constexpr int O_COL = 2 * SC;              // TMEM: S_0 | S_1 | O
  static constexpr int COLS = O_COL + NO;
  static constexpr int TMEM = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  // tiles of the K and of the V ring
  static constexpr int KST = HD == 128 ? (RT == 32 ? 5 : 3) : (RT == 64 ? 7 : RT == 8 ? 3 : 4);
  static constexpr int VST = (HD == 64 && RT == 8) || (HD == 128 && RT == 16) ? KST - 1 : KST;
  static constexpr int SCALES = KST + 2;  // scales outlive their key tile by two tiles
  static constexpr int P_BYTES = kKeys * NO;
  static constexpr int Q_BYTES = NS * HD;
  static constexpr int OFF_V = KST * TILE;
  static constexpr int OFF_P = OFF_V + VST * TILE;
  static constexpr int OFF_Q = OFF_P + 2 * P_BYTES;
  static constexpr int OFF_IN = OFF_Q + Q_BYTES;          // joining: [split][RT HD / splits] partial O
  static constexpr int OFF_INL = OFF_IN + RT * HD * 4;    // ... and (reference, sum) of their columns
  static constexpr int OFF_SC = OFF_INL + 8 * (RT > 16 ? RT : 16);  // scales: [slot][K, V][8]
  static constexpr int OFF_OUT = OFF_SC + SCALES * 64;    // output element of a column (64 bits), -1: none
  static constexpr int OFF_QF = OFF_OUT + RT * 8;         // factor of a column's scores
  static constexpr int OFF_REF = OFF_QF + RT * 4;         // bias - reference
  static constexpr int OFF_FAC = OFF_REF + RT * 4;  // rescaling factors
  static constexpr int OFF_HAVE = OFF_FAC + RT * 4; // whether a column has seen a key
  static constexpr int OFF_L = OFF_HAVE + RT * 4;   // sums
  static constexpr int OFF_QHI = OFF_L + RT * 4;    // last key of a column
  static constexpr int OFF_SLOPE = OFF_QHI + RT * 4;
  static constexpr int OFF_RED = OFF_SLOPE + RT * 4;      // [4 warps][RT]
  static constexpr int OFF_BAR = OFF_RED + 4 * RT * 4;
  static constexpr int SMEM = 1024 + OFF_BAR + 8 * (2 * (KST + VST) + SCALES + 7) + 32;
  // resident CTAs of an SM
  static constexpr int BY_SMEM = 228 * 1024 / (SMEM + 1024), BY_TMEM = 512 / TMEM;
  static constexpr int PER_SM = BY_SMEM < BY_TMEM ? BY_SMEM : BY_TMEM;
  // A CTA that waits for TMEM columns while its cluster waits for it could wait for a
  // CTA of another stream in the same state. Shared memory rules that out: CTAs of these
  // kernels that fit an SM together never need more than its 512 columns (128 columns
  // take at least 1/4 of it, 256 columns 1/2 with what is left over too small for a
  // third CTA, 512 all but what is too small for one).
  static_assert(SMEM > 50 * 1024 && (TMEM < 256 || SMEM > 91 * 1024) && (TMEM < 512 || SMEM > 178 * 1024) &&
                    (TMEM < 256 || PER_SM <= 2), "TMEM columns of co-resident CTAs");
  static_assert(COLS <= TMEM, "TMEM columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// D[tmem] (+)= A[smem] B[smem]^T with 8-bit operands; descriptors as 32-bit halves.
WV_DEV void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                    uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// High descriptor word: stride byte offset, version 1, layout type (0 none, 2 128-byte,
// 4 64-byte swizzle).
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo_bytes, uint32_t layout) {
  return ((sbo_bytes >> 4) & 0x3FFFu) | (1u << 14) | (layout << 29);
}
// Instruction descriptor of kind::f8f6f4, FP32 accumulators; formats: 0 E4M3, 1 E5M2.
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t a_fmt, uint32_t b_fmt, int M, int N, uint32_t a_mn, uint32_t b_mn) {
  return (1u << 4) | (a_fmt << 7) | (b_fmt << 10) | (a_mn << 15) | (b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// N consecutive TMEM columns of this thread's lane.
template <int N> WV_DEV void tmem_ld(uint32_t addr, uint32_t* r) {
  if constexpr (N == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
  } else if constexpr (N == 16) {
    tmem_ld16(addr, *reinterpret_cast<uint32_t(*)[16]>(r));
  } else {
    tmem_ld32(addr, *reinterpret_cast<uint32_t(*)[32]>(r));
  }
}
template <int N> WV_DEV void tmem_st(uint32_t addr, const uint32_t* r) {
  if constexpr (N == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else if constexpr (N == 16) {
    tmem_st16(addr, *reinterpret_cast<const uint32_t(*)[16]>(r));
  } else {
    tmem_st32(addr, *reinterpret_cast<const uint32_t(*)[32]>(r));
  }
}
// Shared-memory loads and stores by 32-bit address (a generic access costs an address
// in 64 bits and a longer path).
WV_DEV float lds(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
WV_DEV float4 lds4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
WV_DEV void sts(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
WV_DEV void sts4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Maximum over the warp; NaN lanes are left out.
WV_DEV float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Barrier of a warpgroup that also says whether any thread's predicate holds.
template <int ID> WV_DEV bool bar_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(ID)
      : "memory");
  return r != 0;
}
template <int ID> WV_DEV void bar_sync() { asm volatile("barrier.cta.sync %0, 128;" ::"n"(ID) : "memory"); }
// ... of warpgroup w of N (barrier 0 is the CTA's; numbers known to the compiler, since a
// barrier by register made the prompt piece above take 563 us instead of 557).
template <int N> WV_DEV bool wg_any(int w, bool v) {
  if (N == 1 || w == 0) return bar_any<1>(v);
  if (N == 2 || w == 1) return bar_any<2>(v);
  return w == 2 ? bar_any<3>(v) : bar_any<4>(v);
}
template <int N> WV_DEV void wg_sync(int w) {
  if (N == 1 || w == 0) bar_sync<1>();
  else if (N == 2 || w == 1) bar_sync<2>();
  else if (w == 2) bar_sync<3>();
  else bar_sync<4>();
}
// The softmax warps wait for the MMA warp's part of the columns' values.
template <int WARPS> WV_DEV void cols_sync() { asm volatile("barrier.cta.sync 5, %0;" ::"n"(WARPS * 32) : "memory"); }
template <int WARPS> WV_DEV void cols_arrive() { asm volatile("barrier.cta.arrive 5, %0;" ::"n"(WARPS * 32) : "memory"); }
// Two FP16 pairs to four E5M2 codes (nearest), and the FP16 values of codes 0, 1 and 2,
// 3 of a word: an E5M2 code is the upper byte of the FP16 pattern of its value.
WV_DEV uint32_t e5m2x4(__half2 u, __half2 w) {
  uint32_t r;
  asm("{\n\t.reg .b16 t, v;\n\t"
      "cvt.rn.satfinite.e5m2x2.f16x2 t, %1;\n\t"
      "cvt.rn.satfinite.e5m2x2.f16x2 v, %2;\n\t"
      "mov.b32 %0, {t, v};\n\t}"
      : "=r"(r)
      : "r"(*reinterpret_cast<uint32_t*>(&u)), "r"(*reinterpret_cast<uint32_t*>(&w)));
  return r;
}
WV_DEV __half2 e5m2_lo(uint32_t c) {
  const uint32_t h = __byte_perm(c, 0u, 0x1404);
  return *reinterpret_cast<const __half2*>(&h);
}
WV_DEV __half2 e5m2_hi(uint32_t c) {
  const uint32_t h = __byte_perm(c, 0u, 0x3424);
  return *reinterpret_cast<const __half2*>(&h);
}
WV_DEV uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
WV_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
WV_DEV uint32_t peer_addr(const void* local, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
WV_DEV void st_peer(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
WV_DEV void st_peer2(uint32_t addr, float v, float w) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v), "f"(w) : "memory");
}
// The two halves of cluster_sync.
WV_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
WV_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <int HD, int RT, bool ALIBI>
__global__ void __launch_bounds__(KT<HD, RT>::THREADS, KT<HD, RT>::PER_SM)
    kv8_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const Kv8AttnArgs a, int splits) {
  using T = KT<HD, RT>;
  constexpr int CPW = T::CPW, KST = T::KST, VST = T::VST, NCG = T::NCG, kSoftWarps = T::SOFT_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + T::OFF_BAR);
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;
  uint64_t* v_empty = v_full + VST;
  uint64_t* sc_full = v_empty + VST;  // [SCALES] a tile's scales
  uint64_t* s_full = sc_full + T::SCALES;  // [2]
  uint64_t* p_full = s_full + 2;  // [2]
  uint64_t* pv_done = p_full + 2; // [2]
  uint64_t* q_full = pv_done + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(q_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int64_t* outs = reinterpret_cast<int64_t*>(smem + T::OFF_OUT);
  float* qf = reinterpret_cast<float*>(smem + T::OFF_QF);
  float* refs = reinterpret_cast<float*>(smem + T::OFF_REF);
  float* facs = reinterpret_cast<float*>(smem + T::OFF_FAC);
  float* haves = reinterpret_cast<float*>(smem + T::OFF_HAVE);
  float* lsum = reinterpret_cast<float*>(smem + T::OFF_L);
  int* qhi = reinterpret_cast<int*>(smem + T::OFF_QHI);
  float* slope = reinterpret_cast<float*>(smem + T::OFF_SLOPE);
  const int warp = (int)warp_id(), lane = (int)lane_id();

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * (KST + VST) + T::SCALES; ++s) mbar_init(&k_full[s], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], NCG * 4);  // the warps that share a tile
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, kSoftWarps);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kSoftWarps) {
    tmem_alloc(tmem_holder, T::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();  // the append (or whatever filled the cache, q and the lengths) is complete
  pdl_trigger();  // behind the TMEM allocation: a dependent's CTA must not take the columns first
  if (splits > 1) cluster_arrive();  // waited for before the first access to another CTA

  // ---- this CTA's columns and keys; its query rows are requested with the lengths
  const int split = blockIdx.x % splits, b = blockIdx.z;
  const int kh = blockIdx.y, r0 = (int)(blockIdx.x / splits) * RT;
  const int G = a.heads / a.c.kv_heads;
  // Eight lanes a column, QD dims each: 4 columns a warp.
  constexpr int QD = HD / 8;
  static_assert(RT <= kSoftWarps * 4, "columns of the softmax warps");
  uint32_t xq[QD / 2];
  const int qc = warp * 4 + lane / 8, qd = lane % 8 * QD;
  int tq = 0;  // the column's token
  if (warp < kSoftWarps) {
    tq = (r0 + qc) / G;
    const uint16_t* x = static_cast<const uint16_t*>(a.q) + ((int64_t)b * a.seq + tq) * a.ldq +
                        (int64_t)(kh * G + (r0 + qc) - tq * G) * HD + qd;
#pragma unroll
    for (int i = 0; i < QD / 2; ++i) xq[i] = 0u;
    if (qc < RT && tq < a.seq) {
      if (reinterpret_cast<uintptr_t>(x) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < QD / 2; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(x + 2 * i);
          xq[i] = v.x;
          xq[i + 1] = v.y;
          xq[i + 2] = v.z;
          xq[i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < QD / 2; ++i) xq[i] = x[2 * i] | (uint32_t)x[2 * i + 1] << 16;
      }
    }
  }
  const int n = kv8_new(a.seq_lens, b, a.seq);
  const int shift = a.c.ctx_len[b] - n;  // position of the first new token
  const int t0 = max(r0 / G, max(0, -shift)), t1 = min((r0 + RT - 1) / G, n - 1);  // live tokens
  const int qlo = shift + t0;
  int k1 = t1 >= t0 ? shift + t1 + 1 : 0;
  if (k1 > a.c.max_pages * kKv8Page) {
    if (threadIdx.x == 0) atomicCAS(a.err, 0u, kErrKvPage);
    k1 = a.c.max_pages * kKv8Page;
  }
  const int page0 = (a.window > 0 ? max(0, qlo + 1 - a.window) : 0) / kKv8Page;
  const int all = k1 > page0 * kKv8Page ? (k1 - page0 * kKv8Page + kKeys - 1) / kKeys : 0;
  const int per = (all + splits - 1) / splits;
  const int tile0 = min(all, split * per), tiles = min(all, tile0 + per) - tile0;
  const int base0 = page0 * kKv8Page + tile0 * kKeys;  // first key of tile 0
  bool ok = true;

  if (warp == kSoftWarps) {
    // ------------------------------------------------------------- TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int* bt = a.c.block_table + (size_t)b * a.c.max_pages;
    const int p0 = base0 / kKv8Page;
    const int np = tiles > 0 ? min((k1 + kKv8Page - 1) / kKv8Page - p0, 2 * tiles) : 0;  // pages of this CTA
    // Page ids 32 at a time, requested one batch ahead; V follows two tiles behind K,
    // as PV_j follows S_{j+2}.
    int next = lane < np ? bt[p0 + lane] : 0, ids = 0, held = 0;
    for (int j = 0; j < tiles + 2; ++j) {
      if (j % 16 == 0) {
        held = ids;
        ids = next;
        const int at = 2 * j + 32 + lane;
        next = at < np ? bt[p0 + at] : 0;
        if (ids < 0 || ids >= a.c.pages) {  // reported; page 0 in its place keeps every access inside
          if (2 * j + lane < np) atomicCAS(a.err, 0u, kErrKvPage);
          ids = 0;
        }
      }
      // K_j and the scales of tile j, then V_{j-2}
      const int kp[2] = {__shfl_sync(0xffffffffu, ids, (2 * j) & 31), __shfl_sync(0xffffffffu, ids, (2 * j + 1) & 31)};
      const int jv = j - 2, from = j % 16 < 2 ? held : ids;
      const int vp[2] = {__shfl_sync(0xffffffffu, from, (2 * jv) & 31), __shfl_sync(0xffffffffu, from, (2 * jv + 1) & 31)};
      if (lane == 0 && ok) {
        if (j < tiles) {
          const int s = j % KST, two = 2 * j + 1 < np ? 2 : 1;
          if (j >= KST) ok = mbar_wait(&k_empty[s], ((j / KST) & 1) ^ 1, abort_flag, a.err, kErrWaitEmpty);
          if (ok) {
            float* sc = reinterpret_cast<float*>(smem + T::OFF_SC + (j % T::SCALES) * 64);
            uint64_t* sb = &sc_full[j % T::SCALES];
            mbar_arrive_expect_tx(&k_full[s], two * kKv8Page * HD);
            mbar_arrive_expect_tx(sb, two * 32);
            for (int i = 0; i < two; ++i) {
              const int ph = kp[i] * a.c.kv_heads + kh;
              tma_load_2d(smem + s * T::TILE + i * kKv8Page * HD, &tmK, &k_full[s], 0, ph * kKv8Page);
              bulk_load(sc + i * 4, a.c.k_scale + (size_t)ph * kKv8Subs, 16, sb);
              bulk_load(sc + 8 + i * 4, a.c.v_scale + (size_t)ph * kKv8Subs, 16, sb);
            }
          }
        }
        if (jv >= 0 && ok) {
          const int s = jv % VST, two = 2 * jv + 1 < np ? 2 : 1;
          if (jv >= VST) ok = mbar_wait(&v_empty[s], ((jv / VST) & 1) ^ 1, abort_flag, a.err, kErrWaitEmpty);
          if (ok) {
            mbar_arrive_expect_tx(&v_full[s], two * kKv8Page * HD);
            for (int i = 0; i < two; ++i)
              tma_load_2d(smem + T::OFF_V + s * T::TILE + i * kKv8Page * HD, &tmV, &v_full[s], 0,
                          (vp[i] * a.c.kv_heads + kh) * kKv8Page);
          }
        }
        if (!ok) {  // the copies in flight land before the CTA ends (bounded)
          int none = 0;
          for (int k = max(0, j - KST); k < min(j, tiles); ++k) {
            mbar_wait_for(&k_full[k % KST], (k / KST) & 1, &none, a.err, kErrWaitFull, 1000000000ull);
            mbar_wait_for(&sc_full[k % T::SCALES], (k / T::SCALES) & 1, &none, a.err, kErrWaitFull, 1000000000ull);
          }
          for (int k = max(0, jv - VST); k < jv; ++k)
            mbar_wait_for(&v_full[k % VST], (k / VST) & 1, &none, a.err, kErrWaitFull, 1000000000ull);
        }
      }
    }
  } else if (warp == kSoftWarps + 1) {
    // --------------------------------------------------------------- MMA issuer
    // The whole warp walks the loop (descriptors stay warp-uniform), one lane issues.
    constexpr uint32_t kRow = HD == 128 ? 2u : 4u;  // swizzle of the code tiles
    constexpr uint32_t HI_KV = desc_hi(8 * HD, kRow);       // 8 keys of HD bytes
    constexpr uint32_t HI_Q = desc_hi(128, 0);              // 8 rows of 16 bytes
    constexpr uint32_t HI_P = desc_hi(kKeys * 16, 0);       // 16 columns of every key
    constexpr uint32_t IDESC_S = idesc_f8(0, 0, 128, T::SC, 0, 0);
    constexpr uint32_t IDESC_PV = idesc_f8(0, 1, HD, T::NO, 1, 1);
    for (int c = lane; c < RT; c += 32) {  // the columns' values, while it has nothing to issue
      const int t = (r0 + c) / G, h = kh * G + (r0 + c) - t * G;
      const bool live = t >= t0 && t <= t1;
      refs[c] = 0.f;
      haves[c] = 0.f;
      // a column without a query sees whatever there is; its output is zero, or none
      qhi[c] = live ? min(shift + t, k1 - 1) : k1 - 1;
      outs[c] = t >= a.seq ? -1 : (((int64_t)b * a.seq + t) * a.ldo + (int64_t)h * HD) * 2 + (live ? 1 : 0);
      if (ALIBI) slope[c] = exp2f(-(float)(a.head_base + h + 1) * 8.0f / (float)a.total_heads) * kLog2e;
    }
    __syncwarp();
    cols_arrive<kSoftWarps + 1>();
    const uint32_t base = smem_u32(smem);
    const uint32_t q_lo = sdesc_lo(base + T::OFF_Q, T::NS * 16);
    const bool lead = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.err, code)) != 0;
    };
    // S_j: HD / 32 MMAs; PV_i: kKeys / 32. An MMA waits for the one before it on the
    // same accumulator, so PV_i and S_{i+2} are issued in turn when both can run.
    const auto s_mma = [&](int j, int kk) {
      const uint32_t s_col = tmem + (uint32_t)((j & 1) * T::SC), k_lo = sdesc_lo(base + (j % KST) * T::TILE, 16) + kk * 2;
      umma_f8(s_col, k_lo, HI_KV, q_lo + kk * 2 * T::NS, HI_Q, IDESC_S, kk > 0);
      if (T::SUM) umma_f8(s_col, k_lo, HI_KV, q_lo + kk * 2 * T::NS + RT, HI_Q, IDESC_S, 1);
    };
    const auto pv_mma = [&](int i, int kk) {
      umma_f8(tmem + T::O_COL, sdesc_lo(base + T::OFF_V + (i % VST) * T::TILE, 16) + kk * (32 * HD / 16),
              HI_KV, sdesc_lo(base + T::OFF_P + (i & 1) * T::P_BYTES, 128) + kk * 32, HI_P, IDESC_PV,
              kk > 0 || i > 0 ? 1u : 0u);
    };
    constexpr int kS = HD / 32, kPV = kKeys / 32;
    if (tiles > 0) ok = wait(q_full, 0, kErrWaitOther);
    for (int j = 0; ok && j < min(2, tiles); ++j) {
      ok = wait(&k_full[j % KST], (j / KST) & 1, kErrWaitFull);
      if (!ok) break;
      tc_fence_after();
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < kS; ++kk) s_mma(j, kk);
        umma_commit(&s_full[j & 1]);
        umma_commit(&k_empty[j % KST]);
      }
      __syncwarp();
    }
    for (int i = 0; ok && i < tiles; ++i) {
      ok = wait(&v_full[i % VST], (i / VST) & 1, kErrWaitFull) && wait(&p_full[i & 1], (i >> 1) & 1, kErrWaitOther);
      if (!ok) break;
      const int j = i + 2;
      uint64_t* jf = &k_full[j % KST];
      const uint32_t jp = (j / KST) & 1;
      const bool both = j < tiles && __all_sync(0xffffffffu, mbar_test_wait(jf, jp));
      tc_fence_after();
      if (lead) {
#pragma unroll
        for (int kk = 0; kk < kPV; ++kk) {
          pv_mma(i, kk);
          if (both && kk < kS) s_mma(j, kk);
        }
        umma_commit(&pv_done[i & 1]);
        if (both) {
          umma_commit(&s_full[j & 1]);
          umma_commit(&k_empty[j % KST]);
        }
        umma_commit(&v_empty[i % VST]);
      }
      __syncwarp();
      if (j < tiles && !both) {
        ok = wait(jf, jp, kErrWaitFull);
        if (!ok) break;
        tc_fence_after();
        if (lead) {
#pragma unroll
          for (int kk = 0; kk < kS; ++kk) s_mma(j, kk);
          umma_commit(&s_full[j & 1]);
          umma_commit(&k_empty[j % KST]);
        }
        __syncwarp();
      }
    }
  } else {
    // ---- queries: hi and lo codes, [16-byte chunk of hd][RT hi rows, RT lo rows][16]
    const bool live = tq >= t0 && tq <= t1;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < QD; ++i) {
      if (!live) xq[i / 2] = 0u;
      const float x = __uint_as_float(i & 1 ? xq[i / 2] & 0xffff0000u : xq[i / 2] << 16);
      m = fmaxf(m, x - x == 0.f ? fabsf(x) : INFINITY);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool bad = m == INFINITY;  // a query that is not finite: its column is NaN
    const float s = bad ? 1.f : kv8_scale(m);
    const float rs = bad ? 0.f : __uint_as_float((254u << 23) - __float_as_uint(s));  // 1 / s, powers of two
    uint32_t hi[QD / 4], lo[QD / 4];  // the lane's codes
#pragma unroll
    for (int i = 0; i < QD; i += 2) {
      const float x0 = __uint_as_float(xq[i / 2] << 16), x1 = __uint_as_float(xq[i / 2] & 0xffff0000u);
      const float y0 = bad ? 0.f : x0 * rs, y1 = bad ? 0.f : x1 * rs;
      const uint32_t h2 = e4m3x2(y0, y1);
      const float2 v = e4m3x2_value(h2);
      const uint32_t l2c = e4m3x2(y0 - v.x, y1 - v.y);
      hi[i / 4] = i % 4 ? hi[i / 4] | h2 << 16 : h2;
      lo[i / 4] = i % 4 ? lo[i / 4] | l2c << 16 : l2c;
    }
    if (qc < RT) {
      uint8_t* dst = smem + T::OFF_Q + (qd / 16) * (T::NS * 16) + qd % 16 + qc * 16;
      if constexpr (QD == 16) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dst + RT * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(dst + RT * 16) = make_uint2(lo[0], lo[1]);
      }
      if (lane % 8 == 0) qf[qc] = bad ? __uint_as_float(0x7fc00000u) : s * a.scale * kLog2e;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    cols_sync<kSoftWarps + 1>();

    // ------------------------------------------------------------------ softmax
    const int wg = warp >> 2, w4 = warp & 3, c0 = wg * CPW;
    const int key = 32 * w4 + lane;  // of the tile; this thread's TMEM lane
    const uint32_t tl = tmem + ((uint32_t)(32 * w4) << 16);
    const uint32_t sm = smem_u32(smem);
    const uint32_t ref = sm + T::OFF_REF + c0 * 4, fac = sm + T::OFF_FAC + c0 * 4;
    const uint32_t have = sm + T::OFF_HAVE + c0 * 4, red = sm + T::OFF_RED + c0 * 4;
    const uint32_t fq = sm + T::OFF_QF + c0 * 4;
    bool known = false;  // every column has a reference
    uint64_t l2[CPW / 2];  // sums of the columns, in pairs
#pragma unroll
    for (int c = 0; c < CPW / 2; ++c) l2[c] = 0ull;
    int slot = 0;  // of the scales' ring, and its pass
    uint32_t pass = 0;
    // Tiles up to low_edge (a window) and from high_edge on hold some column's edge.
    const int low_edge = a.window > 0 && k1 - 1 - a.window >= base0 ? (k1 - 1 - a.window - base0) / kKeys : -1;
    const int high_edge = qlo + 1 >= base0 + kKeys ? (qlo + 1 - base0) / kKeys : 0;
    for (int i = 0; i < tiles; ++i) {
      const int kpos = base0 + i * kKeys + key;
      // After a wait that gave up, the tiles are still walked (the waits return at once):
      // the warpgroup's barriers need every thread.
      mbar_wait(&sc_full[slot], pass, abort_flag, a.err, kErrWaitFull);
      const uint32_t sc = sm + T::OFF_SC + slot * 64 + (key >> 4) * 4;
      if (++slot == T::SCALES) {
        slot = 0;
        pass ^= 1;
      }
      const bool on = kpos < k1;
      const float ks = lds(sc), vs = lds(sc + 32);
      float ev;
      asm("lg2.approx.f32 %0, %1;" : "=f"(ev) : "f"(vs));
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(vs));
      if (!on || vs != vs) inv = 0.f;
      mbar_wait(&s_full[i & 1], (i >> 1) & 1, abort_flag, a.err, kErrWaitAccFull);
      // Rows past the context may hold NaN codes, and 0 * NaN is NaN: cleared, now that
      // S_i has come and PV_{i-2}, the last reader of an earlier tile in this slot, is done.
      if (base0 + (i + 1) * kKeys > k1 && c0 == 0) {
        mbar_wait(&v_full[i % VST], (i / VST) & 1, abort_flag, a.err, kErrWaitFull);
        if (!on) {
          const uint32_t row = sm + T::OFF_V + (i % VST) * T::TILE + key * HD;
#pragma unroll 1
          for (int x = 0; x < HD; x += 16) sts4(row + x, 0u, 0u, 0u, 0u);
        }
      }
      __syncwarp();  // lanes leave a wait one by one; the TMEM loads need them together
      tc_fence_after();
      // y of this key for the group's columns: z + bias - ref (ref = bias before the first)
      float y[CPW];
      {
        uint32_t hi[CPW], lo[T::SUM ? 1 : CPW];
        tmem_ld<CPW>(tl + (i & 1) * T::SC + c0, hi);
        if constexpr (!T::SUM) tmem_ld<CPW>(tl + (i & 1) * T::SC + RT + c0, lo);
        tmem_ld_wait();
        const uint64_t ks2 = f2pack(ks, ks), ev2 = f2pack(ev, ev);
#pragma unroll
        for (int c = 0; c < CPW; c += 4) {
          const float4 f4 = lds4(fq + c * 4), r4 = lds4(ref + c * 4);
          const uint64_t f2[2] = {f2pack(f4.x, f4.y), f2pack(f4.z, f4.w)}, r2[2] = {f2pack(r4.x, r4.y), f2pack(r4.z, r4.w)};
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            uint64_t s2 = f2pack(__uint_as_float(hi[c + e]), __uint_as_float(hi[c + e + 1]));
            if constexpr (!T::SUM) s2 = fadd2(s2, f2pack(__uint_as_float(lo[c + e]), __uint_as_float(lo[c + e + 1])));
            f2unpack(ffma2(s2, fmul2(ks2, f2[e / 2]), fadd2(ev2, r2[e / 2])), y[c + e], y[c + e + 1]);
          }
        }
      }
      if (ALIBI) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) y[c] -= slope[c0 + c] * (float)(qhi[c0 + c] - kpos);
      }
      if (i >= high_edge || i <= low_edge) {
        const int w = a.window > 0 ? a.window : INT_MAX;
#pragma unroll
        for (int c = 0; c < CPW; ++c) {
          const int back = qhi[c0 + c] - kpos;
          if (back < 0 || back >= w) y[c] = -INFINITY;
        }
      }
      float top = fmaxf(y[0], y[1]);
#pragma unroll
      for (int c = 2; c < CPW; c += 2) top = fmax3(top, y[c], y[c + 1]);
      // S_i was committed behind PV_{i-2}, so P's buffer is free.
      if (wg_any<NCG>(wg, !known || top > kBias + kSlack)) {
        // new references: the maximum of every column over the tile's keys
#pragma unroll
        for (int c = 0; c < CPW; c += 4) {
          const float4 r = lds4(ref + c * 4);
          y[c] -= r.x;
          y[c + 1] -= r.y;
          y[c + 2] -= r.z;
          y[c + 3] -= r.w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float m = warp_max(y[c + e]);
            if (lane == 0) sts(red + (w4 * RT + c + e) * 4, m);
          }
        }
        if (i > 0) mbar_wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1, abort_flag, a.err, kErrWaitAccEmpty);
        __syncwarp();
        tc_fence_after();
        wg_sync<NCG>(wg);
        if (key < CPW) {
          const uint32_t at = red + key * 4;
          const float m = fmaxf(fmaxf(lds(at), lds(at + RT * 4)), fmaxf(lds(at + 2 * RT * 4), lds(at + 3 * RT * 4)));
          const float was = lds(ref + key * 4);
          const bool first = lds(have + key * 4) == 0.f;
          float now = was;  // a column whose keys are all masked stays without
          if (m != -INFINITY) {
            now = first ? kBias - m : fminf(was, kBias - m);
            sts(have + key * 4, 1.f);
          }
          sts(fac + key * 4, first ? 1.f : fast_exp2(now - was));
          sts(ref + key * 4, now);
        }
        wg_sync<NCG>(wg);
#pragma unroll
        for (int c = 0; c < CPW; c += 4) {
          const float4 f = lds4(fac + c * 4);
          l2[c / 2] = fmul2(l2[c / 2], f2pack(f.x, f.y));
          l2[c / 2 + 1] = fmul2(l2[c / 2 + 1], f2pack(f.z, f.w));
        }
        if (i > 0) {
#pragma unroll 1
          for (int term = 0; term < 3; ++term) {
            uint32_t o[CPW];
            const uint32_t at = tl + T::O_COL + term * RT + c0;
            tmem_ld<CPW>(at, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < CPW; c += 4) {
              const float4 f = lds4(fac + c * 4);
              o[c] = __float_as_uint(__uint_as_float(o[c]) * f.x);
              o[c + 1] = __float_as_uint(__uint_as_float(o[c + 1]) * f.y);
              o[c + 2] = __float_as_uint(__uint_as_float(o[c + 2]) * f.z);
              o[c + 3] = __float_as_uint(__uint_as_float(o[c + 3]) * f.w);
            }
            tmem_st<CPW>(at, o);
          }
          tmem_st_wait();
        }
        known = __all_sync(0xffffffffu, lds(have + (lane % CPW) * 4) != 0.f);
#pragma unroll
        for (int c = 0; c < CPW; c += 4) {
          const float4 r = lds4(ref + c * 4);
          y[c] += r.x;
          y[c + 1] += r.y;
          y[c + 2] += r.z;
          y[c + 3] += r.w;
        }
      }
      // probabilities, and their three codes: chunks of 16 columns (of 8 + 8 when RT = 8)
      const uint64_t inv2 = f2pack(inv, inv);
      const __half2 eight = __float2half2_rn(8.f);
      uint32_t code[3][CPW / 4];
#pragma unroll
      for (int c = 0; c < CPW; c += 4) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = fast_exp2(y[c + e]);
        l2[c / 2] = ffma2(f2pack(p[0], p[1]), inv2, l2[c / 2]);
        l2[c / 2 + 1] = ffma2(f2pack(p[2], p[3]), inv2, l2[c / 2 + 1]);
        __half2 u = __floats2half2_rn(p[0], p[1]), w = __floats2half2_rn(p[2], p[3]);
#pragma unroll
        for (int term = 0; term < 3; ++term) {
          const uint32_t four = e5m2x4(u, w);
          code[term][c / 4] = four;
          if (term < 2) {  // 8 (u - code), exact: the remainder has fewer bits than FP16 holds
            u = __hmul2(__hsub2(u, e5m2_lo(four)), eight);
            w = __hmul2(__hsub2(w, e5m2_hi(four)), eight);
          }
        }
      }
      const uint32_t pt = sm + T::OFF_P + (i & 1) * T::P_BYTES + key * 16;
      if constexpr (RT == 8) {
        sts4(pt, code[0][0], code[0][1], code[1][0], code[1][1]);
        sts4(pt + kKeys * 16, code[2][0], code[2][1], 0u, 0u);
      } else {
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
          for (int x = 0; x < CPW / 16; ++x)
            sts4(pt + ((term * RT + c0) / 16 + x) * (kKeys * 16), code[term][4 * x], code[term][4 * x + 1],
                         code[term][4 * x + 2], code[term][4 * x + 3]);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i & 1]);
    }
    // sums of the columns over the keys of the four warps, in warp order
#pragma unroll
    for (int c = 0; c < CPW; ++c) {
      float v, w;
      f2unpack(l2[c / 2], v, w);
      if (c & 1) v = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) sts(red + (w4 * RT + c) * 4, v);
    }
    wg_sync<NCG>(wg);
    if (key < CPW) {
      const uint32_t at = red + key * 4;
      lsum[c0 + key] = (lds(at) + lds(at + RT * 4)) + (lds(at + 2 * RT * 4) + lds(at + 3 * RT * 4));
    }
    // every PV has completed (the last two cover the others: MMAs finish in order)
    for (int i = max(0, tiles - 2); i < tiles; ++i)
      mbar_wait(&pv_done[i & 1], (i >> 1) & 1, abort_flag, a.err, kErrWaitAccEmpty);
    ok = *abort_flag == 0;  // a wait that gave up has set it
    tc_fence_after();
  }
  // A bounded wait that gave up is in the error word: every thread still takes the
  // barriers below, and the outputs are not written.
  ok = __syncthreads_and(ok ? 1 : 0) != 0;

  // ---- joining the splits of the context, in rank order: every CTA of the cluster owns a piece of the [column][dim] outputs, and
  // the others write their part of it, unnormalised, with references and sums, into its
  // shared memory. This code runs once and is kept short: fetching it costs more than
  // running it.
  if (threadIdx.x < RT) {
    const int c = threadIdx.x;
    const float den = lsum[c];
    if (haves[c] == 0.f) refs[c] = kNoRef;
    facs[c] = 1.f;
    if (splits == 1) {  // nothing to join: the factors normalise
      facs[c] = 1.f / den;
      if (den == 0.f) outs[c] &= ~1ll;  // a column that saw nothing
    }
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out);
  if (splits > 1) cluster_wait();  // every CTA of the cluster has started
  __syncthreads();
  const int piece = RT * HD / splits, cols = max(1, piece / HD);  // of one owner (powers of two)
  const int lp = 31 - __clz(piece), lc = 31 - __clz(cols);
  const float* in = reinterpret_cast<const float*>(smem + T::OFF_IN);
  const float2* inl = reinterpret_cast<const float2*>(smem + T::OFF_INL);
  if (splits > 1 && (int)threadIdx.x < splits * cols) {
    const int to = (int)threadIdx.x >> lc, k = (int)threadIdx.x & (cols - 1), c = (to << lp) / HD + k;
    st_peer2(peer_addr(inl + split * cols + k, to), refs[c], lsum[c]);
  }
  if (warp < NCG * 4) {
    // lane = dim (head_dim 64: 16 lanes of every warp), a column group per warpgroup
    const int w4 = warp & 3, c0 = (warp >> 2) * CPW;
    const int dim = HD == 128 ? 32 * w4 + lane : 16 * w4 + lane;
    const uint32_t tl = tmem + ((uint32_t)(32 * w4) << 16) + T::O_COL;
#pragma unroll 1
    for (int c = c0; c < c0 + CPW; c += 8) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.f;
      __syncwarp();
      if (tiles > 0) {
        uint32_t v[3][8];
#pragma unroll
        for (int term = 0; term < 3; ++term) tmem_ld<8>(tl + term * RT + c, v[term]);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 8; ++e)
          o[e] = facs[c + e] * fmaf(0.015625f, __uint_as_float(v[2][e]), fmaf(0.125f, __uint_as_float(v[1][e]), __uint_as_float(v[0][e])));
      }
      const bool own = HD == 128 || lane < 16;
      if (splits == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t to = outs[c + e];
          if (own && ok && to >= 0) out[(to >> 1) + dim] = __float2bfloat16_rn(to & 1 ? o[e] : 0.f);
        }
      } else if (own) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int idx = (c + e) * HD + dim;
          st_peer(peer_addr(in + (split << lp) + (idx & (piece - 1)), idx >> lp), o[e]);
        }
      }
    }
  }
  tc_fence_before();
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == kSoftWarps) tmem_dealloc(tmem, T::TMEM);
  if (splits == 1) return;
  const int first = split * piece / HD;
  for (int idx = (int)threadIdx.x * 4; ok && idx < piece; idx += T::THREADS * 4) {
    const int e = split * piece + idx, c = e / HD;
    const int64_t to = outs[c];
    if (to < 0) break;
    const float2* rl = inl + c - first;  // the splits' references and sums
    float ref = kNoRef, den = 0.f, v[4] = {};
    for (int s = 0; s < splits; ++s) ref = fminf(ref, rl[s * cols].x);
    for (int s = 0; s < splits; ++s) {
      const float2 w = rl[s * cols];
      const float4 x = *reinterpret_cast<const float4*>(in + s * piece + idx);
      const float f = fast_exp2(ref - w.x);
      den = fmaf(f, w.y, den);
      v[0] = fmaf(f, x.x, v[0]);
      v[1] = fmaf(f, x.y, v[1]);
      v[2] = fmaf(f, x.z, v[2]);
      v[3] = fmaf(f, x.w, v[3]);
    }
    const float inv = 1.f / den;
    uint2 codes = make_uint2(0u, 0u);
    if ((to & 1) && den != 0.f) codes = make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
    __nv_bfloat16* dst = out + (to >> 1) + e % HD;
    if (reinterpret_cast<uintptr_t>(dst) % 8 == 0) {
      *reinterpret_cast<uint2*>(dst) = codes;
    } else {
      uint16_t* d = reinterpret_cast<uint16_t*>(dst);
      d[0] = (uint16_t)codes.x;
      d[1] = (uint16_t)(codes.x >> 16);
      d[2] = (uint16_t)codes.y;
      d[3] = (uint16_t)(codes.y >> 16);
    }
  }
}

// Share of the SMs' CTAs, in thousandths, that run at once in clusters of 2^k: a cluster
// has to fit the SMs of one GPC. From cudaOccupancyMaxActiveClusters on kernels of the
// same threads and shared memory (148, 148, 132, 120, 112 CTAs with one to an SM; 296,
// 296, 284, 264, 224 with two); for a kernel with TMEM the runtime counts one CTA an SM.
constexpr int kMaxLog = 4;
static_assert(1 << kMaxLog == kMaxCluster, "");
constexpr int kResident[2][kMaxLog + 1] = {{1000, 1000, 891, 810, 756}, {1000, 1000, 940, 880, 756}};

template <int HD, int RT, bool ALIBI>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const Kv8AttnArgs& a, cudaStream_t s) {
  using T = KT<HD, RT>;
  auto kern = kv8_attn_kernel<HD, RT, ALIBI>;
  static std::atomic<uint64_t> ready{0};  // devices whose attributes are set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit, std::memory_order_release);
  }
  const int group = a.heads / a.c.kv_heads;
  const int64_t row_tiles = ((int64_t)a.seq * group + RT - 1) / RT;
  const int64_t pairs = row_tiles * a.c.kv_heads * a.batch;
  // A context is split while every cluster is resident at once and a CTA has a tile:
  // 8 pairs of 32768 keys (head_dim 128) take 179 us unsplit, 28 in clusters of 8, 19 in
  // clusters of 16; 128 pairs of 4096 keys (head_dim 64) 28, and 17 in clusters of 4;
  // 512 pairs of them 48, and 52 in clusters of 2, which no longer fit at once.
  const int64_t keys = a.window > 0 ? std::min<int64_t>(a.max_ctx, (int64_t)a.window + a.seq + kKv8Page) : a.max_ctx;
  const int64_t slots = (int64_t)a.sm_count * T::PER_SM;
  int k = 0;
  while (k < kMaxLog && pairs << (k + 1) <= slots * kResident[T::PER_SM > 1][k + 1] / 1000 && (kKeys << (k + 1)) <= keys) ++k;
  const int splits = 1 << k;
  cudaLaunchConfig_t lc{};
  lc.gridDim = dim3((unsigned)(row_tiles * splits), a.c.kv_heads, a.batch);
  lc.blockDim = dim3(T::THREADS);
  lc.dynamicSmemBytes = T::SMEM;
  lc.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = splits;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&lc, kern, mk, mv, a, splits);
}

template <int HD> cudaError_t launch_hd(const CUtensorMap& mk, const CUtensorMap& mv, const Kv8AttnArgs& a, cudaStream_t s) {
  const int64_t rows = (int64_t)a.seq * (a.heads / a.c.kv_heads);
  const auto go = [&](auto alibi) {
    constexpr bool A = decltype(alibi)::value;
    // The fewest columns that hold a KV group's rows, since absent ones cost the same: 64
    // x 4096 keys with 4 rows of 64: 46 us with 8 columns, 61 with 16, 79 with 32; 32 x
    // 4096 with 12 rows of 128: 45 us with 16, 64 with 32; 8 x 20 rows of 128 in a window
    // of 8192: 34 us with 32, 46 with 64.
    if (rows <= 8) return launch<HD, 8, A>(mk, mv, a, s);
    if (rows <= 16) return launch<HD, 16, A>(mk, mv, a, s);
    if (rows <= 32) return launch<HD, 32, A>(mk, mv, a, s);
    return launch<HD, 64, A>(mk, mv, a, s);
  };
  return a.alibi ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

bool kv8_attention_tc_supported(const Kv8AttnArgs& a) {
  const auto low4 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
  return (a.c.head_dim == 64 || a.c.head_dim == 128) && !low4(a.c.k) && !low4(a.c.v) && !low4(a.c.k_scale) &&
         !low4(a.c.v_scale) && (int64_t)a.c.pages * a.c.kv_heads * kKv8Page <= INT_MAX;
}

cudaError_t kv8_attention_tc(const Kv8AttnArgs& a, cudaStream_t s) {
  alignas(64) CUtensorMap mk, mv;
  const int hd = a.c.head_dim;
  const int sw = hd == 128 ? (int)CU_TENSOR_MAP_SWIZZLE_128B : (int)CU_TENSOR_MAP_SWIZZLE_64B;
  const uint64_t rows = (uint64_t)a.c.pages * a.c.kv_heads * kKv8Page;
  if (!make_tma_2d(&mk, a.c.k, (int)CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, hd, rows, hd, hd, kKv8Page, sw) ||
      !make_tma_2d(&mv, a.c.v, (int)CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, hd, rows, hd, hd, kKv8Page, sw))
    return cudaErrorInvalidValue;
  return hd == 64 ? launch_hd<64>(mk, mv, a, s) : launch_hd<128>(mk, mv, a, s);
}

}  // namespace wv
