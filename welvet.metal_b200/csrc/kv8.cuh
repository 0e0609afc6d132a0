// Device helpers of the E4M3 KV cache shared by its append and attention kernels.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace wv {

// Two FP32 values as E4M3 codes (nearest, ties to even, saturating): lo in bits 0-7.
WV_DEV uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The values of two E4M3 codes (bits 0-7 and 8-15), exact.
WV_DEV float2 e4m3x2_value(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
WV_DEV float e4m3_value(uint8_t code) { return e4m3x2_value(code).x; }

// Smallest power of two s >= 2^-64 with amax / s <= 448 = 1.75 * 2^8, from the
// exponent and mantissa bits of amax (finite, not negative).
WV_DEV float kv8_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 8;                  // amax = m 2^(E-127), m in [1, 2): s = 2^(E-127-8)
  if ((u & 0x7fffffu) > 0x600000u) ++e;        // m > 1.75
  return __uint_as_float((uint32_t)max(e, 127 - 64) << 23);
}

// Page of a sequence's token block, or -1 (recorded in the error word) when the table
// names a page outside the pool or the position lies past the table.
WV_DEV int kv8_page(const Kv8Cache& c, int b, int page_index, uint32_t* err) {
  const int page = page_index < c.max_pages ? c.block_table[(size_t)b * c.max_pages + page_index] : -1;
  if (page >= 0 && page < c.pages) return page;
  if (err) atomicCAS(err, 0u, kErrKvPage);
  return -1;
}

// New tokens of sequence b: min(seq_lens[b], seq), not negative.
WV_DEV int kv8_new(const int* seq_lens, int b, int seq) {
  return seq_lens ? max(0, min(seq_lens[b], seq)) : seq;
}

}  // namespace wv
