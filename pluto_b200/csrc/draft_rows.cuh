// Rows of a key/value page pool, and the 8-bit storage of a row.
//
// An 8-bit row holds E4M3 codes and one power-of-two scale 2^n, n >= -127 the smallest with
// max|x| <= 448 * 2^n, kept as the byte n + 127 (E8M0).  E4M3 is a floating format, so a scale between two
// powers of two would buy no relative precision; a power of two makes x * 2^-n, the value read back and its
// bf16 form exact, so the only rounding is the one to the code, and attention over an 8-bit cache is
// attention over the bf16 cache of the values read back.  A row with an infinity or a NaN holds byte 255
// and codes 0x7f and reads back as NaN.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "engine.h"

namespace pluto {

// Page of slot t of sequence b, or -1 (reported) where the slot lies outside the sequence's pages or the
// table's entry outside the pool.
__device__ __forceinline__ long long draft_page(const DraftPool& p, int b, int t, uint32_t site) {
  if (t < 0) {
    report_status(p.status, site, kBadLength);
    return -1;
  }
  const int block = t / p.page_size;
  if (block >= (p.table ? p.max_blocks : 1)) {
    report_status(p.status, site, kBadLength);
    return -1;
  }
  if (!p.table) return b;
  const int page = p.table[static_cast<size_t>(b) * p.max_blocks + block];
  if (page < 0 || page >= p.num_pages) {
    report_status(p.status, site, kBadPage);
    return -1;
  }
  return page;
}
__device__ __forceinline__ size_t draft_row(const DraftPool& p, long long page, int t) {
  return static_cast<size_t>(page) * p.page_stride + static_cast<size_t>(t % p.page_size) * p.token_stride;
}
__device__ __forceinline__ size_t draft_scale(const DraftPool& p, long long page, int t) {
  return static_cast<size_t>(page) * p.scale_page + static_cast<size_t>(t % p.page_size) * p.scale_token;
}

// Tokens of sequence b: counts[b], or all of them; a count outside [0, tokens] is reported and clamped.
__device__ __forceinline__ int draft_count(const int32_t* counts, int b, int tokens, uint32_t* status, uint32_t site) {
  if (counts == nullptr) return tokens;
  const int n = counts[b];
  if (n < 0 || n > tokens) {
    report_status(status, site, kBadLength);
    return n < 0 ? 0 : tokens;
  }
  return n;
}

// Scale byte of a row from the bits of its largest magnitude (as integers, so that infinities and NaN
// are the largest).  1.m * 2^e <= 448 * 2^n = 1.75 * 2^(n + 8).
__device__ __forceinline__ uint32_t e8m0_of(uint32_t largest) {
  const uint32_t e = largest >> 23;
  if (e == 255u) return 255u;
  const uint32_t drop = (largest & 0x7fffffu) <= 0x600000u ? 8u : 7u;
  return e > drop ? e - drop : 0u;
}
// 2^-n and 2^n of a scale byte that is not 255 (2^n also of 255: NaN).
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {   // two codes in the low 16 bits
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 e4m3_values(uint32_t pair) {   // the low 16 bits hold two codes
  uint32_t halves;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<const __half2*>(&halves));
}
__device__ __forceinline__ float e4m3_value(uint8_t code) { return e4m3_values(code).x; }

// The output stage of the cached attention (src/llm/layers/util/cached_attention_ops.cc:120-125):
// R(R(value) * R(sigmoid(gate))), R the rounding to bf16 or nothing.
__device__ __forceinline__ float tree_output(const TreeArgs& a, size_t token, int head, int d, float value) {
  if (a.round) value = bf16_round(value);
  if (a.gate) {
    const size_t g = token * a.gate_token + static_cast<size_t>(head) * a.gate_head + d;
    const float x = a.gate_is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[g])
                                   : static_cast<const float*>(a.gate)[g];
    const float factor = sigmoid(x);
    value *= a.round ? bf16_round(factor) : factor;
    if (a.round) value = bf16_round(value);
  }
  return value;
}

}  // namespace pluto
