// Operand fragments of mma.sync m16n8k16 out of e4m3 pages (attention_decode_fp8.cu says how the pages and the contraction index are laid out).
#pragma once
#include "common.cuh"

namespace nrl {

NRL_DEVICE void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  // rows 8..15 of the A tile are padding (G <= 8 query heads): a1 = a3 = 0
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(0u), "r"(a2), "r"(0u), "r"(b0), "r"(b1));
}
NRL_DEVICE uint32_t e4m3x2_to_f16x2(uint32_t v16) {
  uint32_t r;
  asm volatile("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(v16)));
  return r;
}
NRL_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
NRL_DEVICE uint32_t lds32(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(addr));
  return r;
}
NRL_DEVICE uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
// K rows are 128 B = 8 chunks of 16 B; chunk c of token row r lives at chunk c ^ 4 (r & 1): the eight lanes that are served together read chunks t = 0..3
// (or 4..7) of an even and an odd row, which are all eight chunks' banks.
NRL_DEVICE int k_sigma(int r) { return (r & 1) << 2; }

// Weights of fp8 values are f16, a value's scale riding in its weight, and all times a power of two that makes the largest weight of the largest scale so far 2^13 to 2^14,
// whatever scales there are.  A weight is off by 2^-11 of itself, or by 2^-25, 2^-38 of the largest, where it is denormal.
// (Times a constant 2^10, scales of 2.2e-5, of values up to 0.01, made weights under 2.7e-3 denormal: one of 6e-6 is 2.3 steps there, and all of a long tail of them were
// off by a seventh to the same side.)
constexpr uint32_t kMostFactor = 0x78800000u;                        // 2^114: for scales of 2^-100 and less
// the factor, shrunk to a step's scales, of which each lane has some (a whole warp)
NRL_DEVICE float shrink_factor(float factor, float scale) {
  const uint32_t top = min((__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(scale))) + 0x7fffffu) & 0x7f800000u, 0x7e800000u);      // a power of two at or above
  return fminf(factor, __uint_as_float(min(0x86000000u - top, kMostFactor)));
}
NRL_DEVICE float inverse_factor(float factor) { return __uint_as_float(0x7f000000u - __float_as_uint(factor)); }

// a page's values V^T [128][16] in shared memory: tokens outside [from, to) become 0 (a whole warp; synchronised before and after)
NRL_DEVICE void fp8_clear_values(uint8_t* vt, int from, int to, int lane) {
  uint32_t keep[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int lo = max(0, min(4, from - c * 4)), hi = max(0, min(4, to - c * 4));          // bytes [lo, hi) of this word stay
    keep[c] = hi > lo ? (0xffffffffu >> (32 - 8 * hi)) & (0xffffffffu << (8 * lo)) : 0u;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t* w = reinterpret_cast<uint32_t*>(vt + (lane + i * 32) * 16);
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] &= keep[c];
  }
  __syncwarp();
}

}  // namespace nrl
