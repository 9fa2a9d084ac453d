// Unpacking of the 4-bit cache and small PTX shared by the attention kernels.
#pragma once

#include "common.cuh"
#include "kv4.h"

namespace specb200 {
namespace kv4 {

constexpr float kNone = -3.402823466e38f;  // the softmax reference before any score: no finite one is below it
constexpr float kSlack = 8.f;    // a score may pass the reference by this many octaves before it moves
constexpr float kLog2e = 1.4426950408889634f;

SPEC_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPEC_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
SPEC_DEV uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
SPEC_DEV uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Values of nibbles N and N + 4 of w: s (1 + code / 16) + o.  The low nibbles
// are read in place as 1 + code / 2^10 or 1 + code / 2^6 and brought to
// 1 + code / 16 by an exact multiply-add, the high ones by a shift, which
// loads the integer and the f16 pipe alike (6 and 6 instructions a word).
template <int N>
SPEC_DEV uint32_t dq(uint32_t w, uint32_t s2, uint32_t o2) {
  uint32_t x;
  if (N == 0) x = hfma2(lop3_and_or(w, 0x000F000Fu, 0x3C003C00u), 0x54005400u, 0xD3E0D3E0u);       // 64 x - 63
  else if (N == 1) x = hfma2(lop3_and_or(w, 0x00F000F0u, 0x3C003C00u), 0x44004400u, 0xC200C200u);  // 4 x - 3
  else x = lop3_and_or(N == 2 ? w >> 2 : w >> 6, 0x03C003C0u, 0x3C003C00u);
  return hfma2(x, s2, o2);
}
// The power of two (its exponent) that a row of largest magnitude `top` is
// divided by before it goes to f16: bf16 rows may leave f16's range.
SPEC_DEV int row_exponent(const int dtype, float top) {
  if (dtype != T_BF16 || !(top > 0.f && top < INFINITY)) return 0;
  return min(max((__float_as_int(top) >> 23) - 127, -100), 126);
}
SPEC_DEV float pow2i(int e) { return __int_as_float((127 + e) << 23); }

// Which of the 32 tokens from `tok` on a row sees: all cached ones, and of the
// step's those in its mask (or not after it, row index idx; -1: none).
SPEC_DEV uint32_t seen32(int tok, int kv_len, bool masked, unsigned long long mask, int idx) {
  const int x = tok - kv_len;
  if (masked) {
    if (x >= 64) return 0u;
    if (x >= 0) return (uint32_t)(mask >> x);
    return x <= -32 ? ~0u : ((uint32_t)mask << -x) | ((1u << -x) - 1);
  }
  const int n = idx + 1 - x;
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
}
SPEC_DEV uint32_t first32(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

}  // namespace kv4
}  // namespace specb200
