// Per-pattern lookups of the soft-capped logit z = cap tanh(x / cap) of a bf16 logit x, shared
// by the kernels that stream logits (softcap_ce.hip, token_loss.hip).
#pragma once

#include "kda_device.hpp"

namespace kda {

// Per-element transcendentals (tanh's exp and reciprocal, then exp(z)) at a quarter of the
// VALU rate would cost more than the row's HBM read.  A bf16 logit has only 2^16 bit
// patterns, so the per-pattern values are tabulated in LDS (accurate tanhf / expf), once
// per workgroup of a persistent grid.  The table covers the binary
// exponents kTabELo .. kTabEHi, i.e. |x| in [2^-24, 2^9); a pattern outside is clamped to
// the nearest end of the range.  Below it exp(z) = 1 to within 2^-23; above it
// 1 - tanh(x / cap) <= 2 e^(-2 * 512 / 60) < 1e-7 for every cap <= 60, i.e. tanh has
// saturated to within one f32 ulp.  Inf clamps to +-(2^9 - 2).  NaN patterns (magnitude bits
// above 0x7f80) would clamp too, so the forward keeps a running packed maximum of the
// magnitude bits per lane and makes the row's sum NaN when it exceeds 0x7f80: a NaN logit
// gives a NaN row loss and lse (as tanh + library cross entropy would) and so a NaN gradient
// row in the backward.  Index: sign * kTabHalf + clamp(bits & 0x7fff) - (kTabELo << 7).
constexpr int kTabELo = 127 - 24, kTabEHi = 127 + 8;
constexpr int kTabHalf = (kTabEHi - kTabELo + 1) * 128;  // 4224 patterns per sign
constexpr int kTabSize = 2 * kTabHalf;

__device__ __forceinline__ float tab_pattern_value(int i) {
  const unsigned sign = i >= kTabHalf ? 0x8000u : 0u;
  const unsigned key = (unsigned)(i % kTabHalf) + (kTabELo << 7);
  return __uint_as_float((sign | key) << 16);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Table indices of the two bf16 patterns packed in one 32-bit word, in packed 16-bit integer
// arithmetic: clamp(bits & 0x7fff) - (kTabELo << 7) + sign * kTabHalf, both < 2^14.  The fast
// paths drop the constant - (kTabELo << 7) (tab_index2_biased) and index a table pointer
// moved back by it instead.
__device__ __forceinline__ unsigned tab_index2_packed(unsigned w) {  // both, biased, in one word
  u16x2 k = __builtin_bit_cast(u16x2, w & 0x7fff7fffu);
  k = __builtin_elementwise_max(k, (u16x2)(kTabELo << 7));
  k = __builtin_elementwise_min(k, (u16x2)((kTabEHi << 7) | 127));
  const u16x2 sg = __builtin_bit_cast(u16x2, (w >> 15) & 0x00010001u);
  const u16x2 idx = k + sg * (u16x2)kTabHalf;  // < 17408 + 4224
  return __builtin_bit_cast(unsigned, idx);
}

__device__ __forceinline__ void tab_index2_biased(unsigned w, int& lo, int& hi) {
  const unsigned r = tab_index2_packed(w);
  lo = (int)(r & 0xffffu);
  hi = (int)(r >> 16);
}

__device__ __forceinline__ void tab_index2(unsigned w, int& lo, int& hi) {
  tab_index2_biased(w, lo, hi);
  lo -= kTabELo << 7;
  hi -= kTabELo << 7;
}

__device__ __forceinline__ unsigned bf16_bits(bf16 v) { return (unsigned)__builtin_bit_cast(unsigned short, v); }

__device__ __forceinline__ int tab_index(unsigned bits16) {
  int lo, hi;
  tab_index2(bits16, lo, hi);
  return lo;
}

}  // namespace kda
