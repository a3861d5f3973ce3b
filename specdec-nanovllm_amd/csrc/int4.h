// int4.h — 4-bit codes on the matrix cores, shared by the 4-bit cache and the 4-bit weight
// kernels.
//
// A code u in 0..15 becomes the 16-bit float 16 + u by bit operations alone: with exponent
// 2^4, bf16 (7 mantissa bits) holds u in mantissa bits 3..6 and fp16 (10 bits) in bits 6..9,
// exactly. Two codes take a shift and an and-or (v_and_or_b32). The products x (16 + u) are
// exact in the fp32 accumulator; what the 16 adds is taken off afterwards from sums of x
// (weights, keys) or of the softmax weights (values). The small base keeps that subtraction
// harmless: it costs at most log2(24 / 8) bits of 24.
#pragma once

#include "sd_common.h"

namespace sd {

template <typename T> struct Magic;
template <> struct Magic<__bf16> {
  static constexpr int kBit = 3;  // mantissa bit of a code's lowest bit
  static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u;
};
template <> struct Magic<_Float16> {
  static constexpr int kBit = 6;
  static constexpr uint32_t kMask = 0x03C003C0u, kBase = 0x4C004C00u;
};

// kBase in a vector register, once a kernel: v_and_or_b32 takes one scalar operand, so with the mask
// and the base both in scalar registers the pair costs an and and an or.
template <typename T> __device__ __forceinline__ uint32_t code_base() {
  uint32_t v = Magic<T>::kBase;
  asm("" : "+v"(v));
  return v;
}

// The codes at bits P .. P + 3 and 16 + P .. 16 + P + 3 of w as two T of 16 + u.
template <typename T, int P> __device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t base) {
  constexpr int kShift = Magic<T>::kBit - P;
  const uint32_t s = kShift >= 0 ? w << (kShift & 31) : w >> (-kShift & 31);
  return (s & Magic<T>::kMask) | base;
}

// The 8 codes of a dword as 8 T of 16 + u, in the order nibble 0, 4, 1, 5, 2, 6, 3, 7.
template <typename T> __device__ __forceinline__ u32x4 unpack8(uint32_t w, uint32_t base) {
  return u32x4{code_pair<T, 0>(w, base), code_pair<T, 4>(w, base), code_pair<T, 8>(w, base),
               code_pair<T, 12>(w, base)};
}

}  // namespace sd
