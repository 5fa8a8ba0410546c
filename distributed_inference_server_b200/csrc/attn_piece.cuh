// attn_piece.cuh -- what the attention kernels that cut one history into pieces share: states (m, l, O) of pieces and their merge.
//
// The state of a set of keys under one query row: a reference m near its largest score (in the log2 domain), l = sum 2^(s - m), O = sum
// 2^(s - m) v.  Two states join as (M = max m, sum l 2^(m - M), sum O 2^(m - M)); a set without keys is (kPieceNone, 0, 0).  Raising a row's m
// costs a pass over its O, so m follows the largest score only where that has grown by more than kPieceLazy: weights are then at most
// 2^kPieceLazy instead of 1, and as far from it as before in the types they are kept in.
#pragma once
#include "kernels.h"
#include "ptx.cuh"

namespace dis {

// 2^x by the special function unit, two units in the last place; 2^-inf = 0, a NaN stays one
__device__ __forceinline__ float piece_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Finite, and below any score of finite rows: the difference of two references is a number.  A score of -inf weighs nothing, one of +inf or a NaN
// makes the sums NaN.
constexpr float kPieceNone = -1e30f;
constexpr float kPieceLazy = 8.f;

// log2 of a value row's scale, of 2^-87 for one below it (a row of zeros; the smallest scale otherwise) and for NaN
__device__ __forceinline__ float piece_log2_scale(float s) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(s, 6.462348536e-27f)));
  return y;
}

// ---- 8-bit rows as operands: a whole number x in [-127, 127] is exact in fp16.  Byte x + 128 behind 0x64 is the fp16 number 1024 + 128 + x.
__device__ __forceinline__ uint32_t half2_sub_1152(uint32_t v) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x64806480u));
  return r;
}
// four bytes, each already x + 128: bytes 0, 1 and bytes 2, 3 as pairs
__device__ __forceinline__ void bytes_to_half2(uint32_t w, uint32_t &lo, uint32_t &hi) {
  lo = half2_sub_1152(__byte_perm(w, 0x64646464u, 0x4140));
  hi = half2_sub_1152(__byte_perm(w, 0x64646464u, 0x4342));
}

}  // namespace dis
