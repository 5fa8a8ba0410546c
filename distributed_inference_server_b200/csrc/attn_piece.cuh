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
// 8-bit pages: weights times value scales are fp16 in the products, which ends at 2^16 and has no numbers between multiples of 2^-24.  The reference stays
// this far below the largest, so that they are at most 2^(kPieceLazy + kPieceDown) and lose 2^-32 of the largest, not 2^-25: the sum of weights counts what
// they lose, and many small ones behind a large one would all be lost to the same side.
constexpr float kPieceDown = 7.f;

// log2 of a value row's scale, of 2^-80 for one below it (a row of zeros, or one whose largest entry is below 2^-73: 2^7 less room under the largest product,
// the room that kPieceDown makes) and for NaN.  Weights are then at most 2^95, and sums of 2^31 of them numbers
__device__ __forceinline__ float piece_log2_scale(float s) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(s, 8.271806126e-25f)));
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
