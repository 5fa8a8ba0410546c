// k_gemm_f8.cu -- products in 8-bit floating point with a scale for each block of 128, on tcgen05 (kind::f8f6f4, e4m3 x e4m3 -> fp32):
//
//   y[t][n] = sum_b xs[b][t] ws[n / 128][b] sum_{k in block b} x8[t][k] w8[n][k]      x8 [T][K], w8 [N][K], b = k / 128
//
// plain (fp32 or bf16 rows) or as the gate-up product of a feed-forward block: h = silu(g) u of the fused [2][I][K] weight, itself turned
// into 8 bits (f8.cuh).  A block's 128 entries are one 128-byte swizzle row, so a stage of the TMA ring is a block: its four MMAs make
// a fresh accumulator in tensor memory, and the epilogue warps add it, times both scales, to sums that they keep in registers.  Scales
// that are not powers of two and differ from block to block cannot be left to the MMA.
//
// Tokens are the MMA's rows (TMEM lanes) and features its columns at every size: a thread owns one token, so a block's two scales are one
// factor per thread.  With few tokens most lanes compute on what happens to lie in shared memory; nothing waits for them: what bounds
// such a product is the weight coming from HBM.
//
// Two kernels:
//   tile  a CTA per 128 x 128 (gate-up: 128 x 128 + 128) tile and, where the tiles are few, a cluster of up to eight CTAs that share its K:
//         each leaves its sums in its own shared memory, and after a cluster barrier every CTA finishes a share of the tokens.
//   pair  two CTAs per 256 x 256 (or 256 x 128) tile (cta_group::2), persistent, for many tokens: an SM brings 32 KB per block for 512 clocks of the
//         tensor pipe, and reads its 128 x 256 sums from TMEM in the meantime.
#include <cuda.h>
#include <cuda_fp16.h>

#include "f8.cuh"
#include "kernels.h"

namespace dis {

namespace {

constexpr int kF8Threads = 320;  // warp 0 TMA, warp 1 MMA + TMEM, warps 2-9 sums: warp % 4 picks 32 tokens, (warp - 2) / 4 half of the columns
constexpr int kF8Box = 128 * kF8Block;  // bytes of 128 rows of a block

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kUmmaDescHi)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kUmmaDescHi)
      : "memory");
}
// An arrival at a barrier of either CTA of the pair that publishes no memory: what it says, that tensor memory has been read, is ordered by the
// fences of tcgen05.  (With release at cluster scope, and the waits with acquire, every block waited for the scales still on their way: the
// pair kernel took 2.9 thousand clocks a block.)
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Instruction descriptor: D = f32, A = B = e4m3, both K-major
__host__ __device__ constexpr uint32_t f8_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// sums += factor * (kCols columns of tensor memory)
template <int kCols>
__device__ __forceinline__ void add_scaled(const uint32_t (&v)[kCols], float factor, uint64_t *sums) {
  uint64_t f;
  asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "f"(factor));
#pragma unroll
  for (int i = 0; i < kCols / 2; i++) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(v[2 * i]), "r"(v[2 * i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[i]) : "l"(p), "l"(f));
  }
}
__device__ __forceinline__ float2 pair_of(uint64_t s) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(s));
  return r;
}

// Weight scales are any numbers, and a token's times one of them need not be a number: as a factor it would make NaN of a block of zeros.  A block's sum is 0 or
// at least 2^-18, so what it is under two such scales is a number only if it is 0 or their product below 2^146.  No rows and weights that were turned into 8
// bits here come near it, so there are two ways out that cost the others next to nothing: gate-up tiles hold their sums in units of 2^24 from the first such
// block on, their factors, x w 2^-24, end at the largest number (with which any sum but 0 becomes infinite); elsewhere redo_token.
constexpr float kF8Largest = 3.40282347e38f, kF8Unit = 16777216.f;
__device__ __forceinline__ bool f8_too_large(float x, float w) { return fabsf(x * w) > kF8Largest && fabsf(x) <= kF8Largest && fabsf(w) <= kF8Largest; }
__device__ __forceinline__ float f8_factor_in_units(float x, float w) {
  const float f = fabsf(x) > fabsf(w) ? x * (1.f / kF8Unit) * w : w * (1.f / kF8Unit) * x;
  return fabsf(x) <= kF8Largest && fabsf(w) <= kF8Largest ? fminf(fmaxf(f, -kF8Largest), kF8Largest) : f;
}
template <int kPairs>
__device__ __forceinline__ void times(uint64_t (&sums)[kPairs], float by) {
  uint64_t f;
  asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "f"(by));
#pragma unroll
  for (int i = 0; i < kPairs; i++) asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(sums[i]) : "l"(f));
}

// The scales of a thread's token and of its columns' weight rows, fetched ahead (from L2, where the kernel ahead has left them, perhaps while this one was
// there already, which the read-only path is not made for): the token's four blocks at a time, the weight's 32, one
// per lane (they are the same for the whole warp).
template <int kW>
struct Scales {
  const float *xs, *ws[kW];
  int T, t, first, step, end;  // blocks first, first + step, ... below end
  float x[4], x_next[4], w[kW], w_next[kW];
  __device__ __forceinline__ void fetch_x(int i) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int b = first + (i + j) * step;
      x_next[j] = t < T && b < end ? __ldcg(xs + (size_t)b * T + t) : 0.f;
    }
  }
  __device__ __forceinline__ void fetch_w(int i) {
    const int l = first + (i + (int)(threadIdx.x & 31)) * step;
#pragma unroll
    for (int j = 0; j < kW; j++) w_next[j] = l < end ? __ldcg(ws[j] + l) : 0.f;
  }
  // The factors of the i-th block, for sums in units or not.  True if they have to be (for any thread of the warp)
  __device__ __forceinline__ bool get_in_units(int i, bool in_units, float (&f)[kW]) {
    get(i, f);
    bool large = false;
#pragma unroll
    for (int j = 0; j < kW; j++) large |= fabsf(f[j]) > kF8Largest;
    if (!in_units && !__any_sync(0xffffffffu, large)) return false;
    const float a = (i & 2) ? ((i & 1) ? x[3] : x[2]) : ((i & 1) ? x[1] : x[0]);
    large = false;
#pragma unroll
    for (int j = 0; j < kW; j++) large |= f8_too_large(a, __shfl_sync(0xffffffffu, w[j], i & 31));
    in_units |= __any_sync(0xffffffffu, large);
    if (in_units)
#pragma unroll
      for (int j = 0; j < kW; j++) f[j] = f8_factor_in_units(a, __shfl_sync(0xffffffffu, w[j], i & 31));
    return in_units;
  }
  // The factors of the i-th block
  __device__ __forceinline__ void get(int i, float (&f)[kW]) {
    if ((i & 3) == 0) {
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = x_next[j];
      fetch_x(i + 4);
    }
    if ((i & 31) == 0) {
#pragma unroll
      for (int j = 0; j < kW; j++) w[j] = w_next[j];
      fetch_w(i + 32);
    }
    const float a = (i & 2) ? ((i & 1) ? x[3] : x[2]) : ((i & 1) ? x[1] : x[0]);
#pragma unroll
    for (int j = 0; j < kW; j++) f[j] = a * __shfl_sync(0xffffffffu, w[j], i & 31);
  }
};

// g / (1 + e^-g), the approximate exponential and reciprocal as they come: a few parts in 10^6, and half the instructions of gate_act_fast, whose
// division guards against denominators beyond 2^126.  Here the result is 0 with those, for g below -87.3; it would be below 10^-36.
__device__ __forceinline__ float silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}
// The larger magnitude; NaN if any is
__device__ __forceinline__ float max_mag(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ------------------------------------------------------------------------------------------------ the end of a tile
// What the CTAs of a cluster that share a tile's K have in common: sums of a tile's columns per token, rows of kLd floats in each CTA's shared
// memory.  Token rows first, first + step, ... are finished here: the slices' sums are added in order (the same result at every call), a
// warp a token, four columns (gated: and the four that lie 128 behind) a lane, four tokens at once: one token's way through loads, activation,
// maximum and stores takes half a microsecond and they have to overlap.
//   plain     128 columns, features n0 + [0, 128)
//   gated     256 columns, gate and up of features n0 + [0, 128)
struct TileOut {
  void *out;
  float *scale;   // gated: of the rows in 8 bits
  int T, N, t0, n0, wide, bf16;
};
__device__ __forceinline__ void ld_peer4(float (&v)[4], uint32_t at) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void store4(const TileOut &o, int t, int n, const float (&v)[4]) {
  if (o.bf16) {
    uint16_t *p = static_cast<uint16_t *>(o.out) + (size_t)t * o.N + n;
    if (o.wide && n < o.N) *reinterpret_cast<uint2 *>(p) = make_uint2(float2_to_bf16x2(v[0], v[1]), float2_to_bf16x2(v[2], v[3]));
    else
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (n + i < o.N) p[i] = float_to_bf16_bits(v[i]);
  } else {
    float *p = static_cast<float *>(o.out) + (size_t)t * o.N + n;
    if (o.wide && n < o.N) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (n + i < o.N) p[i] = v[i];
  }
}

// The rows of tokens with a factor that is too large (see kF8Largest) are taken from memory once more, their blocks added in 64 bits: 0.3 ms for a token's 128
// features at a K of 4096.
struct F8Memory {
  const uint8_t *x8, *w8;  // (w8: the call's first row)
  const float *xs, *ws;
  int K;
};
__device__ __forceinline__ float dot16(uint4 a, uint4 b, float sum) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; i++) {
    uint32_t p, q;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(p) : "h"((uint16_t)(x[i >> 1] >> (i & 1) * 16)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(q) : "h"((uint16_t)(w[i >> 1] >> (i & 1) * 16)));
    const float2 u = __half22float2(*reinterpret_cast<__half2 *>(&p)), v = __half22float2(*reinterpret_cast<__half2 *>(&q));
    sum = fmaf(u.x, v.x, sum);
    sum = fmaf(u.y, v.y, sum);
  }
  return sum;
}
// A warp: token t's 128 features from o.n0 on, four a lane, if one of the factors there is too large to be a number
template <bool kGated>
__device__ __forceinline__ void redo_token(const F8Memory &m, const TileOut &o, int t) {
  const int lane = threadIdx.x & 31, num_kb = (m.K + kF8Block - 1) / kF8Block, block = o.n0 / kF8Block, ups = (o.N + kF8Block - 1) / kF8Block;
  bool large = false;
  for (int kb = lane; kb < num_kb; kb += 32) {
    const float x = __ldcg(m.xs + (size_t)kb * o.T + t), w = __ldcg(m.ws + (size_t)block * num_kb + kb);
    large |= f8_too_large(x, w) || (kGated && f8_too_large(x, __ldcg(m.ws + (size_t)(ups + block) * num_kb + kb)));
  }
  if (!__any_sync(0xffffffffu, large)) return;
  auto sum = [&](int n, int up) {
    const uint8_t *x = m.x8 + (size_t)t * m.K, *w = m.w8 + ((size_t)up * o.N + n) * m.K;
    const float *ws = m.ws + (size_t)(up * ups + block) * num_kb;
    double y = 0.;
#pragma unroll 1
    for (int kb = 0; kb < num_kb; kb++) {
      float s = 0.f;
#pragma unroll 1
      for (int k = kb * kF8Block; k < min(m.K, (kb + 1) * kF8Block); k += 16)
        s = dot16(__ldcg(reinterpret_cast<const uint4 *>(x + k)), __ldcg(reinterpret_cast<const uint4 *>(w + k)), s);
      y += (double)__ldcg(m.xs + (size_t)kb * o.T + t) * (double)__ldcg(ws + kb) * (double)s;
    }
    return (float)y;
  };
  const int n0 = o.n0 + lane * 4;
  if (kGated) {
    auto h = [&](int n) { return silu(sum(n, 0)) * sum(n, 1); };
    uint32_t top = 0;
#pragma unroll 1
    for (int n = n0; n < min(n0 + 4, o.N); n++) top = max(top, f8_bits(h(n)));
    const float s = f8_scale(__reduce_max_sync(0xffffffffu, top)), q = f8_inverse(s);
#pragma unroll 1
    for (int n = n0; n < min(n0 + 4, o.N); n++) static_cast<uint8_t *>(o.out)[(size_t)t * o.N + n] = (uint8_t)f8_pack4(h(n) * q, 0.f, 0.f, 0.f);
    if (lane == 0) o.scale[(size_t)block * o.T + t] = s;
  } else {
#pragma unroll 1
    for (int n = n0; n < min(n0 + 4, o.N); n++) {
      const float y = sum(n, 0);
      if (o.bf16) static_cast<uint16_t *>(o.out)[(size_t)t * o.N + n] = float_to_bf16_bits(y);
      else static_cast<float *>(o.out)[(size_t)t * o.N + n] = y;
    }
  }
}

template <bool kGated, int kLd>
__device__ __forceinline__ bool finish_tokens(uint32_t base, int rows, int first, int step, int split, const TileOut &o) {
  const int lane = threadIdx.x & 31;
  float top = 0.f;
  for (int r0 = first; r0 < rows; r0 += 4 * step) {
    float a[4][4], b[4][4];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) a[j][i] = b[j][i] = 0.f;
    for (int p = 0; p < split; p++) {
      const uint32_t from = (split > 1 ? cluster_bar(base, (uint32_t)p) : base) + (uint32_t)lane * 16u;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (r0 + j * step < rows) {
          float v[4], u[4];
          const uint32_t at = from + (uint32_t)((r0 + j * step) * kLd) * 4u;
          ld_peer4(v, at);
          if (kGated) ld_peer4(u, at + 512u);
#pragma unroll
          for (int i = 0; i < 4; i++) { a[j][i] += v[i]; if (kGated) b[j][i] += u[i]; }
        }
    }
    const int n = o.n0 + lane * 4;
#pragma unroll
    for (int j = 0; j < 4 && !kGated; j++) top = max_mag(max_mag(top, a[j][0], a[j][1]), a[j][2], a[j][3]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int t = o.t0 + r0 + j * step;
      if (r0 + j * step >= rows) break;
      if (kGated) {  // N features are a multiple of 16: a lane's four are all there or none
#pragma unroll
        for (int i = 0; i < 4; i++) a[j][i] = n < o.N ? silu(a[j][i]) * b[j][i] : 0.f;
        const float s = f8_scale(__reduce_max_sync(0xffffffffu, f8_top4(a[j][0], a[j][1], a[j][2], a[j][3]))), q = f8_inverse(s);
        if (n < o.N) *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(o.out) + (size_t)t * o.N + n) = f8_pack4(a[j][0] * q, a[j][1] * q, a[j][2] * q, a[j][3] * q);
        if (lane == 0) o.scale[(size_t)(o.n0 / kF8Block) * o.T + t] = s;
      } else {
        store4(o, t, n, a[j]);
      }
    }
  }
  return __any_sync(0xffffffffu, !(top <= kF8Largest));
}
// A thread's sums to its token's row: 64 columns from col on (sums: 32 pairs)
__device__ __forceinline__ void put_sums(uint32_t row, int col, const uint64_t *sums) {
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const float2 a = pair_of(sums[2 * i]), b = pair_of(sums[2 * i + 1]);
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(row + (uint32_t)(col + 4 * i) * 4u), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y) : "memory");
  }
}
// A cluster barrier that publishes nothing: reads of other CTAs' shared memory are over.  (With release it waits for the stores to global memory too, a microsecond.)
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------ tile kernel
// The ring's stages, then the barriers.  kGated: 128 gate rows and 128 up rows per stage, 256 accumulator columns; else 128 of each.
template <bool kGated>
struct TileCfg {
  static constexpr int kCols = kGated ? 256 : 128;
  static constexpr int kTmem = 2 * kCols;  // two accumulators: a block's sums are taken while the next block's MMAs run
  static constexpr int kLd = kCols + 4;    // floats of a token's row of sums in shared memory: rows of 32 lanes start on different banks
  static int stage_bytes(int tile_t) { return tile_t * kF8Block + (kGated ? 2 : 1) * kF8Box; }
  // The sums take the ring's place.  (The MMA reads 128 token rows whatever tile_t is: past a shorter tile lie the stage's weight rows.)
  static int body_bytes(int stages, int tile_t, int rows) {
    const int ring = stages * stage_bytes(tile_t), sums = rows * kLd * 4;
    return ring > sums ? ring : sums;
  }
};

template <bool kGated>
__global__ void __launch_bounds__(kF8Threads, kGated ? 1 : 2)
gemm_f8_tile_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const float *__restrict__ xs,
                    const float *__restrict__ ws, const uint8_t *__restrict__ x8, const uint8_t *__restrict__ w8, void *__restrict__ out,
                    float *__restrict__ out_scale, int out_bf16, int T, int N, int K, int w_row0, int split, int tile_t, int stages, uint32_t bar_off,
                    int weights_first, int wide) {
  using Cfg = TileCfg<kGated>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t a_bytes = (uint32_t)tile_t * kF8Block, stage_bytes = a_bytes + (kGated ? 2u : 1u) * kF8Box;
  const uint32_t bar_base = smem_base + bar_off;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (stages + s); };
  auto acc_full = [&](uint32_t b) { return bar_base + 8u * (2 * stages + b); };
  auto acc_empty = [&](uint32_t b) { return bar_base + 8u * (2 * stages + 2 + b); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * stages + 4);

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int tile = blockIdx.x / split, slice = blockIdx.x - tile * split;  // a cluster is one tile's slices, in order
  const int n0 = tile * 128, t0 = blockIdx.y * tile_t, rows = min(tile_t, T - t0);
  const int num_kb = (K + kF8Block - 1) / kF8Block;
  // A slice's blocks, kb0, kb0 + kb_step, ... below kb1: a run of them (every split-th took 4096 x 14336, 1 token in eight slices from 13.7 to 14.3 us), or for
  // gate-up products every split-th, in which form their loop spills no register: 14336 x 4096, 1 / 128 tokens 21.9 / 28.4 -> 21.1 / 26.0 us.
  const int kb_step = kGated ? split : 1, kb0 = kGated ? slice : (int)((long long)num_kb * slice / split);
  const int kb1 = kGated ? num_kb : (int)((long long)num_kb * (slice + 1) / split);
  const int quarters = (rows + 31) >> 5;  // of the lanes that hold tokens

  const int pre = min((kb1 - kb0 + kb_step - 1) / kb_step, stages);
  auto load_w = [&](int kb, int s) {
    const uint32_t dst = smem_base + s * stage_bytes + a_bytes;
    tma_load_2d(dst, &w_map, kb * kF8Block, w_row0 + n0, full_bar(s), kEvictFirst);
    if (kGated) tma_load_2d(dst + kF8Box, &w_map, kb * kF8Block, w_row0 + N + n0, full_bar(s), kEvictFirst);
  };
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
    for (int s = 0; s < stages; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (uint32_t b = 0; b < 2; b++) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 2 * quarters); }
    fence_barrier_init();
    fence_proxy_async();
    if (weights_first)
      for (int i = 0; i < pre; i++) { mbar_expect_tx(full_bar(i), stage_bytes); load_w(kb0 + i * kb_step, i); }
    else
      for (int i = 0; i < pre; i++) {  // a weight that the kernel ahead may be writing: as far as L2
        tma_prefetch_2d(&w_map, (kb0 + i * kb_step) * kF8Block, w_row0 + n0);
        if (kGated) tma_prefetch_2d(&w_map, (kb0 + i * kb_step) * kF8Block, w_row0 + N + n0);
      }
  }
  if (warp == 1) tmem_alloc<Cfg::kTmem>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  pdl_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      for (int i = 0; i < pre; i++) {
        if (!weights_first) { mbar_expect_tx(full_bar(i), stage_bytes); load_w(kb0 + i * kb_step, i); }
        tma_load_2d(smem_base + i * stage_bytes, &x_map, (kb0 + i * kb_step) * kF8Block, t0, full_bar(i), kEvictLast);
      }
      int s = pre == stages ? 0 : pre;
      uint32_t phase = pre == stages ? 1u : 0u;
      for (int kb = kb0 + pre * kb_step; kb < kb1; kb += kb_step) {
        mbar_wait(empty_bar(s), phase ^ 1u);
        mbar_expect_tx(full_bar(s), stage_bytes);
        load_w(kb, s);
        tma_load_2d(smem_base + s * stage_bytes, &x_map, kb * kF8Block, t0, full_bar(s), kEvictLast);
        if (++s == stages) { s = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = f8_idesc(128, Cfg::kCols);
    const uint32_t lo0 = umma_lo(smem_base);
    uint32_t lo = lo0, phase = 0, buf = 0, aphase = 0;
    int s = 0;
    for (int kb = kb0; kb < kb1; kb += kb_step) {
      mbar_wait(acc_empty(buf), aphase ^ 1u);  // (passes on first use)
      mbar_wait(full_bar(s), phase);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) umma_f8(tmem_base + buf * Cfg::kCols, lo + 2 * k, lo + (a_bytes >> 4) + 2 * k, idesc, k > 0 ? 1u : 0u);
        umma_commit(empty_bar(s));
        umma_commit(acc_full(buf));
      }
      __syncwarp();
      lo += stage_bytes >> 4;
      if (++s == stages) { s = 0; phase ^= 1u; lo = lo0; }
      aphase ^= buf;
      buf ^= 1u;
    }
  } else if ((warp & 3) < quarters) {
    // Columns of a warp: its half of the features; gate-up: 64 gate columns and the 64 up columns of the same features
    const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
    pdl_wait();
    Scales<kGated ? 2 : 1> sc;
    sc.xs = xs; sc.T = T; sc.t = r < rows ? t0 + r : T; sc.first = kb0; sc.step = kb_step; sc.end = kb1;
    sc.ws[0] = ws + (size_t)tile * num_kb;
    if (kGated) sc.ws[kGated ? 1 : 0] = ws + ((size_t)((N + 127) / 128) + tile) * num_kb;
    sc.fetch_x(0);
    sc.fetch_w(0);
    uint64_t sums[Cfg::kCols / 4];
#pragma unroll
    for (int i = 0; i < Cfg::kCols / 4; i++) sums[i] = 0;
    const uint32_t cols = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 64;
    uint32_t buf = 0, aphase = 0;
    bool in_units = false;  // (gated; plain tiles see to it at their end, which spilled registers here: 14336 x 4096, 1 / 128 tokens 21.9 / 27.3 us, in units 21.6 / 26.6)
    for (int kb = kb0, i = 0; kb < kb1; kb += kb_step, i++) {
      float f[kGated ? 2 : 1];
      if constexpr (kGated) {
        if (sc.get_in_units(i, in_units, f) && !in_units) {
          in_units = true;
          times(sums, 1.f / kF8Unit);
        }
      } else {
        sc.get(kb - kb0, f);
      }
      mbar_wait(acc_full(buf), aphase);
      tc_fence_after();
      constexpr int CH = 16, kChunks = Cfg::kCols / 2 / CH;  // (32 columns at a time cost registers that two CTAs an SM do not have)
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        uint32_t v[CH];
        tmem_ld_cols(cols + buf * Cfg::kCols + (c * CH / 64) * 128 + c * CH % 64, v);
        tmem_ld_wait();
        if (c == kChunks - 1) {  // everything of this buffer is in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty(buf));
        }
        add_scaled(v, f[kGated ? c * CH / 64 : 0], sums + CH / 2 * c);
      }
      aphase ^= buf;
      buf ^= 1u;
    }
    if (kGated && in_units) times(sums, kF8Unit);
    // The last MMAs have read the ring: the tokens' sums take its place
    if (r < rows) {
      const uint32_t row = smem_base + (uint32_t)(r * Cfg::kLd) * 4u;
      put_sums(row, half * 64, sums);
      if (kGated) put_sums(row, 128 + half * 64, sums + (kGated ? 32 : 0));
    }
    __syncwarp();
  }
  tc_fence_before();
  if (split > 1) cluster_sync(); else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<Cfg::kTmem>(tmem_base);
  pdl_wait();  // (not all warps have been there, and all write)

  // every CTA of the cluster finishes a share of the tokens
  const TileOut o{out, out_scale, T, N, t0, n0, wide, out_bf16};
  const bool odd = finish_tokens<kGated, Cfg::kLd>(smem_base, rows, slice + split * warp, split * (kF8Threads / 32), split, o);
  if (split > 1) cluster_meet();  // no CTA leaves while another reads its sums
  if (!kGated && odd) {  // an infinite factor leaves no number behind (and so do other things)
    auto anew = [](int v) { int r; asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v)); return r; };  // (nothing of this is worth a register in the loop above)
    const int sp = anew(split), tt = anew(tile_t), TT = anew(T);
    int bx, by, tid;
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(bx));
    asm volatile("mov.u32 %0, %%ctaid.y;" : "=r"(by));
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
    const TileOut again{out, out_scale, TT, anew(N), 0, bx / sp * 128, 0, anew(out_bf16)};
#pragma unroll 1
    for (int r = bx % sp + sp * (tid >> 5); r < min(tt, TT - by * tt); r += sp * (kF8Threads / 32)) redo_token<false>(F8Memory{x8, w8, xs, ws, anew(K)}, again, by * tt + r);
  }
}

// ------------------------------------------------------------------------------------------------ pair kernel
// What bounds a block is the way of an accumulator: MMAs, commit, the sums' warps reading it, their arrival at the first CTA.  With two
// buffers of 256 columns that way is longer than two blocks' MMAs; so products have 128 columns, four buffers and, of a tile of 256 columns,
// warps of their own: product h takes rows [64 h, 64 h + 64) of each CTA's 128 feature rows, its columns are 64 features of the first CTA's
// and 64 of the second's (gated: the gate and the up of the same 64 features).
// A tile of 128 columns (64 feature rows a CTA, one product a block, half of its columns a warpgroup) is for few tiles: it brings 24 KB into an SM
// for half the MMAs of 32.
// Three warpgroups.  Warp 0 TMA.  Warps 1 and 3 MMA: two waits, four MMAs and their commits take one warp as long as a block's MMAs take, so
// each issues one of a block's two products (128 columns: every second block).  Warp 2 the products of both scales, [block][token][two] in
// shared memory, in groups of four blocks: fetched and multiplied by the sums' warps themselves they cost a fifth of the kernel's time (8192^3 of
// one value: 392 us against 329 without any).  Warpgroups 1 and 2 the sums, BN / 2 columns a thread in registers, which the first
// warpgroup leaves them (setmaxnreg).
constexpr int kF8PairThreads = 384;
constexpr int kF8PairRegs = 168, kF8PairRegsLow = 56, kF8PairRegsHigh = 224;  // at launch, of the first warpgroup, of the others
static_assert(128 * kF8PairRegsLow + 256 * kF8PairRegsHigh <= kF8PairThreads * kF8PairRegs, "more registers than the block is launched with");

constexpr int kF8Group = 4, kF8Groups = 4;                  // blocks whose factors are made together; such groups kept
constexpr int kF8GroupBytes = kF8Group * 128 * 2 * 4;
// Behind the barriers, a bit a tile of the CTA's, from the 257th on shared with the one 256 tiles earlier: whether one of its factors is no number
constexpr int kF8Large = 208, kF8LargeWords = 8;

// Where a warp turns 32 tokens x 16 words from a token a lane to lanes side by side, [token][17 words]; of a gated tile, the tokens' largest magnitudes
constexpr int kF8TurnRow = 17 * 4, kF8TurnWarp = 32 * kF8TurnRow, kF8Turn = 8 * kF8TurnWarp;

template <int BN>
struct PairCfg {
  static constexpr int kProducts = BN / 128, kBufs = 4 / kProducts;   // of a block; accumulators of each product
  static constexpr int kFeatBox = BN / 2 * kF8Block;                  // bytes of one CTA's feature rows of a block
  static constexpr int kStage = 2 * kF8Box + 2 * kFeatBox;            // one CTA's part of two blocks: token rows, token rows, feature rows, feature rows
  static constexpr int kStages = BN == 256 ? 3 : 4;
  static constexpr int kSmem = kStages * kStage + kF8Groups * kF8GroupBytes + 1024 + 256 + kF8Turn;
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
  static_assert(8 * (2 * kStages + 8 + 2 * kF8Groups) + 4 <= kF8Large && kF8Large + 4 * kF8LargeWords <= 256, "barriers, the address of tensor memory, words");
};

enum { kF8OutF32 = 0, kF8OutBf16 = 1, kF8OutGated = 2 };

// mbar_wait where the barrier has mostly been passed already: one look first, which costs less than a wait
__device__ __forceinline__ void mbar_wait_soon(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  if (!ok) mbar_wait(bar, parity);
}
// Two blocks of a box's rows, {128 entries, rows, blocks} (make_f8_map with depth 2), one behind the other; the same into L2 only
__device__ __forceinline__ void tma_prefetch_3d(const void *map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void *map, int c0, int c1, int c2, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

// Rows of `out` that start anywhere: a warp's 32 tokens (from `first` on) by 16 or 32 features, which lie a token a lane, are turned so that lanes side by
// side store what lies side by side.  (A lane that stores its own token's 16, 32 rows at once, writes every sector eight times: 5000 x 4143, K 512, 228 us
// against the 20 of 4144 columns; 36 turned.)  out: the first of the features in token 0's row; n: that feature.
__device__ __forceinline__ void turn_f32(uint32_t mine, const uint32_t (&v)[16], float *out, int first, int T, int n, int N) {
  const int lane = threadIdx.x & 31, col = lane & 15;
#pragma unroll
  for (int i = 0; i < 16; i++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + (uint32_t)lane * kF8TurnRow + 4u * i), "r"(v[i]) : "memory");
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int row = 2 * i + (lane >> 4);
    float x;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(mine + (uint32_t)row * kF8TurnRow + 4u * col) : "memory");
    if (first + row < T && n + col < N) out[(size_t)(first + row) * N + col] = x;
  }
  __syncwarp();
}
// The same with two features in a word.  A row that starts in the middle of a word has its first and last feature by themselves, and words in between
// from two halves.
__device__ __forceinline__ void turn_bf16(uint32_t mine, const uint32_t (&p)[16], uint16_t *out, int first, int T, int n, int N) {
  const int lane = threadIdx.x & 31, l = lane & 15;
#pragma unroll
  for (int i = 0; i < 16; i++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + (uint32_t)lane * kF8TurnRow + 4u * i), "r"(p[i]) : "memory");
  __syncwarp();
  const int many = min(N - n, 32);  // features that the row still has here
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int row = 2 * i + (lane >> 4);
    uint32_t a, b;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(a) : "r"(mine + (uint32_t)row * kF8TurnRow + 4u * l) : "memory");
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b) : "r"(mine + (uint32_t)row * kF8TurnRow + 4u * min(l + 1, 15)) : "memory");
    uint16_t *o = out + (size_t)(first + row) * N;
    const int off = (int)((uintptr_t)o >> 1) & 1, e = 2 * l + off;
    if (first + row < T && e + 1 < many) *reinterpret_cast<uint32_t *>(o + e) = off ? __funnelshift_r(a, b, 16) : a;
  }
  if (first + lane < T) {  // a lane its token's single ones
    uint16_t *o = out + (size_t)(first + lane) * N;
    const int off = (int)((uintptr_t)o >> 1) & 1;
    auto single = [&](int e) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(mine + (uint32_t)lane * kF8TurnRow + 2u * e) : "memory");
      o[e] = v;
    };
    if (off) single(0);
    if ((many - off) & 1) single(many - 1);
  }
  __syncwarp();
}

template <int kOut, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kF8PairThreads, 1)
gemm_f8_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const float *__restrict__ xs,
                    const float *__restrict__ ws, const uint8_t *__restrict__ x8, const uint8_t *__restrict__ w8, void *__restrict__ out,
                    float *__restrict__ out_scale, int T, int N, int K, int w_row0, int w_row_step, int tiles_n, int tiles_t, int t_fast, int deep, int wide) {
  using Cfg = PairCfg<BN>;
  constexpr bool kGated = kOut == kF8OutGated;
  constexpr int kTileN = kGated ? BN / 2 : BN;
  constexpr int kW = Cfg::kProducts;  // weight scales of a thread's columns
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t factors = smem_base + Cfg::kStages * Cfg::kStage, bar_base = factors + kF8Groups * kF8GroupBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };                                  // (first CTA's are used)
  auto empty_bar = [&](int s) { return bar_base + 8u * (Cfg::kStages + s); };
  auto acc_full = [&](uint32_t slot) { return bar_base + 8u * (2 * Cfg::kStages + slot); };
  auto acc_empty = [&](uint32_t slot) { return bar_base + 8u * (2 * Cfg::kStages + 4 + slot); };  // (first CTA's are used)
  auto f_full = [&](uint32_t g) { return bar_base + 8u * (2 * Cfg::kStages + 8 + g); };
  auto f_empty = [&](uint32_t g) { return bar_base + 8u * (2 * Cfg::kStages + 8 + kF8Groups + g); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * Cfg::kStages + 8 + 2 * kF8Groups);
  const uint32_t large_at = bar_base + kF8Large;
  const uint32_t turn = bar_base + 256u, tops = turn;  // (tops: [128 tokens][2 halves])

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
  const int num_kb = (K + kF8Block - 1) / kF8Block, n_tiles = tiles_n * tiles_t;
  auto tile_n = [&](int tile) { return t_fast ? tile / tiles_t : tile % tiles_n; };
  auto tile_t0 = [&](int tile) { return (t_fast ? tile % tiles_t : tile / tiles_n) * 256 + (int)rank * 128; };
  const uint64_t w_hint = t_fast ? kEvictFirst : kEvictLast, x_hint = t_fast ? kEvictLast : kEvictFirst;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
    for (int s = 0; s < Cfg::kStages; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 2); }
    for (uint32_t i = 0; i < 4; i++) { mbar_init(acc_full(i), 1); mbar_init(acc_empty(i), 16 / Cfg::kProducts); }  // warps of both CTAs
    for (uint32_t g = 0; g < kF8Groups; g++) { mbar_init(f_full(g), 1); mbar_init(f_empty(g), 8); }
    for (uint32_t i = 0; i < kF8LargeWords; i++) asm volatile("st.shared.u32 [%0], 0;" ::"r"(large_at + 4u * i) : "memory");
    fence_barrier_init();
    fence_proxy_async();
    // One round of tiles: the first weight rows, as far as L2, where what the kernel ahead may still write arrives too (gate-up 5632 x 2048, 200 tokens
    // 14.4 -> 13.5 us; of several rounds it took a hundredth).
    const int wr = w_row0 + tile_n(pair) * kTileN + (int)rank * w_row_step;
    for (int kb = 0; n_tiles <= pairs && kb < num_kb && kb < 2 * Cfg::kStages; kb += 2) {
      if (deep) tma_prefetch_3d(&w_map, 0, wr, kb);
      else {
        tma_prefetch_2d(&w_map, kb * kF8Block, wr);
        if (kb + 1 < num_kb) tma_prefetch_2d(&w_map, (kb + 1) * kF8Block, wr);
      }
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers and tensor memory are ready as well
  tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  pdl_launch_dependents();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8PairRegsLow));
    if (warp == 0) {
      if (lane == 0) {
        pdl_wait();
        int s = 0;
        uint32_t phase = 0;
        for (int tile = pair; tile < n_tiles; tile += pairs) {
          const int t0 = tile_t0(tile), wr = w_row0 + tile_n(tile) * kTileN + (int)rank * w_row_step;  // (gated: gate rows | up rows)
          for (int kb = 0; kb < num_kb; kb += 2) {
            mbar_wait_soon(empty_bar(s), phase ^ 1u);  // passes on the first lap
            const bool two = deep || kb + 1 < num_kb;  // (past K a box is zeros, as long as any other)
            if (rank == 0) mbar_expect_tx(full_bar(s), two ? 2 * Cfg::kStage : Cfg::kStage);
            const uint32_t bar = cluster_bar(full_bar(s), 0), a = smem_base + s * Cfg::kStage, w = a + 2 * kF8Box;
            if (deep) {
              tma_load_3d_pair(a, &x_map, 0, t0, kb, bar, x_hint);
              tma_load_3d_pair(w, &w_map, 0, wr, kb, bar, w_hint);
            } else {
              tma_load_2d_pair(a, &x_map, kb * kF8Block, t0, bar, x_hint);
              tma_load_2d_pair(w, &w_map, kb * kF8Block, wr, bar, w_hint);
              if (two) {
                tma_load_2d_pair(a + kF8Box, &x_map, (kb + 1) * kF8Block, t0, bar, x_hint);
                tma_load_2d_pair(w + Cfg::kFeatBox, &w_map, (kb + 1) * kF8Block, wr, bar, w_hint);
              }
            }
            if (++s == Cfg::kStages) { s = 0; phase ^= 1u; }
          }
        }
        // The first CTA's commits still arrive at this CTA's barriers: wait for the last of every stage before the CTA may end.
        for (int i = 0; i < Cfg::kStages; i++) {  // (a stage never filled passes at once)
          mbar_wait(empty_bar(s), phase ^ 1u);
          if (++s == Cfg::kStages) { s = 0; phase ^= 1u; }
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // Factors of four tokens a lane, two blocks at a time, the next two's scales on their way meanwhile (fetched when they are needed, with the comparison
      // below: 4096 x 14336, 512 tokens 33.9 us)
      pdl_wait();
      const int blocks_n = (N + 127) / 128;
      uint32_t g = 0, phase = 0, tiles = 0;
      for (int tile = pair; tile < n_tiles; tile += pairs, tiles++) {
        const int t0 = tile_t0(tile) + lane, b = tile_n(tile) * (kTileN / 128), b2 = kGated ? blocks_n + b : b + 1;
        const float *w0 = ws + (size_t)b * num_kb, *w1 = BN == 256 && (kGated || b2 < blocks_n) ? ws + (size_t)b2 * num_kb : w0;  // (columns past N: whatever)
        struct Two { float x[2][4], a[2], c[2]; } now, next;
        auto fetch = [&](int kb, Two &v) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int at_kb = min(kb + i, num_kb - 1);
#pragma unroll
            for (int j = 0; j < 4; j++) v.x[i][j] = t0 + 32 * j < T ? __ldcg(xs + (size_t)at_kb * T + t0 + 32 * j) : 0.f;
            v.a[i] = __ldcg(w0 + at_kb);
            v.c[i] = __ldcg(w1 + at_kb);
          }
        };
        bool large = false;
        fetch(0, now);
#pragma unroll 2
        for (int kb = 0; kb < num_kb; kb += 2) {
          const uint32_t at = factors + g * (uint32_t)kF8GroupBytes + (kb & (kF8Group - 1)) * 1024u + (uint32_t)lane * 8u;
          fetch(kb + 2, next);
          if ((kb & 2) == 0) mbar_wait(f_empty(g), phase ^ 1u);  // passes on the first lap
#pragma unroll
          for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at + i * 1024u + j * 256u), "f"(now.x[i][j] * now.a[i]), "f"(now.x[i][j] * now.c[i]) : "memory");
            large |= fmaxf(fmaxf(fabsf(now.x[i][0]), fabsf(now.x[i][1])), fmaxf(fabsf(now.x[i][2]), fabsf(now.x[i][3]))) * fmaxf(fabsf(now.a[i]), fabsf(now.c[i])) > kF8Largest;
          }
          if (kb + 2 >= num_kb) {
            large = __any_sync(0xffffffffu, large);
            if (large && lane == 0) asm volatile("red.shared.or.b32 [%0], %1;" ::"r"(large_at + (tiles >> 5 & (kF8LargeWords - 1)) * 4u), "r"(1u << (tiles & 31)) : "memory");
          }
          if ((kb & 2) || kb + 2 >= num_kb) {
            __syncwarp();
            if (lane == 0) mbar_arrive(f_full(g));
            if (++g == kF8Groups) { g = 0; phase ^= 1u; }
          }
          now = next;
        }
      }
    } else if (rank == 0) {
      constexpr uint32_t idesc = f8_idesc(256, 128);
      const uint32_t mine = (uint32_t)warp >> 1;  // warp 1: 0, warp 3: 1
      const uint32_t lo0 = umma_lo(smem_base);
      uint32_t lo = lo0, phase = 0, buf = 0, aphase = 0;
      int s = 0;
      for (int tile = pair; tile < n_tiles; tile += pairs)
        for (int kb = 0; kb < num_kb; kb++) {
          const uint32_t second = kb & 1;  // of the stage's two blocks
          const bool last = second || kb == num_kb - 1;
          if (BN == 256 || (buf & 1u) == mine) {
            const uint32_t h = BN == 256 ? mine : 0u, slot = buf * Cfg::kProducts + h;
            if (BN == 128 || !second) mbar_wait_soon(full_bar(s), phase);
            mbar_wait_soon(acc_empty(slot), aphase ^ 1u);  // both CTAs have taken this buffer (passes on first use)
            tc_fence_after();
            if (elect_one()) {
              const uint32_t a = lo + second * (kF8Box >> 4), w = lo + ((2 * kF8Box + second * Cfg::kFeatBox + h * (kF8Box / 2)) >> 4);
#pragma unroll
              for (uint32_t k = 0; k < 4; k++) umma_f8_pair(tmem_base + slot * 128u, a + 2 * k, w + 2 * k, idesc, k > 0 ? 1u : 0u);
              umma_commit_pair(acc_full(slot));
              // A stage is empty after two commits: of both warps (256 columns) or of both blocks, whoever issued them (128)
              if (BN == 256 ? last : true) umma_commit_pair(empty_bar(s));
              if (BN == 128 && last && !second) umma_commit_pair(empty_bar(s));
            }
            __syncwarp();
          }
          if (last) {
            lo += Cfg::kStage >> 4;
            if (++s == Cfg::kStages) { s = 0; phase ^= 1u; lo = lo0; }
          }
          if (++buf == Cfg::kBufs) { buf = 0; aphase ^= 1u; }
        }
    }
    // Tiles with a factor that is no number, behind all others.  (In the sums' warps, within their loop or behind it, it cost every tile: 4096 x 14336, 512 tokens
    // 30 -> 32 to 37 us.)
    asm volatile("bar.sync 15, 384;" ::: "memory");
    pdl_wait();  // (not all of these warps have been there)
    uint32_t tiles = 0;
    for (int tile = pair; tile < n_tiles; tile += pairs, tiles++) {
      uint32_t large;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(large) : "r"(large_at + (tiles >> 5 & (kF8LargeWords - 1)) * 4u) : "memory");
      if (large >> (tiles & 31) & 1u)
#pragma unroll 1
        for (int n0 = tile_n(tile) * kTileN; n0 < min((tile_n(tile) + 1) * kTileN, N); n0 += kF8Block)
#pragma unroll 1
          for (int t = tile_t0(tile) + warp; t < min(tile_t0(tile) + 128, T); t += 4)
            redo_token<kGated>(F8Memory{x8, w8, xs, ws, K}, TileOut{out, out_scale, T, N, 0, n0, 0, kOut == kF8OutBf16}, t);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8PairRegsHigh));
    const int quarter = warp & 3, half = (warp >> 2) - 1, r = quarter * 32 + lane;
    const uint32_t empty0 = cluster_bar(acc_empty(0), 0), my_factors = factors + (uint32_t)r * 8u;
    const uint32_t cols = tmem_base + ((uint32_t)(quarter * 32) << 16) + (BN == 256 ? 0u : half * 64u);
    pdl_wait();
    uint32_t g = 0, fphase = 0;
    uint32_t buf = 0, aphase = 0;
    for (int tile = pair; tile < n_tiles; tile += pairs) {
      uint64_t sums[BN / 4];
#pragma unroll
      for (int i = 0; i < BN / 4; i++) sums[i] = 0;
      for (int kb = 0; kb < num_kb; kb++) {
        if ((kb & (kF8Group - 1)) == 0) mbar_wait_soon(f_full(g), fphase);
        float f[2];  // (of the first CTA's features and of the second's)
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f[0]), "=f"(f[1]) : "r"(my_factors + g * (uint32_t)kF8GroupBytes + (kb & (kF8Group - 1)) * 1024u) : "memory");
        const uint32_t slot = buf * Cfg::kProducts + (BN == 256 ? half : 0), at = cols + slot * 128u;
        mbar_wait_soon(acc_full(slot), aphase);
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld_32x32(at, v[0]);
        tmem_ld_32x32(at + 32u, v[1]);
        tmem_ld_wait();
        if (BN == 256) {
          add_scaled(v[0], f[0], sums);
          tmem_ld_32x32(at + 64u, v[0]);
          add_scaled(v[1], f[0], sums + 16);
          tmem_ld_32x32(at + 96u, v[1]);
          tmem_ld_wait();
        }
        tc_fence_before();  // everything of this buffer is in registers
        __syncwarp();
        if (lane == 0) mbar_arrive_at(empty0 + 8u * slot);
        if ((kb & (kF8Group - 1)) == kF8Group - 1 || kb == num_kb - 1) {
          if (lane == 0) mbar_arrive(f_empty(g));
          if (++g == kF8Groups) { g = 0; fphase ^= 1u; }
        }
        add_scaled(v[0], f[kW - 1], sums + (BN / 4 - 32));
        add_scaled(v[1], f[kW - 1], sums + (BN / 4 - 16));
        if (++buf == Cfg::kBufs) { buf = 0; aphase ^= 1u; }
      }
      const int t = tile_t0(tile) + r, n0 = tile_n(tile) * kTileN + half * 64;
      if constexpr (kGated) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i++) {
          const float2 g = pair_of(sums[i]), u = pair_of(sums[32 + i]);
          const float a = n0 + 2 * i < N ? silu(g.x) * u.x : 0.f, b = n0 + 2 * i < N ? silu(g.y) * u.y : 0.f;  // (N is even)
          most = max_mag(most, a, b);
          asm("mov.b64 %0, {%1, %2};" : "=l"(sums[i]) : "f"(a), "f"(b));
        }
        // the token's other 64 features are a thread of the other warpgroup's: 64 threads of two warps meet
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(tops + (uint32_t)(r * 2 + half) * 4), "r"(f8_bits(most)) : "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        uint32_t other;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(other) : "r"(tops + (uint32_t)(r * 2 + (half ^ 1)) * 4) : "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        const float s = f8_scale(max(f8_bits(most), other)), q = f8_inverse(s);
        if (t < T) {
          uint8_t *o = static_cast<uint8_t *>(out) + (size_t)t * N + n0;
#pragma unroll
          for (int i = 0; i < 4; i++) {  // 16 features at a time: N is a multiple of 16
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 a = pair_of(sums[8 * i + 2 * j]), b = pair_of(sums[8 * i + 2 * j + 1]);
              w[j] = f8_pack4(a.x * q, a.y * q, b.x * q, b.y * q);
            }
            if (n0 + 16 * i < N) *reinterpret_cast<uint4 *>(o + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (half == 0) out_scale[(size_t)tile_n(tile) * T + t] = s;
        }
      } else {
        // 32 features at a time: twice of the first 128, twice of the second
        const int first = t - lane;  // the warp's tokens: first + [0, 32)
        const uint32_t mine = turn + (uint32_t)(warp - 4) * kF8TurnWarp;
#pragma unroll
        for (int c = 0; c < BN / 64; c++) {
          const int n = n0 + 32 * c + (c >= 2 ? 64 : 0);
          if (n >= N) continue;
          if constexpr (kOut == kF8OutF32) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              uint32_t v[16];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float2 a = pair_of(sums[16 * c + 8 * h + i]);
                v[2 * i] = __float_as_uint(a.x);
                v[2 * i + 1] = __float_as_uint(a.y);
              }
              const int m = n + 16 * h;
              if (wide && m + 16 <= N) {
                float *o = static_cast<float *>(out) + (size_t)t * N + m;
                if (t < T) { st_32(o, v); st_32(o + 8, v + 8); }
              } else {
                turn_f32(mine, v, static_cast<float *>(out) + m, first, T, m, N);
              }
            }
          } else {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float2 a = pair_of(sums[16 * c + i]);
              p[i] = float2_to_bf16x2(a.x, a.y);
            }
            if (wide && n + 32 <= N) {
              uint16_t *o = static_cast<uint16_t *>(out) + (size_t)t * N + n;
              if (t < T) { st_32(o, p); st_32(o + 16, p + 8); }
            } else {
              turn_bf16(mine, p, static_cast<uint16_t *>(out) + n, first, T, n, N);
            }
          }
        }
      }
    }
    asm volatile("bar.arrive 15, 384;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_meet();  // neither CTA leaves while the other's MMAs, commits or arrivals may still reach it
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
}

constexpr int kF8MaxSmem = 227 * 1024;
constexpr int kTileRest = 1024 + 256;  // alignment, barriers

// How a tile kernel's work is laid out: tokens of a tile and CTAs of a cluster
int tile_tokens(int T) { return T <= 32 ? 32 : T <= 64 ? 64 : 128; }
// CTAs that share a tile's K: about eight blocks each and four CTAs at least, as far as all are resident at once (two an SM, fewer in large clusters,
// which have to fit a GPC; gated one) and leave each two blocks; more than four only with few tokens.  Measured with 1 to 8 for nine shapes
// and 1, 32, 64 and 128 tokens, the rule's choice is within 6 % of the best at 34 of the 36 and within 13 % at the rest.  us with 2 / 4 / 8:
// 4096 x 4096, 32 tokens 10.8 / 8.3 / 9.0; 4096 x 14336, 32 tokens 23 / 17.0 / 14.7 and 128 tokens 27 / 18.5 / 20.6.
int tile_split(int T, int N, int K, bool gated) {
  const long long tiles = (long long)((N + 127) / 128) * ((T + tile_tokens(T) - 1) / tile_tokens(T));
  const int num_kb = (K + kF8Block - 1) / kF8Block;
  const int want = num_kb / 8 < 4 || T > 64 ? 4 : num_kb / 8 > 8 ? 8 : num_kb / 8;
  int s = 1;
  while (s < want && num_kb >= 2 * (s + 1) && tiles * (s + 1) <= (gated ? (s + 1 <= 2 ? 148 : 120) : (s + 1 <= 2 ? 296 : 264))) s++;
  return s;
}

template <bool kGated>
cudaError_t tile_launch(const TmaMap &w_map, const TmaMap &x_map, const float *xs, const float *ws, const uint8_t *x8, const uint8_t *w8, void *out,
                        float *out_scale, int out_bf16, int T, int N, int K, int w_row0, int wide, cudaStream_t st) {
  using Cfg = TileCfg<kGated>;
  static DeviceOnce once;
  DIS_CUDA_TRY(once.run([&] { return cudaFuncSetAttribute(gemm_f8_tile_kernel<kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize, kF8MaxSmem); }));
  const int tile_t = tile_tokens(T), split = tile_split(T, N, K, kGated);
  const int tiles_n = (N + 127) / 128, tiles_t = (T + tile_t - 1) / tile_t, rows = tile_t;
  if (tiles_t > 65535) { set_last_error("gemm_f8: too many tokens"); return cudaErrorInvalidValue; }
  const int per = ((K + kF8Block - 1) / kF8Block + split - 1) / split;  // blocks of a slice, at most
  const bool two = !kGated && (long long)tiles_n * tiles_t * split > kNumSMs;
  // (two an SM: a ring of four stages with up to 64 tokens is faster than one of five: 8192 x 8192, 32 tokens 15.5 and 15.8 us)
  const int budget = (two ? tile_t < 128 ? 92 : 106 : 220) * 1024;
  int stages = 2;
  while (stages < per && stages < 12 && Cfg::body_bytes(stages + 1, tile_t, rows) + kTileRest <= budget) stages++;
  const uint32_t bar_off = (uint32_t)Cfg::body_bytes(stages, tile_t, rows);
  const int smem = (int)bar_off + kTileRest;
  const int weights_first = !(pdl_enabled() && !pdl_weights_settled());
  return launch_k_cluster(gemm_f8_tile_kernel<kGated>, dim3(tiles_n * split, tiles_t), dim3(kF8Threads), (size_t)smem, st, split,
                          *reinterpret_cast<const CUtensorMap *>(&w_map), *reinterpret_cast<const CUtensorMap *>(&x_map), xs, ws, x8, w8 + (size_t)w_row0 * K, out, out_scale, out_bf16, T, N, K,
                          w_row0, split, tile_t, stages, bar_off, weights_first, wide);
}

// Blocks that a load of the pair kernel brings: two where rows hold whole blocks only (past the end of a row that does not, the second would be
// the next row's start).  A thread's wait, expectation and two loads take it 0.37 us, as long as a block's MMAs, whatever the boxes' size.
uint32_t f8_depth(int K) { return K % kF8Block == 0 ? 2u : 1u; }

// What a product takes, in hundredths of a microsecond, fitted to ten shapes from 1024 x 1024 to 10240 x 8192 and 8192 x 28672 at 128 to 4096 tokens:
// in pairs a start and an end for every round of tiles, and 20 (128 columns; 25 a block a load) or 34 (256; 39 with several rounds, at the power limit) per block; in
// tiles 60 per block of a slice for every round of CTAs, and the tokens' sums that the slices exchange.
int pair_f8_cost(int T, int N, int K, int columns) {
  const long long tiles = (long long)((N + columns - 1) / columns) * ((T + 255) / 256), num_kb = (K + kF8Block - 1) / kF8Block;
  const long long rounds = (tiles + kNumSMs / 2 - 1) / (kNumSMs / 2);
  const long long cost = columns == 128 ? 230 + rounds * (300 + (f8_depth(K) == 2 ? 20 : 25) * num_kb) : 300 + rounds * (400 + (rounds > 1 ? 39 : 34) * num_kb);
  return cost > 0x7fffffff ? 0x7fffffff : (int)cost;
}
int tile_cost(int T, int N, int K) {
  const int split = tile_split(T, N, K, false), tile_t = tile_tokens(T);
  const long long ctas = (long long)((N + 127) / 128) * ((T + tile_t - 1) / tile_t) * split;
  const long long per = ((K + kF8Block - 1) / kF8Block + split - 1) / split, rounds = (ctas + 2 * kNumSMs - 1) / (2 * kNumSMs);
  const long long cost = 500 + (split > 1 ? 100 : 0) + 60 * per * rounds + (T - 128ll) * 50 / 64;
  return cost > 0x7fffffff ? 0x7fffffff : (int)cost;
}
// Columns of a pair's tile.  (Gated: 256, a tile is a block of 128 features under one scale.)  us with 128 / 256: 4096 x 4096, 512 tokens 11.9 / 18.0, 1024
// tokens 19.3 / 18.6.
int pair_f8_columns(int T, int N, int K, bool gated) { return gated || pair_f8_cost(T, N, K, 256) <= pair_f8_cost(T, N, K, 128) ? 256 : 128; }

template <int kOut, int BN>
cudaError_t pair_f8_launch(const TmaMap &w_map, const TmaMap &x_map, const float *xs, const float *ws, const uint8_t *x8, const uint8_t *w8, void *out,
                           float *out_scale, int T, int N, int K, int w_row0, int wide, cudaStream_t st) {
  using Cfg = PairCfg<BN>;
  static DeviceOnce once;
  DIS_CUDA_TRY(once.run([&] {
    // a block launched with fewer registers would wait for those that its warpgroups ask for
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, gemm_f8_pair_kernel<kOut, BN>);
    if (e == cudaSuccess && at.numRegs < kF8PairRegs) {
      set_last_error("gemm_f8: built with " + std::to_string(at.numRegs) + " registers a thread for the pair kernel, which divides up " + std::to_string(kF8PairRegs));
      e = cudaErrorInvalidKernelImage;
    }
    return e == cudaSuccess ? cudaFuncSetAttribute(gemm_f8_pair_kernel<kOut, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem) : e;
  }));
  const int feats = kOut == kF8OutGated ? BN / 2 : BN;
  const int tiles_n = (N + feats - 1) / feats, tiles_t = (T + 255) / 256;
  const long long n_tiles = (long long)tiles_n * tiles_t;
  if (n_tiles > (1 << 30)) { set_last_error("gemm_f8: too many tiles"); return cudaErrorInvalidValue; }
  const int pairs = n_tiles < kNumSMs / 2 ? (int)n_tiles : kNumSMs / 2;
  const int t_fast = (long long)(kOut == kF8OutGated ? 2 : 1) * N > (long long)T ? 1 : 0;  // as gemm_pair_kernel: the smaller operand stays in L2
  return launch_k(gemm_f8_pair_kernel<kOut, BN>, dim3(2 * pairs), dim3(kF8PairThreads), (size_t)Cfg::kSmem, st, *reinterpret_cast<const CUtensorMap *>(&w_map),
                  *reinterpret_cast<const CUtensorMap *>(&x_map), xs, ws, x8, w8 + (size_t)w_row0 * K, out, out_scale, T, N, K, w_row0, kOut == kF8OutGated ? N : BN / 2, tiles_n, tiles_t,
                  t_fast, f8_depth(K) == 2, wide);
}

}  // namespace

// Which products run in pairs.  Up to 128 tokens none: a pair's tile is half empty (4096 x 14336, 128 tokens: 18.9 us in tiles, 27.7 in pairs; gate-up
// 14336 x 4096, 128 tokens 30.6 and 35.3).  Gate-up products from there on (129 tokens: 49.5 and 35.1; 1024 x 1024, 129 tokens 11.0 and 9.8), plain ones
// where the estimates say so (8192 x 8192, 200 tokens 24.0 and 20.3; but 2048 x 5632, 192 tokens 11.4 and 13.6).
bool gemm_f8_in_pairs(int T, int N, int K, bool gated) {
  if (T <= 128 || gated) return T > 128;
  const int narrow = pair_f8_cost(T, N, K, 128), wide = pair_f8_cost(T, N, K, 256);
  return (narrow < wide ? narrow : wide) < tile_cost(T, N, K);
}
F8Boxes gemm_f8_boxes(int T, int N, int K, bool gated) {
  if (!gemm_f8_in_pairs(T, N, K, gated)) return {(uint32_t)tile_tokens(T), 128u, 1u};
  return {128u, pair_f8_columns(T, N, K, gated) == 128 ? 64u : 128u, f8_depth(K)};
}

cudaError_t launch_gemm_f8(const TmaMap &w_map, const TmaMap &x_map, const uint8_t *x8, const uint8_t *w8, const float *xs, const float *ws, void *out, bool bf16, int T,
                           int N, int K, int w_row0, cudaStream_t st) {
  if (T <= 0 || N <= 0) return cudaSuccess;
  const uintptr_t at = (uintptr_t)out;
  if (gemm_f8_in_pairs(T, N, K, false)) {
    const int wide = (at & 31u) == 0 && N % (bf16 ? 16 : 8) == 0;  // every piece of a row starts on 32 bytes
    const bool narrow = pair_f8_columns(T, N, K, false) == 128;
    auto f = bf16 ? (narrow ? pair_f8_launch<kF8OutBf16, 128> : pair_f8_launch<kF8OutBf16, 256>)
                  : (narrow ? pair_f8_launch<kF8OutF32, 128> : pair_f8_launch<kF8OutF32, 256>);
    return f(w_map, x_map, xs, ws, x8, w8, out, nullptr, T, N, K, w_row0, wide, st);
  }
  const int wide = N % 4 == 0 && (at & (bf16 ? 7u : 15u)) == 0;
  return tile_launch<false>(w_map, x_map, xs, ws, x8, w8, out, nullptr, bf16 ? 1 : 0, T, N, K, w_row0, wide, st);
}

// h = silu(gate) * up in 8 bits; gate rows at w_row0, up rows at w_row0 + I; ws: the gate's blocks, then the up's
cudaError_t launch_gemm_silu_f8(const TmaMap &w_map, const TmaMap &x_map, const uint8_t *x8, const uint8_t *w8, const float *xs, const float *ws, uint8_t *h8, float *hs, int T, int I, int K,
                                int w_row0, cudaStream_t st) {
  if (T <= 0 || I <= 0) return cudaSuccess;
  if (gemm_f8_in_pairs(T, I, K, true)) return pair_f8_launch<kF8OutGated, 256>(w_map, x_map, xs, ws, x8, w8, h8, hs, T, I, K, w_row0, 0, st);
  return tile_launch<true>(w_map, x_map, xs, ws, x8, w8, h8, hs, 0, T, I, K, w_row0, 0, st);
}

}  // namespace dis
