// k_quant_f8.cu -- rows and weights into 8-bit floating point (f8.cuh): rows of bf16, the residual add and RMS norm in front of a product,
// weights in blocks of 128 x 128.  Bound by memory: each value is read once, its block's maximum found within a warp, and written as a byte.
// Rows [T][K] have their scales as [ceil(K / 128)][T]: the products read the scales of a block's tokens side by side.
#include "f8.cuh"
#include "kernels.h"

namespace dis {

namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantRows = kQuantThreads / 16;  // 16 lanes take a block of a row, 8 entries each

// grid.x: groups of kQuantRows rows, grid.y: shares of the blocks.  Four blocks' loads are on their way at once: 64 KB an SM (with two, 8192 x 6000
// took 35 us, 4.2 TB/s).
__global__ void __launch_bounds__(kQuantThreads)
quant_f8_kernel(const uint16_t *__restrict__ x, uint8_t *__restrict__ x8, float *__restrict__ scale, int T, int K, int per) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kAtOnce = 4;
  const int t = blockIdx.x * kQuantRows + (threadIdx.x >> 4), part = (threadIdx.x & 15) * 8;
  const int blocks = (K + kF8Block - 1) / kF8Block, b1 = min(blocks, ((int)blockIdx.y + 1) * per);
  for (int b0 = blockIdx.y * per; b0 < b1; b0 += kAtOnce) {
    uint4 v[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const int k = (b0 + j) * kF8Block + part;
      v[j] = make_uint4(0u, 0u, 0u, 0u);
      if (t < T && b0 + j < b1 && k < K) v[j] = __ldcg(reinterpret_cast<const uint4 *>(x + (size_t)t * K + k));
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      if (b0 + j >= b1) break;
      const float2 p0 = bf16x2_to_float2(v[j].x), p1 = bf16x2_to_float2(v[j].y), p2 = bf16x2_to_float2(v[j].z), p3 = bf16x2_to_float2(v[j].w);
      uint32_t top = max(f8_top4(p0.x, p0.y, p1.x, p1.y), f8_top4(p2.x, p2.y, p3.x, p3.y));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float s = f8_scale(top), r = f8_inverse(s);
      const int k = (b0 + j) * kF8Block + part;
      if (t < T && k < K) {
        const uint2 o = make_uint2(f8_pack4(p0.x * r, p0.y * r, p1.x * r, p1.y * r), f8_pack4(p2.x * r, p2.y * r, p3.x * r, p3.y * r));
        *reinterpret_cast<uint2 *>(x8 + (size_t)t * K + k) = o;
        if (part == 0) scale[(size_t)(b0 + j) * T + t] = s;
      }
    }
  }
}

// A CTA per 128 x 128 block, a warp per 16 of its rows
__global__ void __launch_bounds__(256)
quant_weight_f8_kernel(const uint16_t *__restrict__ w, uint8_t *__restrict__ w8, float *__restrict__ scale, int N, int K) {
  __shared__ uint32_t tops[8];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = blockIdx.x * kF8Block + lane * 4;
  const long long n0 = (long long)blockIdx.y * kF8Block + warp * 16;
  uint2 v[16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    v[i] = make_uint2(0u, 0u);
    if (n0 + i < N && k < K) v[i] = __ldcg(reinterpret_cast<const uint2 *>(w + (size_t)(n0 + i) * K + k));
    const float2 a = bf16x2_to_float2(v[i].x), b = bf16x2_to_float2(v[i].y);
    top = max(top, f8_top4(a.x, a.y, b.x, b.y));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, tops[i]);
  const float s = f8_scale(top), r = f8_inverse(s);
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (n0 + i < N && k < K) {
      const float2 a = bf16x2_to_float2(v[i].x), b = bf16x2_to_float2(v[i].y);
      *reinterpret_cast<uint32_t *>(w8 + (size_t)(n0 + i) * K + k) = f8_pack4(a.x * r, a.y * r, b.x * r, b.y * r);
    }
  if (threadIdx.x == 0) scale[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// A byte of a weight back as the bf16 nearest to what it stands for
__global__ void unquant_weight_f8_kernel(const uint8_t *__restrict__ w8, const float *__restrict__ scale, uint16_t *__restrict__ w, long long n, int K, int blocks) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / K;
    const int k = (int)(i - r * K);
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)w8[i]));
    float f;
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;}" : "=f"(f) : "r"(h));
    w[i] = float_to_bf16_bits(f * scale[r / kF8Block * blocks + k / kF8Block]);
  }
}

// A load that the SM's own cache serves, which rows of an SM share, and not the read-only path: that is for what does not change while a kernel lives, and the
// kernel in front may still write what this one reads.  (The gain from L2: 8192 rows of 8192 139 us against 130.)
__device__ __forceinline__ float4 ld_coherent(const float *p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}

// add_rmsnorm (k_elementwise.cu) whose rows leave in 8 bits: a CTA per row, and a warp per block of 128 entries, four a lane, so that a
// block's maximum is one warp reduction.  The normed row is not rounded to bf16 on its way.  A thread keeps its kGroups groups of four entries from the sum to
// the store, all of their loads on their way at once: in registers up to eight, while sixteen (rows of more than 32768 entries) spill 904 bytes to
// local memory, which L1 holds.
template <int kGroups>
__global__ void __launch_bounds__(1024)
add_rmsnorm_f8_kernel(float *__restrict__ x, const uint32_t *__restrict__ tokens, const uint16_t *__restrict__ embed, const float *__restrict__ partial,
                      int n_partial, long long partial_stride, const float *__restrict__ gain, uint8_t *__restrict__ x8, float *__restrict__ scale,
                      const int *__restrict__ row_map, int T, int H, float eps) {
  __shared__ float red[32];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = blockDim.x * 4;
  pdl_launch_dependents();
  pdl_wait();
  const int src = row_map ? __ldcg(row_map + t) : t;
  float4 v[kGroups];
  if (tokens) {
    const uint16_t *row = embed + (size_t)__ldcg(tokens + src) * H;
#pragma unroll
    for (int j = 0; j < kGroups; j++) {
      const int i = threadIdx.x * 4 + j * step;
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < H) {
        const uint2 e = __ldcg(reinterpret_cast<const uint2 *>(row + i));
        const float2 a = bf16x2_to_float2(e.x), b = bf16x2_to_float2(e.y);
        v[j] = make_float4(a.x, a.y, b.x, b.y);
      }
    }
  } else {
    const float *row = x + (size_t)src * H;
#pragma unroll
    for (int j = 0; j < kGroups; j++) {
      const int i = threadIdx.x * 4 + j * step;
      v[j] = i < H ? __ldcg(reinterpret_cast<const float4 *>(row + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float *pp = partial + (size_t)src * H;
#pragma unroll(kGroups == 1 ? 4 : 1)
    for (int s = 0; s < n_partial; s++, pp += partial_stride) {
#pragma unroll
      for (int j = 0; j < kGroups; j++) {
        const int i = threadIdx.x * 4 + j * step;
        if (i < H) {
          const float4 p = __ldcg(reinterpret_cast<const float4 *>(pp + i));
          v[j].x += p.x; v[j].y += p.y; v[j].z += p.z; v[j].w += p.w;
        }
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < kGroups; j++) {
    const int i = threadIdx.x * 4 + j * step;
    if (!row_map && i < H) *reinterpret_cast<float4 *>(x + (size_t)t * H + i) = v[j];
    ss += v[j].x * v[j].x + v[j].y * v[j].y + v[j].z * v[j].z + v[j].w * v[j].w;
  }
  ss = warp_sum(ss);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  ss = warp_sum(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.f);
  const float inv = rsqrtf(ss / (float)H + eps);
#pragma unroll
  for (int j = 0; j < kGroups; j++) {
    const int i = threadIdx.x * 4 + j * step, b = i / kF8Block;
    if (b * kF8Block >= H) break;  // (for the whole warp)
    float4 n = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < H) {
      const float4 g = ld_coherent(gain + i);
      n = make_float4(v[j].x * inv * g.x, v[j].y * inv * g.y, v[j].z * inv * g.z, v[j].w * inv * g.w);
    }
    const float s = f8_scale(__reduce_max_sync(0xffffffffu, f8_top4(n.x, n.y, n.z, n.w))), r = f8_inverse(s);
    if (i < H) *reinterpret_cast<uint32_t *>(x8 + (size_t)t * H + i) = f8_pack4(n.x * r, n.y * r, n.z * r, n.w * r);
    if (lane == 0) scale[(size_t)b * T + t] = s;
  }
}

}  // namespace

cudaError_t launch_quant_f8(const uint16_t *x, uint8_t *x8, float *scale, int T, int K, cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  const int groups = (T + kQuantRows - 1) / kQuantRows, blocks = (K + kF8Block - 1) / kF8Block;
  // shares of the blocks so that about eight CTAs an SM are there, of one block each where that is not reached
  int shares = (8 * kNumSMs + groups - 1) / groups;
  shares = shares > blocks ? blocks : shares;
  const int per = (blocks + shares - 1) / shares;
  return launch_k(quant_f8_kernel, dim3(groups, (blocks + per - 1) / per), dim3(kQuantThreads), 0, st, x, x8, scale, T, K, per);
}

cudaError_t launch_quant_weight_f8(const uint16_t *w, uint8_t *w8, float *scale, int N, int K, cudaStream_t st) {
  if (N <= 0) return cudaSuccess;
  const int bn = (N + kF8Block - 1) / kF8Block;
  if (bn > 65535) { set_last_error("quant_weight_f8: more than 65535 * 128 rows"); return cudaErrorInvalidValue; }
  return launch_k(quant_weight_f8_kernel, dim3((K + kF8Block - 1) / kF8Block, bn), dim3(256), 0, st, w, w8, scale, N, K);
}

cudaError_t launch_unquant_weight_f8(const uint8_t *w8, const float *scale, uint16_t *w, int N, int K, cudaStream_t st) {
  if (N <= 0) return cudaSuccess;
  unquant_weight_f8_kernel<<<kNumSMs * 8, 256, 0, st>>>(w8, scale, w, (long long)N * K, K, (K + kF8Block - 1) / kF8Block);
  return cudaGetLastError();
}

cudaError_t launch_add_rmsnorm_f8(float *x, const uint32_t *tokens, const uint16_t *embed, const float *partial, int n_partial, long long partial_stride,
                                  const float *gain, uint8_t *x8, float *scale, const int *row_map, int T, int H, float eps, cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  if (H % 4 != 0 || H * 4 > 200 * 1024) { set_last_error("add_rmsnorm_f8: H must be a multiple of 4 and <= 51200"); return cudaErrorInvalidValue; }
  // Few rows: as many threads as a row takes, up to 1024.  Many: 256 or 512 and two to eight groups each, so that an SM has rows in different phases
  // beside each other (residual add of 8192 rows of 8192: 256 threads 138 us, 512 131; of 1000 rows 24 and 20.6; 2000 rows of 2048 10.7 and 11.2).
  const int quads = H / 4;
  int threads = (quads + 31) / 32 * 32;
  if (T >= 512 && threads > 256) threads = quads <= 512 ? 256 : quads <= 8 * 512 ? 512 : (quads + 8 * 32 - 1) / (8 * 32) * 32;
  threads = threads > 1024 ? 1024 : threads;
  const int groups = (quads + threads - 1) / threads;
  auto f = groups == 1 ? add_rmsnorm_f8_kernel<1> : groups == 2 ? add_rmsnorm_f8_kernel<2> : groups <= 4 ? add_rmsnorm_f8_kernel<4>
           : groups <= 8 ? add_rmsnorm_f8_kernel<8> : add_rmsnorm_f8_kernel<16>;  // (16 * 1024 * 4 > 51200)
  return launch_k(f, dim3(T), dim3(threads), 0, st, x, tokens, embed, partial, n_partial, partial_stride, gain, x8, scale, row_map, T, H, eps);
}

}  // namespace dis
