// k_cache_i8.cu -- keys and values kept in 8 bits: written as a pass makes them, read back into bf16 pages.
//
// A row (one token and kv head, d entries) stands for x8 s with s = max|x| / 127 and x8 = rint(x 127 / max|x|), so that an entry is at most s / 2
// off (and 2^-23 of it).  Pages are laid out as in bf16, [page][2 (K, V)][n_kv][page_size][d] int8, beside [page][2][n_kv][page_size] fp32
// scales.  A row whose largest magnitude is below 2^-80 is stored as zeros with scale 0 (attention takes
// sums of weights under a reference that follows the scales, and those have to stay within fp32); one that holds an infinity or a NaN gets the scale NaN and reads back as NaN, in attention too.
#include "kernels.h"
#include "ptx.cuh"

namespace dis {

// ------------------------------------------------------------------------------------------------ rope_kv_write_i8
// d / 8 lanes take a row of q, k or v: four entries and the four that rotate with them each, so that a row's maximum is three or four shuffles
// away and nothing is kept in between.  Bound by HBM at prompt size (the fp32 projection is read once, 4 bytes an entry and K slice), by
// latency (positions -> page -> row) for a decode step's tokens.
constexpr int kCwThreads = 256;

__global__ void __launch_bounds__(kCwThreads)
rope_kv_write_i8_kernel(const float *__restrict__ qkv, int n_partial, long long partial_stride, uint16_t *__restrict__ q, int8_t *__restrict__ pool,
                        float *__restrict__ scale, const int *__restrict__ page_table, int max_pages, const int *__restrict__ pt_row,
                        const int *__restrict__ pos, const float *__restrict__ rope_cos, const float *__restrict__ rope_sin, int T, int n_heads,
                        int n_kv, int d, int page_shift) {
  const int lanes = d >> 3, half = d >> 1, rows = n_heads + 2 * n_kv;
  const long long unit = ((long long)blockIdx.x * kCwThreads + threadIdx.x) / lanes;
  const int i = threadIdx.x % lanes * 4;
  pdl_launch_dependents();
  pdl_wait();
  if (unit >= (long long)T * rows) return;  // (whole groups of lanes: shuffles below stay inside one)
  const int t = (int)(unit / rows), r = (int)(unit % rows);
  const float *src = qkv + unit * d + i;
  float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + half);
#pragma unroll 4
  for (int s = 1; s < n_partial; s++) {
    const float4 x = *reinterpret_cast<const float4 *>(src + s * partial_stride), y = *reinterpret_cast<const float4 *>(src + s * partial_stride + half);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
  }
  const int p = pos[t];
  float v[8];
  if (r < n_heads + n_kv) {
    const float4 c = *reinterpret_cast<const float4 *>(rope_cos + (size_t)p * half + i), n = *reinterpret_cast<const float4 *>(rope_sin + (size_t)p * half + i);
    v[0] = a.x * c.x - b.x * n.x; v[1] = a.y * c.y - b.y * n.y; v[2] = a.z * c.z - b.z * n.z; v[3] = a.w * c.w - b.w * n.w;
    v[4] = b.x * c.x + a.x * n.x; v[5] = b.y * c.y + a.y * n.y; v[6] = b.z * c.z + a.z * n.z; v[7] = b.w * c.w + a.w * n.w;
  } else {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  if (r < n_heads) {
    uint16_t *dst = q + ((size_t)t * n_heads + r) * d + i;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(float2_to_bf16x2(v[0], v[1]), float2_to_bf16x2(v[2], v[3]));
    *reinterpret_cast<uint2 *>(dst + half) = make_uint2(float2_to_bf16x2(v[4], v[5]), float2_to_bf16x2(v[6], v[7]));
    return;
  }
  // the other lanes of a group are here too: a group is one row
  const unsigned mask = (lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u)) << (threadIdx.x & 31 & ~(lanes - 1));
  uint32_t top = 0;  // largest magnitude's bits: as whole numbers they are in order, and a NaN's are above infinity's
#pragma unroll
  for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
  const float big = __uint_as_float(top);
  const bool tiny = big < 8.271806126e-25f;  // 2^-80
  const float inv = tiny || top >= 0x7f800000u ? 0.f : 127.f / big;
  const float s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : tiny ? 0.f : big / 127.f;
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    int x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = inv == 0.f ? 0 : __float2int_rn(v[4 * k + j] * inv);
    w[k] = (uint32_t)(x[0] & 255) | (uint32_t)(x[1] & 255) << 8 | (uint32_t)(x[2] & 255) << 16 | (uint32_t)x[3] << 24;
  }
  const int kv = r >= n_heads + n_kv, h = r - n_heads - kv * n_kv;
  const long long page = page_table[(size_t)pt_row[t] * max_pages + (p >> page_shift)];
  const long long row = (((page * 2 + kv) * n_kv + h) << page_shift) + (p & ((1 << page_shift) - 1));
  *reinterpret_cast<uint32_t *>(pool + row * d + i) = w[0];
  *reinterpret_cast<uint32_t *>(pool + row * d + half + i) = w[1];
  if (i == 0) scale[row] = s;
}

cudaError_t launch_rope_kv_write_i8(const float *qkv, int n_partial, long long partial_stride, uint16_t *q, int8_t *pool, float *scale,
                                    const int *page_table, int max_pages, const int *pt_row, const int *pos, const float *rope_cos,
                                    const float *rope_sin, int T, int n_heads, int n_kv, int d, int page_size, cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  int shift = 0;
  while ((1 << shift) < page_size) shift++;
  const long long threads = (long long)T * (n_heads + 2 * n_kv) * (d / 8);
  return launch_k(rope_kv_write_i8_kernel, dim3((unsigned)((threads + kCwThreads - 1) / kCwThreads)), dim3(kCwThreads), 0, st, qkv, n_partial,
                  partial_stride, q, pool, scale, page_table, max_pages, pt_row, pos, rope_cos, rope_sin, T, n_heads, n_kv, d, shift);
}

// ------------------------------------------------------------------------------------------------ kv_read_i8
// HBM-bound: d + 4 bytes in, 2 d out per row.  A CTA takes up to 16 KB of one page of one history; a thread turns 16 entries at a time.
constexpr int kCrThreads = 256, kCrUnroll = 4, kCrBytes = kCrThreads * kCrUnroll * 16;

__global__ void __launch_bounds__(kCrThreads)
kv_read_i8_kernel(const int8_t *__restrict__ pool, const float *__restrict__ scale, uint16_t *__restrict__ out, const int *__restrict__ src_table,
                  const int *__restrict__ dst_table, int max_pages, const int *__restrict__ pt_row, const int *__restrict__ first,
                  const int *__restrict__ ctx, int n_kv, int d_shift, int page_shift) {
  const int r = blockIdx.z, pi = blockIdx.y, page_size = 1 << page_shift;
  pdl_launch_dependents();
  pdl_wait();
  const int lo = (first ? max(first[r], 0) : 0) - (pi << page_shift), hi = ctx[r] - (pi << page_shift);  // of this page: positions [lo, hi)
  if (hi <= 0 || lo >= page_size || lo >= hi) return;
  const size_t entry = (size_t)pt_row[r] * max_pages + pi;
  const long long planes = 2ll * n_kv << page_shift;  // rows of a page
  const long long src = (long long)src_table[entry] * planes, dst = (long long)dst_table[entry] * planes;
  uint4 x[kCrUnroll];
  float s[kCrUnroll];
  const int per = d_shift - 4;  // log2 of the 16-byte chunks of a row
#pragma unroll
  for (int k = 0; k < kCrUnroll; k++) {
    const long long c = ((long long)blockIdx.x * kCrUnroll + k) * kCrThreads + threadIdx.x, row = c >> per;
    const int slot = (int)(row & (page_size - 1));
    if (row < planes && slot >= lo && slot < hi) {
      x[k] = ld_stream_16(pool + (src << d_shift) + c * 16);
      s[k] = scale[src + row];
    }
  }
#pragma unroll
  for (int k = 0; k < kCrUnroll; k++) {
    const long long c = ((long long)blockIdx.x * kCrUnroll + k) * kCrThreads + threadIdx.x, row = c >> per;
    const int slot = (int)(row & (page_size - 1));
    if (row < planes && slot >= lo && slot < hi) {
      uint4 *o = reinterpret_cast<uint4 *>(out + (dst << d_shift) + c * 16);
      const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
      uint32_t y[8];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const char4 b = *reinterpret_cast<const char4 *>(&w[j]);
        y[2 * j] = float2_to_bf16x2(b.x * s[k], b.y * s[k]);
        y[2 * j + 1] = float2_to_bf16x2(b.z * s[k], b.w * s[k]);
      }
      o[0] = make_uint4(y[0], y[1], y[2], y[3]);
      o[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
  }
}

cudaError_t launch_kv_read_i8(const int8_t *pool, const float *scale, uint16_t *kv_pool, const int *src_table, const int *dst_table, int max_pages,
                              const int *pt_row, const int *first, const int *ctx, int n_rows, int n_kv, int d, int page_size, cudaStream_t st) {
  int shift = 0, d_shift = d == 128 ? 7 : 6;
  while ((1 << shift) < page_size) shift++;
  const long long bytes = 2ll * n_kv * page_size * d;
  for (int p0 = 0; p0 < n_rows; p0 += 65535) {  // (grid limits)
    const int n = n_rows - p0 < 65535 ? n_rows - p0 : 65535;
    DIS_CUDA_TRY(launch_k(kv_read_i8_kernel, dim3((unsigned)((bytes + kCrBytes - 1) / kCrBytes), max_pages, n), dim3(kCrThreads), 0, st, pool, scale,
                          kv_pool, src_table, dst_table, max_pages, pt_row + p0, first ? first + p0 : first, ctx + p0, n_kv, d_shift, shift));
  }
  return cudaSuccess;
}

}  // namespace dis
