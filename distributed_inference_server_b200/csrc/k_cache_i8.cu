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
// D / 8 lanes take a row of q, k or v: four entries and the four that rotate with them each, so that a row's maximum is three or four shuffles
// away and nothing is kept in between.  Bound by HBM at prompt size: the fp32 projection is read once, 4 bytes an entry and K slice; by latency
// (positions -> page -> row) for a decode step's tokens.
// kMany: eight CTAs to an SM (32 registers) keep more loads on their way; few CTAs keep a row's K slices on their way instead.  They cross at about five
// CTAs an SM.  us, many / few (CTAs): 32 + 2 x 8 heads of 128, one slice 384 2.6 / 2.6, 600 2.8 / 3.0, 1200 3.7 / 4.1, 4800 9.6 / 11.8, 14400 30.8 / 42.0; four slices
// 96 3.1 / 2.9, 384 3.3 / 3.3, 900 4.6 / 5.1; 32 + 2 x 4 heads of 64, one slice 600 2.6 / 2.4, 800 2.8 / 3.0; four slices 800 3.7 / 3.6, 1200 4.3 / 5.0.
// With the read-back of all histories: six prompts to 2500 tokens (5404 in all) behind 5318, 32 / 8 heads of 128, 45.5 us (37.6 at a plain copy's rate).
constexpr int kCwThreads = 256;

template <int D, bool kMany>
__global__ void __launch_bounds__(kCwThreads, kMany ? 8 : 1)
rope_kv_write_i8_kernel(const float *__restrict__ qkv, int n_partial, long long partial_stride, uint16_t *__restrict__ q, int8_t *__restrict__ pool,
                        float *__restrict__ scale, const int *__restrict__ page_table, int max_pages, const int *__restrict__ pt_row,
                        const int *__restrict__ pos, const float *__restrict__ rope_cos, const float *__restrict__ rope_sin, int n_heads, int n_kv,
                        int page_shift) {
  constexpr int kLanes = D / 8, kHalf = D / 2, kCwRows = kCwThreads / kLanes;
  const int rows = n_heads + 2 * n_kv, groups = (rows + kCwRows - 1) / kCwRows;
  const int t = (int)(blockIdx.x / groups), r = (int)(blockIdx.x % groups) * kCwRows + threadIdx.x / kLanes, i = threadIdx.x % kLanes * 4;
  pdl_launch_dependents();
  pdl_wait();
  if (r >= rows) return;  // (whole groups of lanes: the shuffles below stay inside one)
  const float *src = qkv + ((long long)t * rows + r) * D + i;
  const int p = pos[t];
  float4 a = __ldcs(reinterpret_cast<const float4 *>(src)), b = __ldcs(reinterpret_cast<const float4 *>(src + kHalf));
#pragma unroll 4
  for (int s = 1; s < n_partial; s++) {
    const float4 x = *reinterpret_cast<const float4 *>(src + s * partial_stride), y = *reinterpret_cast<const float4 *>(src + s * partial_stride + kHalf);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
  }
  float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (r < n_heads + n_kv) {
    const float4 c = *reinterpret_cast<const float4 *>(rope_cos + (size_t)p * kHalf + i), n = *reinterpret_cast<const float4 *>(rope_sin + (size_t)p * kHalf + i);
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float x = v[k], y = v[4 + k];
      v[k] = x * cs[k] - y * sn[k];
      v[4 + k] = y * cs[k] + x * sn[k];
    }
  }
  if (r < n_heads) {
    uint16_t *dst = q + ((size_t)t * n_heads + r) * D + i;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(float2_to_bf16x2(v[0], v[1]), float2_to_bf16x2(v[2], v[3]));
    *reinterpret_cast<uint2 *>(dst + kHalf) = make_uint2(float2_to_bf16x2(v[4], v[5]), float2_to_bf16x2(v[6], v[7]));
    return;
  }
  const unsigned mask = ((1u << kLanes) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));  // the group's lanes: all of one row
  uint32_t top = 0;  // largest magnitude's bits: as whole numbers they are in order, and a NaN's are above infinity's
#pragma unroll
  for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
  for (int o = kLanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
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
  *reinterpret_cast<uint32_t *>(pool + row * D + i) = w[0];
  *reinterpret_cast<uint32_t *>(pool + row * D + kHalf + i) = w[1];
  if (i == 0) scale[row] = s;
}

template <int D>
static cudaError_t write_launch(const float *qkv, int n_partial, long long partial_stride, uint16_t *q, int8_t *pool, float *scale, const int *page_table,
                                int max_pages, const int *pt_row, const int *pos, const float *rope_cos, const float *rope_sin, int T, int n_heads, int n_kv,
                                int shift, cudaStream_t st) {
  constexpr int kRows = kCwThreads / (D / 8);
  const long long ctas = (long long)T * ((n_heads + 2 * n_kv + kRows - 1) / kRows);
  auto kern = ctas >= 5 * kNumSMs ? rope_kv_write_i8_kernel<D, true> : rope_kv_write_i8_kernel<D, false>;
  return launch_k(kern, dim3((unsigned)ctas), dim3(kCwThreads), 0, st, qkv, n_partial, partial_stride, q, pool, scale, page_table, max_pages, pt_row, pos,
                  rope_cos, rope_sin, n_heads, n_kv, shift);
}
cudaError_t launch_rope_kv_write_i8(const float *qkv, int n_partial, long long partial_stride, uint16_t *q, int8_t *pool, float *scale,
                                    const int *page_table, int max_pages, const int *pt_row, const int *pos, const float *rope_cos,
                                    const float *rope_sin, int T, int n_heads, int n_kv, int d, int page_size, cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  int shift = 0;
  while ((1 << shift) < page_size) shift++;
  return (d == 128 ? write_launch<128> : write_launch<64>)(qkv, n_partial, partial_stride, q, pool, scale, page_table, max_pages, pt_row, pos, rope_cos,
                                                           rope_sin, T, n_heads, n_kv, shift, st);
}

// ------------------------------------------------------------------------------------------------ kv_read_i8
// HBM-bound: d + 4 bytes in, 2 d out per row.  The pages that the histories' positions lie in are laid end to end, a unit being 16 KB of one of
// them, and dealt to the resident CTAs in turn, whatever the lengths are; a thread turns 16 entries at a time.
constexpr int kCrThreads = 256, kCrUnroll = 4, kCrBytes = kCrThreads * kCrUnroll * 16, kCrMaxRows = 1024;
// CTAs per SM of the grid, twice what is resident: 16 histories to 6000, 8 heads of 128, 31.0 -> 29.0 us; 24 per SM 28.6, but a row's 2 us for a call that
// reads one token back of each of 32
constexpr int kCrCtas = 12;

__global__ void __launch_bounds__(kCrThreads)
kv_read_i8_kernel(const int8_t *__restrict__ pool, const float *__restrict__ scale, uint16_t *__restrict__ out, const int *__restrict__ src_table,
                  const int *__restrict__ dst_table, int max_pages, const int *__restrict__ pt_row, const int *__restrict__ first,
                  const int *__restrict__ ctx, int n_rows, int n_kv, int d_shift, int page_shift) {
  __shared__ int s_pages[kCrMaxRows + 1], s_lo[kCrMaxRows], s_hi[kCrMaxRows], s_scan[kCrThreads / 32];  // pages in front of row r; its positions
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, page_size = 1 << page_shift;
  pdl_launch_dependents();
  pdl_wait();
  for (int r0 = 0, sum = 0; r0 < n_rows; r0 += kCrThreads) {
    const int r = r0 + threadIdx.x;
    int n = 0;
    if (r < n_rows) {
      const int lo = first ? max(first[r], 0) : 0, hi = min(ctx[r], max_pages << page_shift);
      s_lo[r] = lo;
      s_hi[r] = hi;
      if (lo < hi) n = ((hi - 1) >> page_shift) - (lo >> page_shift) + 1;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int before = sum;
    for (int w = 0; w < kCrThreads / 32; w++) {
      if (w < warp) before += s_scan[w];
      sum += s_scan[w];
    }
    if (r < n_rows) s_pages[r + 1] = before + x;
    __syncthreads();
  }
  if (threadIdx.x == 0) s_pages[0] = 0;
  __syncthreads();
  const int planes = 2 * n_kv << page_shift;  // rows of a page
  const int per_page = (int)((((long long)planes << d_shift) + kCrBytes - 1) / kCrBytes), per = d_shift - 4;  // units of a page; log2 of a row's 16-byte chunks
  const long long units = (long long)s_pages[n_rows] * per_page;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;  // (every offset into the pool is a multiple of 32 bytes)
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int pg = (int)(unit / per_page), part = (int)(unit % per_page);
    int b = 0, e = n_rows;  // the row with s_pages[r] <= pg < s_pages[r + 1]
    while (e - b > 1) {
      const int mid = (b + e) >> 1;
      if (s_pages[mid] <= pg) b = mid;
      else e = mid;
    }
    const int pi = (s_lo[b] >> page_shift) + pg - s_pages[b], lo = s_lo[b] - (pi << page_shift), hi = s_hi[b] - (pi << page_shift);
    const size_t entry = (size_t)pt_row[b] * max_pages + pi;
    const long long src = (long long)src_table[entry] * planes, dst = (long long)dst_table[entry] * planes;
    uint4 x[kCrUnroll];
    float s[kCrUnroll];
#pragma unroll
    for (int k = 0; k < kCrUnroll; k++) {
      const int c = (part * kCrUnroll + k) * kCrThreads + threadIdx.x, row = c >> per, slot = row & (page_size - 1);
      if (row < planes && slot >= lo && slot < hi) {
        x[k] = ld_stream_16(pool + (src << d_shift) + (long long)c * 16);
        s[k] = scale[src + row];
      }
    }
#pragma unroll
    for (int k = 0; k < kCrUnroll; k++) {
      const int c = (part * kCrUnroll + k) * kCrThreads + threadIdx.x, row = c >> per, slot = row & (page_size - 1);
      if (row < planes && slot >= lo && slot < hi) {
        const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const char4 q4 = *reinterpret_cast<const char4 *>(&w[j]);
          y[2 * j] = float2_to_bf16x2(q4.x * s[k], q4.y * s[k]);
          y[2 * j + 1] = float2_to_bf16x2(q4.z * s[k], q4.w * s[k]);
        }
        uint16_t *to = out + (dst << d_shift) + (long long)c * 16;
        // a whole 32-byte sector at a time (where the pool starts on one): as two halves, stored by two instructions, L2 takes every sector twice
        if (wide) {
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]),
                       "r"(y[6]), "r"(y[7]) : "memory");
        } else {
          reinterpret_cast<uint4 *>(to)[0] = make_uint4(y[0], y[1], y[2], y[3]);
          reinterpret_cast<uint4 *>(to)[1] = make_uint4(y[4], y[5], y[6], y[7]);
        }
      }
    }
  }
}

cudaError_t launch_kv_read_i8(const int8_t *pool, const float *scale, uint16_t *kv_pool, const int *src_table, const int *dst_table, int max_pages,
                              const int *pt_row, const int *first, const int *ctx, int n_rows, int n_kv, int d, int page_size, cudaStream_t st) {
  int shift = 0, d_shift = d == 128 ? 7 : 6;
  while ((1 << shift) < page_size) shift++;
  for (int r = 0; r < n_rows; r += kCrMaxRows)
    DIS_CUDA_TRY(launch_k(kv_read_i8_kernel, dim3(kNumSMs * kCrCtas), dim3(kCrThreads), 0, st, pool, scale, kv_pool, src_table, dst_table, max_pages,
                          pt_row + r, first ? first + r : first, ctx + r, n_rows - r < kCrMaxRows ? n_rows - r : kCrMaxRows, n_kv, d_shift, shift));
  return cudaSuccess;
}

}  // namespace dis
