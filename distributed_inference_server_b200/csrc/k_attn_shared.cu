// k_attn_shared.cu -- decode attention of a batch whose requests share the first `prefix` positions of their histories.
//
// Positions [0, prefix) hold the same keys and values for all T tokens, so the T G query rows of a kv head are the rows of one matrix product
// against them: K and V of the prefix are read once (per 256 rows) instead of T times, at tcgen05 rate.  Three kernels:
//   attn_stream_kernel   states (m, l, O) of every token over its own positions [prefix, ctx) (k_attn_stream.cu)
//   attn_prefix_kernel   states of 128 or 256 query rows of a kv head over a slice of the prefix; it starts as SMs come free
//   attn_join_kernel     result = the joined states: O / l of their sum under one reference
// A token whose history ends inside the prefix goes through the first alone.
//
// Bytes: nkv 2 d b (prefix + sum of own lengths); operations: 4 G d T prefix nkv on the tensor cores and T G prefix nkv exponentials (16 per
// clock and SM: 512 clocks per 128 rows x 64 keys beside 256 + 256 of the products for d = 128).
//
// attn_prefix_kernel, one CTA per SM:
//   warp 0          bf16 pages: K and V tiles of 64 keys by TMA into a ring; 8-bit pages: their rows into a ring of their own
//   warps 1, 2      the MMAs of softmax group 0 and 1: S = Q K^T (M128 N64), two tiles ahead of O += P V (M128 N = d; bf16: twice)
//   warps 4-7, 8-11 softmax groups, one thread per row.  Up to 128 rows: both groups have the same rows, group 0 the even key tiles, group 1
//                   the odd ones, and their states are joined at the end; more: 128 rows each, and both read every tile (kPair)
//   warps 12-15     8-bit pages: rows turned to fp16 (exact) into the tiles' ring.  They are near to being the bound, so they do nothing else: with the
//                   rows' addresses and copies (cp.async) theirs too, a third of their time, 64 requests behind 64000 tokens took 179 us, now 168
// TMEM: four score buffers of 64 columns, P over its scores, an O of d columns per group.  A group raises a row's reference only when its
// maximum has grown by more than 8 in the log2 domain, so O is seldom rescaled (the reference cancels).
// 8-bit pages: scales stay outside the products, as in k_attn_stream.cu; q and the weights are fp16 there.  bf16 pages: V is bf16, so the weights have to be,
// and enter O += P V as two bf16 halves, one product behind the other: with the upper half alone (2^-9 of a weight) results were 2.0e-3 from 64 bits where
// every token by itself gives 1.7e-3, and what a step's results are worth would have depended on its batch.  P and its rest fill the 64 columns of the scores.
// 32 requests behind 6000 24.2 -> 24.8 us, 64 behind 64000 128 -> 156.
//
// Measured (B200, from graphs, all three kernels): 32 requests behind 6000 tokens, 32 / 8 heads of 128, own parts to 500, bf16: 24.8 us (6.9 for its bytes);
// 64 behind 8000, 64 / 8 heads, own parts to 700, 8 bits: 50.7 (10.6 at a library product's rate, 7.6 for its bytes).  A step of 256 rows x 64 keys takes
// 1.2 to 1.3 us in both (slope from 16000 to 64000 tokens).  bf16: the products take 1792 clocks of the tensor pipe a step (S with N = 64 reads 6 KB of operands
// each, at shared memory's rate, 768; P V twice 1024); exponentials and P, two warps to a scheduler, took 1290 before the weights' rests, 1024 of them the
// exponentials alone.  8 bits: a group's exponentials 970 (in turn), maximum 560 (scales of K and V from shared memory), its turn 190, P's hand-over 125, the
// tile's fp16 rows 330, of 2210: shared memory and issue slots are shared with the warps that turn rows to fp16.  Eight of those instead of four (96 registers) were
// slower (64 behind 64000 161 -> 182 us), as were rows through registers (179 -> 230 before warp 0 copied them) or turned in units of half a tile (-> 210).  The score buffers
// are two per group so that a group's next product runs under its softmax: one of twice the keys, which needs a third less of the tensor pipe for S, was
// slower (bf16 with weights in one half, 131 -> 154 us at 64000), the two groups being in phase.  A CTA's start (queries, barriers, TMEM) and end (128 KB of state)
// are six steps' worth: the 64 behind 8000 have 14 steps a CTA, some 18 us; the rest is that start and end, the own parts in front and the join behind.
#include <algorithm>

#include <cuda_fp16.h>

#include "attn_piece.cuh"

namespace dis {

constexpr int kSpTile = 64;               // keys of a tile
constexpr int kSpBlock = kSpTile * 128;   // 64 keys x 64 dims, 16 bits
constexpr int kSpQBlock = 128 * 128;      // 128 rows x 64 dims
constexpr int kSpRaw = 3;                 // stages of 8-bit rows (and of their scales)
constexpr int kSpMaxSlices = 32;

template <int D, bool I8, bool kPair>
struct SpCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kHalves * kSpBlock;
  static constexpr int kQBytes = (kPair ? 2 : 1) * kHalves * kSpQBlock;
  // One tile of rows: an even number, so that a slot's tiles are all of one group, whose warps then wait for every phase of its barriers in turn.  (A
  // warp that skips a phase takes the one before it for the one it waits for.)
  static constexpr int kRing = D == 64 ? 6 : I8 && kPair ? 3 : 4;
  static_assert(kPair || kRing % 2 == 0, "");
  static constexpr int kRawBytes = 2 * kSpTile * D;  // K and V rows of a tile in 8 bits
  static constexpr int kScaleFloats = 3 * kSpTile;   // of a tile: K factor, V scale, its log2
  static constexpr int kQ = 0, kK = kQBytes, kV = kK + kRing * kTileBytes, kRaw = kV + kRing * kTileBytes;
  static constexpr int kRawScale = kRaw + (I8 ? kSpRaw * kRawBytes : 0);
  static constexpr int kScale = kRawScale + (I8 ? kSpRaw * 2 * kSpTile * 4 : 0);
  static constexpr int kMeet = kScale + (I8 ? kRing * kScaleFloats * 4 : 0);  // [group][row] (m, l)
  static constexpr int kUp = kMeet + 2 * 128 * 8;  // the rows' powers of two
  static constexpr int kBars = kUp + 256 * 4;
  static constexpr int kSmem = kBars + 512;
  static constexpr int kThreads = I8 ? 512 : 384;
};

// A wait with an end: false after about a second, or once another warp of the CTA has given up.  The whole warp calls it.
constexpr long long kSpPatience = 2000000000;  // clocks
__device__ __forceinline__ bool sp_poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ bool sp_failed(uint32_t fail) {
  uint32_t bad;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(bad) : "r"(fail) : "memory");
  return __any_sync(0xffffffffu, bad != 0);
}
__device__ __forceinline__ bool sp_wait(uint32_t bar, uint32_t parity, uint32_t fail) {
  if (sp_poll(bar, parity)) return true;
  const long long began = clock64();
  do {
    if (sp_poll(bar, parity)) return true;
    if (sp_failed(fail)) return false;
  } while (__all_sync(0xffffffffu, clock64() - began < kSpPatience));
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(fail), "r"(1) : "memory");
  return false;
}

__device__ __forceinline__ float2 sp_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 sp_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 sp_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float sp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void sp_tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void sp_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 columns of O from `addr` on, times f
__device__ __forceinline__ void sp_rescale_16(uint32_t addr, float f) {
  uint32_t v[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                 "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(addr) : "memory");
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
  sp_tmem_st_16(addr, v);
}

// size bytes (a multiple of 16, as both addresses are) to shared memory, counted by the barrier
__device__ __forceinline__ void sp_bulk(uint32_t dst, const void *src, uint32_t size, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(size), "r"(bar) : "memory");
}

struct SpArgs {
  const uint16_t *q;
  const int8_t *pool;     // I8
  const float *scale;
  const int *page_table, *pt_row;
  int max_pages, page_shift;
  float *state_o;         // [slice][kv head][128-row tile][D / 4][128] x 4 floats
  float *state_ml;        // [slice][kv head][128-row tile][128] x (m, l)
  int T, g_shift, n_kv, prefix, row_tiles, slices, late_wait, let_next;
  const int *prefix_at;   // where the prefix is instead of in `prefix` (a captured launch serves every prefix of as many slices), or nullptr
};

template <int D, bool I8, bool kPair>
__global__ void __launch_bounds__(SpCfg<D, I8, kPair>::kThreads, 1)
attn_prefix_kernel(const __grid_constant__ CUtensorMap kv_map, const SpArgs a) {
  using Cfg = SpCfg<D, I8, kPair>;
  constexpr int NS = Cfg::kRing, kHalves = Cfg::kHalves;
  extern __shared__ __align__(1024) uint8_t sp_smem[];
  const uint32_t base = smem_u32(sp_smem), bars = base + Cfg::kBars;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 64u + 8u * s; };
  auto v_full = [&](int s) { return bars + 128u + 8u * s; };
  auto v_empty = [&](int s) { return bars + 192u + 8u * s; };
  auto s_full = [&](int g, int b) { return bars + 256u + 16u * g + 8u * b; };
  auto p_full = [&](int g, int b) { return bars + 288u + 16u * g + 8u * b; };
  auto pv_done = [&](int g) { return bars + 320u + 8u * g; };
  auto o_done = [&](int g) { return bars + 352u + 8u * g; };
  auto raw_full = [&](int s) { return bars + 368u + 8u * s; };
  auto raw_empty = [&](int s) { return bars + 400u + 8u * s; };
  auto turn = [&](int g, int quarter) { return bars + 424u + 32u * g + 8u * quarter; };
  const uint32_t q_full = bars + 336, tmem_slot = bars + 344, fail = bars + 348;

  const int slice = blockIdx.x, kvh = blockIdx.z, rt0 = blockIdx.y * (kPair ? 2 : 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int prefix = a.prefix_at ? *a.prefix_at : a.prefix;
  const int n_all = (prefix + kSpTile - 1) / kSpTile;
  const int tile0 = (int)((long long)n_all * slice / a.slices), n = (int)((long long)n_all * (slice + 1) / a.slices) - tile0;  // n >= 1
  auto steps = [&](int g) { return kPair ? n : (n + 1 - g) >> 1; };
  auto tile_of = [&](int g, int i) { return kPair ? i : 2 * i + g; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; s++) {
      mbar_init(k_full(s), I8 ? 4 : 1); mbar_init(v_full(s), I8 ? 4 : 1);
      mbar_init(k_empty(s), kPair ? 2 : 1); mbar_init(v_empty(s), kPair ? 2 : 1);
    }
    for (int g = 0; g < 2; g++) {
      for (int b = 0; b < 2; b++) { mbar_init(s_full(g, b), 1); mbar_init(p_full(g, b), 4); }
      mbar_init(pv_done(g), 1); mbar_init(o_done(g), 1);
      for (int k = 0; k < 4; k++) mbar_init(turn(g, k), 1);
    }
    for (int s = 0; s < kSpRaw; s++) { mbar_init(raw_full(s), 1); mbar_init(raw_empty(s), 4); }
    mbar_init(q_full, 8);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(fail), "r"(0) : "memory");
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (Behind the allocation: a CTA of the next kernel that took its columns first would wait for this grid, and this CTA for those columns.)  The
  // kernel in front let this one start once its own inputs, which are this one's too, were complete: it is waited for at the end
  pdl_launch_dependents();
  if (!a.late_wait) pdl_wait();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  const uint32_t o_base = tmem + 4 * kSpTile;
  const int page_size = 1 << a.page_shift, last_page = (prefix - 1) >> a.page_shift;
  const int *pt = a.page_table + (size_t)a.pt_row[0] * a.max_pages;

  if (!I8 && warp == 0) {
    // ===== K and V tiles by TMA; one lane acts, all hold page numbers
    const int box_rows = min(page_size, kSpTile), last_box = (prefix - 1) / box_rows * box_rows;
    int win_first = 1 << 30, win = 0;
    tma_prefetch_desc(&kv_map);
    int t = 0;
    for (bool ok = true; t < n && ok; t++) {
      const int s = t % NS;
      for (int v = 0; v < 2 && ok; v++) {
        if (t >= NS) ok = sp_wait(v ? v_empty(s) : k_empty(s), (uint32_t)(t / NS - 1) & 1u, fail);
        if (!ok) break;
        const uint32_t full = v ? v_full(s) : k_full(s), dst = base + (v ? Cfg::kV : Cfg::kK) + s * Cfg::kTileBytes;
        if (lane == 0) mbar_expect_tx(full, Cfg::kTileBytes);
        for (int r = 0; r < kSpTile; r += box_rows) {
          const int pos = min((tile0 + t) * kSpTile + r, last_box);  // boxes behind the prefix repeat its last one: their weights are zero
          const int pi = pos >> a.page_shift;
          if (pi < win_first || pi - win_first >= 32) {
            win_first = pi;
            win = pt[min(pi + lane, last_page)];
          }
          const long long page = __shfl_sync(0xffffffffu, win, pi - win_first);
          const long long row = ((page * 2 + v) * a.n_kv + kvh) * page_size + (pos & (page_size - 1));
          if (lane == 0) {
#pragma unroll
            for (int h = 0; h < kHalves; h++) tma_load_2d(dst + h * kSpBlock + r * 128, &kv_map, h * 64, (int)row, full, kEvictLast);
          }
        }
        __syncwarp();
      }
    }
    // Given up: copies that are under way may not outlive this CTA's shared memory.  (After the last tile they were waited for by its readers.)
    if (sp_failed(fail)) {
      const long long began = clock64();
      for (int u = max(0, t - NS); u < t; u++)
        for (int v = 0; v < 2; v++)
          while (!sp_poll(v ? v_full(u % NS) : k_full(u % NS), (uint32_t)(u / NS) & 1u) && __all_sync(0xffffffffu, clock64() - began < kSpPatience)) {}
    }
  } else if (I8 && warp == 0) {
    // ===== 8-bit rows: those of a page that a tile meets are one run of bytes, for K and for V; a lane to a run.  Behind the prefix nothing is
    // copied: what lies there are whole numbers from before, under weights of zero
    const int run = min(page_size, kSpTile);
    int win_first = 1 << 30, win = 0, t = 0;
    for (; t < n; t++) {
      const int st = t % kSpRaw, first = (tile0 + t) * kSpTile, rows = min(kSpTile, prefix - first), p0 = first >> a.page_shift;
      if (t >= kSpRaw && !sp_wait(raw_empty(st), (uint32_t)(t / kSpRaw - 1) & 1u, fail)) break;
      if (p0 < win_first || p0 + 8 - win_first > 32) {  // a tile has at most eight pages
        win_first = p0;
        win = pt[min(p0 + lane, last_page)];
      }
      if (lane == 0) mbar_expect_tx(raw_full(st), 2 * rows * D);
      const int at = lane * run, pos = first + at;
      const long long page = __shfl_sync(0xffffffffu, win, (min(pos >> a.page_shift, last_page) - win_first) & 31);
      if (at < rows) {
        const int8_t *src = a.pool + (((page * 2) * a.n_kv + kvh) * page_size + (pos & (page_size - 1))) * D;
        const uint32_t dst = base + Cfg::kRaw + st * Cfg::kRawBytes + at * D, bytes = min(run, rows - at) * D;
        sp_bulk(dst, src, bytes, raw_full(st));
        sp_bulk(dst + kSpTile * D, src + (long long)a.n_kv * page_size * D, bytes, raw_full(st));
      }
      __syncwarp();
    }
    if (sp_failed(fail)) {  // as above
      const long long began = clock64();
      for (int u = max(0, t - kSpRaw); u < t; u++)
        while (!sp_poll(raw_full(u % kSpRaw), (uint32_t)(u / kSpRaw) & 1u) && __all_sync(0xffffffffu, clock64() - began < kSpPatience)) {}
    }
  } else if (warp == 1 || warp == 2) {
    // ===== MMA issuer of group g: the warp converged, one elected lane issues
    const int g = warp - 1, count = steps(g);
    constexpr uint32_t kTypes = I8 ? (1u << 7) | (1u << 10) : 0u;  // bits that say bf16, off for fp16
    constexpr uint32_t idesc_s = umma_idesc<kSpTile>() & ~kTypes, idesc_o = (umma_idesc<D>() & ~kTypes) | (1u << 16);  // V is MN-major
    const uint32_t q_lo = umma_lo(base + Cfg::kQ + (kPair ? g * kHalves * kSpQBlock : 0)), k_lo = umma_lo(base + Cfg::kK);
    const uint32_t v_lo = umma_lo_mn(base + Cfg::kV, kSpBlock);
    auto issue_s = [&](int i) {
      const int t = tile_of(g, i), s = t % NS;
      if (!sp_wait(k_full(s), (uint32_t)(t / NS) & 1u, fail)) return false;
      if (i >= 2 && !sp_wait(pv_done(g), (uint32_t)i & 1u, fail)) return false;  // S overwrites the columns that the P V two steps before reads
      tc_fence_after();
      if (elect_one()) {
        const uint32_t b = k_lo + s * (Cfg::kTileBytes >> 4), d = tmem + (2 * g + (i & 1)) * kSpTile;
#pragma unroll
        for (uint32_t k = 0; k < D / 16; k++)
          umma_ss(d, q_lo + (k >> 2) * (kSpQBlock >> 4) + (k & 3) * 2, b + (k >> 2) * (kSpBlock >> 4) + (k & 3) * 2, idesc_s, k > 0 ? 1u : 0u);
        umma_commit(s_full(g, i & 1));
        umma_commit(k_empty(s));
      }
      __syncwarp();
      return true;
    };
    bool ok = count > 0 && sp_wait(q_full, 0, fail) && issue_s(0) && (count < 2 || issue_s(1));
    for (int i = 0; i < count && ok; i++) {
      const int t = tile_of(g, i), s = t % NS;
      ok = sp_wait(v_full(s), (uint32_t)(t / NS) & 1u, fail) && sp_wait(p_full(g, i & 1), (uint32_t)(i >> 1) & 1u, fail);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t b = v_lo + s * (Cfg::kTileBytes >> 4), p = tmem + (2 * g + (i & 1)) * kSpTile;
#pragma unroll
        for (uint32_t k = 0; k < kSpTile / 16; k++) umma_ts(o_base + g * D, p + 8 * k, b + k * 128, idesc_o, k > 0 ? 1u : (uint32_t)(i > 0));
        if (!I8) {  // the weights' rests
#pragma unroll
          for (uint32_t k = 0; k < kSpTile / 16; k++) umma_ts(o_base + g * D, p + kSpTile / 2 + 8 * k, b + k * 128, idesc_o, 1u);
        }
        umma_commit(pv_done(g));
        umma_commit(v_empty(s));
        if (i + 1 == count) umma_commit(o_done(g));
      }
      __syncwarp();
      if (i + 2 < count) ok = issue_s(i + 2);
    }
  } else if (warp >= 4 && warp < 12) {
    // ===== softmax: one thread per row; O lives in TMEM
    const int g = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    constexpr float kLog2 = (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f;
    {  // The query rows: K-major, 128B swizzle, rows behind the last zeros; D / 8 lanes take a row.  The eight warps have 16 rows each of the one tile,
       // or a group's four 32 each of the group's
      constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kMine = kPair ? 32 : 16;
      const int c = lane % kLanes, first_row = (kPair ? (warp & 3) : warp - 4) * kMine + lane / kLanes, rho0 = (rt0 + (kPair ? g : 0)) * 128;
      uint4 v[kMine / kAtOnce];
#pragma unroll
      for (int k = 0; k < kMine / kAtOnce; k++) {
        const int rho = rho0 + first_row + k * kAtOnce, t = rho >> a.g_shift;
        v[k] = make_uint4(0u, 0u, 0u, 0u);
        if (t < a.T) v[k] = reinterpret_cast<const uint4 *>(a.q + (((size_t)t * a.n_kv + kvh) * (1 << a.g_shift) + (rho & ((1 << a.g_shift) - 1))) * D)[c];
      }
#pragma unroll
      for (int k = 0; k < kMine / kAtOnce; k++) {
        const int row = first_row + k * kAtOnce;
        if (I8) {  // fp16 after a power of two that brings the row's largest entry to [2^13, 2^14)
          uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w}, big = 0;
#pragma unroll
          for (int j = 0; j < 4; j++) big = max(big, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
#pragma unroll
          for (int o = kLanes >> 1; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int ex = min(max((int)(big >> 7) - 127 - 13, -100), 100);
          const float down = __int_as_float((127 - ex) << 23);
          if (c == 0) reinterpret_cast<float *>(sp_smem + Cfg::kUp)[(kPair ? g * 128 : 0) + row] = __int_as_float((127 + ex) << 23);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 f = bf16x2_to_float2(w[j]);
            const __half2 h = __floats2half2_rn(f.x * down, f.y * down);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
          }
          v[k] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        const uint32_t off = (uint32_t)Cfg::kQ + (kPair ? g * kHalves * kSpQBlock : 0) + (uint32_t)(c >> 3) * kSpQBlock + (uint32_t)(row >> 3) * 1024 +
                             (uint32_t)(row & 7) * 128 + (uint32_t)(((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4 *>(sp_smem + off) = v[k];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }

    float q_up = 1.f;
    if (I8 && sp_wait(q_full, 0, fail)) q_up = reinterpret_cast<const float *>(sp_smem + Cfg::kUp)[(kPair ? g * 128 : 0) + row];
    const int count = steps(g);
    const uint32_t o_addr = o_base + lane_off + g * D;
    float m = kPieceNone, l = 0.f;
    bool ok = true;
    // 8 bits: the two warps of a scheduler take their exponentials in turn, group 0 first, so that one's maximum (scales from shared memory) runs under the
    // other's exponentials: 53.8 -> 52.4 us (64 behind 8000; bf16, whose maximum is short: none)
    if (I8 && g == 1 && lane == 0) mbar_arrive(turn(0, quarter));
    for (int i = 0; i < count; i++) {
      const int t = tile_of(g, i), slot = t % NS;
      ok = sp_wait(s_full(g, i & 1), (uint32_t)(i >> 1) & 1u, fail);
      if (I8 && ok) ok = sp_wait(v_full(slot), (uint32_t)(t / NS) & 1u, fail);  // the tile's scales; they stay until P V has read the tile
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_addr = tmem + lane_off + (2 * g + (i & 1)) * kSpTile;
      float2 s[kSpTile / 2];
      {
        uint32_t raw[2][32];
        tmem_ld_32x32(s_addr, raw[0]);
        tmem_ld_32x32(s_addr + 32, raw[1]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 32; c++) s[c] = make_float2(__uint_as_float(raw[c >> 4][2 * (c & 15)]), __uint_as_float(raw[c >> 4][2 * (c & 15) + 1]));
      }
      const float4 *k_f = reinterpret_cast<const float4 *>(sp_smem + Cfg::kScale + slot * Cfg::kScaleFloats * 4);
      const int rest = prefix - (tile0 + t) * kSpTile;  // keys of the tile that exist
      float2 f2;
      if (I8) {
#pragma unroll
        for (int c = 0; c < 16; c++) {
          const float4 k4 = k_f[c];
          s[2 * c] = sp_mul2(s[2 * c], make_float2(k4.x, k4.y));
          s[2 * c + 1] = sp_mul2(s[2 * c + 1], make_float2(k4.z, k4.w));
        }
        f2 = make_float2(q_up, q_up);
      } else {
        f2 = make_float2(kLog2, kLog2);
      }
      if (rest < kSpTile) {
#pragma unroll
        for (int c = 0; c < 32; c++) {
          if (2 * c >= rest) s[c].x = -INFINITY;
          if (2 * c + 1 >= rest) s[c].y = -INFINITY;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, mx;
      if (I8) {
#pragma unroll
        for (int c = 0; c < 16; c++) {
          const float4 up = k_f[2 * (kSpTile / 4) + c];
          const float2 x = sp_fma2(s[2 * c], f2, make_float2(up.x, up.y)), y = sp_fma2(s[2 * c + 1], f2, make_float2(up.z, up.w));
          mx4[(2 * c) & 3] = sp_max3(mx4[(2 * c) & 3], x.x, x.y);
          mx4[(2 * c + 1) & 3] = sp_max3(mx4[(2 * c + 1) & 3], y.x, y.y);
        }
        mx = sp_max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3]));
      } else {
#pragma unroll
        for (int c = 0; c < 32; c++) mx4[c & 3] = sp_max3(mx4[c & 3], s[c].x, s[c].y);
        mx = sp_max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * kLog2;  // the factor is positive: it commutes with the maximum
      }
      constexpr float kDown = I8 ? kPieceDown : 0.f;
      const bool grow = mx > m + (kPieceLazy + kDown);
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = grow ? mx - kDown : m, f = piece_ex2(m - m_new);
        if (i > 0) {  // O holds the products of every step before this one; none is under way behind it
          ok = sp_wait(pv_done(g), (uint32_t)(i - 1) & 1u, fail);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) sp_rescale_16(o_addr + c, f);
          sp_tmem_st_wait();
        }
        l *= f;
        m = m_new;
      }
      if (I8) {
        ok = sp_wait(turn(g, quarter), (uint32_t)i & 1u, fail);
        if (!ok) break;
      }
      const float2 neg = make_float2(-m, -m);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t w[16], low[16];
#pragma unroll
        for (int c = 0; c < 16; c++) {
          float2 p = sp_fma2(s[16 * h + c], f2, neg);
          p.x = piece_ex2(p.x);
          p.y = piece_ex2(p.y);
          sum[c & 1] = sp_add2(sum[c & 1], p);
          if (I8) {
            const float2 vs = reinterpret_cast<const float2 *>(k_f + kSpTile / 4)[16 * h + c];
            p = sp_mul2(p, vs);
            const __half2 hp = __floats2half2_rn(p.x, p.y);
            w[c] = *reinterpret_cast<const uint32_t *>(&hp);
          } else {
            // two halves, 16 bits of the weight, as decode attention over bf16 pages has them elsewhere
            w[c] = float2_to_bf16x2(p.x, p.y);
            const float2 top = bf16x2_to_float2(w[c]);
            low[c] = float2_to_bf16x2(p.x - top.x, p.y - top.y);
          }
        }
        sp_tmem_st_16(s_addr + 16 * h, w);
        if (!I8) sp_tmem_st_16(s_addr + kSpTile / 2 + 16 * h, low);
      }
      if (I8) {
        __syncwarp();
        if (lane == 0) mbar_arrive(turn(g ^ 1, quarter));
      }
      sp_tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(g, i & 1));
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    // Of the last two products none, one or both may be complete, and pv_done's parity is the same before both and after both: the last has a barrier
    // of its own
    if (ok && count > 0) ok = sp_wait(o_done(g), 0, fail);
    tc_fence_after();
    // ---- the state: of this group's rows (kPair), or of both groups' keys joined, half of the columns each
    float2 *meet = reinterpret_cast<float2 *>(sp_smem + Cfg::kMeet);
    float f0 = 1.f, f1 = 0.f;
    bool other = false;
    if (!kPair) {
      meet[g * 128 + row] = make_float2(m, l);
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      tc_fence_after();
      const float2 x = meet[row], y = meet[128 + row];
      m = fmaxf(x.x, y.x);
      f0 = piece_ex2(x.x - m);
      f1 = piece_ex2(y.x - m);
      other = n > 1;
      l = x.y * f0 + (other ? y.y * f1 : 0.f);
    }
    if (sp_failed(fail)) l = __uint_as_float(0x7fc00000u);  // (a wait ran out: the result says so)
    const int rt = rt0 + (kPair ? g : 0);
    if (rt < a.row_tiles) {  // (uniform)
      const size_t tile = ((size_t)slice * a.n_kv + kvh) * a.row_tiles + rt;
      float4 *dst = reinterpret_cast<float4 *>(a.state_o) + tile * (D / 4) * 128 + row;
      constexpr int kMine = kPair ? D : D / 2;
#pragma unroll
      for (int cc = 0; cc < kMine; cc += 32) {
        const int c = (kPair ? 0 : g * kMine) + cc;
        uint32_t v[32];
        tmem_ld_32x32(o_base + lane_off + (kPair ? g * D : 0) + c, v);
        tmem_ld_wait();
        if (!kPair) {
#pragma unroll
          for (int k = 0; k < 32; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * f0);
          if (other) {
            uint32_t u[32];
            tmem_ld_32x32(o_base + lane_off + D + c, u);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; k++) v[k] = __float_as_uint(fmaf(__uint_as_float(u[k]), f1, __uint_as_float(v[k])));
          }
        }
#pragma unroll
        for (int k = 0; k < 8; k++)
          dst[(size_t)(c / 4 + k) * 128] = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
      }
      if (kPair || g == 0) reinterpret_cast<float2 *>(a.state_ml)[tile * 128 + row] = make_float2(m, l);
    }
  } else if (I8 && warp >= 12) {
    // ===== 8-bit rows to fp16 tiles.  A thread fetches the scale that it turns itself
    const int th = threadIdx.x - 384;
    constexpr int kPer = D / 16, kMine = kSpTile * kPer / 128;  // 16-byte chunks of a row; of K (and of V) for a thread
    const uint32_t raw_s = base + Cfg::kRawScale;
    int win_first = 1 << 30, win = 0;
    auto fetch = [&](int t) {  // scales: threads 0-63 of K, 64-127 of V.  Every lane of a warp looks at rows in order: the page numbers are kept 32 at a time
      if (t < n) {
        const int st = t % kSpRaw, p0 = (tile0 + t) * kSpTile >> a.page_shift;
        if (p0 < win_first || p0 + 8 - win_first > 32) {
          win_first = p0;
          win = pt[min(p0 + lane, last_page)];
        }
        const int r = th & 63, pos = (tile0 + t) * kSpTile + r, pi = min(pos >> a.page_shift, last_page);
        const long long page = __shfl_sync(0xffffffffu, win, pi - win_first);
        const long long row = ((page * 2 + (th >> 6)) * a.n_kv + kvh) * page_size + (pos & (page_size - 1));
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(raw_s + (st * 128 + th) * 4), "l"(a.scale + row), "r"(pos < prefix ? 4 : 0) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int t = 0; t < kSpRaw - 1; t++) fetch(t);
    bool ok = true;
    for (int t = 0; t < n; t++) {
      const int s = t % NS, st = t % kSpRaw;
      fetch(t + kSpRaw - 1);  // into the stage that this thread read last
      asm volatile("cp.async.wait_group %0;" ::"n"(kSpRaw - 1) : "memory");
      ok = sp_wait(raw_full(st), (uint32_t)(t / kSpRaw) & 1u, fail);
      if (!ok) break;
#pragma unroll
      for (int v = 0; v < 2; v++) {
        if (t >= NS) ok = sp_wait(v ? v_empty(s) : k_empty(s), (uint32_t)(t / NS - 1) & 1u, fail);
        if (!ok) break;
        uint8_t *dst = sp_smem + (v ? Cfg::kV : Cfg::kK) + s * Cfg::kTileBytes;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
          const int id = i * 128 + th, r = id / kPer, c = id % kPer;
          const uint4 x = *reinterpret_cast<const uint4 *>(sp_smem + Cfg::kRaw + st * Cfg::kRawBytes + v * kSpTile * D + id * 16);
          uint4 y[2];
          bytes_to_half2(x.x ^ 0x80808080u, y[0].x, y[0].y);
          bytes_to_half2(x.y ^ 0x80808080u, y[0].z, y[0].w);
          bytes_to_half2(x.z ^ 0x80808080u, y[1].x, y[1].y);
          bytes_to_half2(x.w ^ 0x80808080u, y[1].z, y[1].w);
          uint8_t *block = dst + (c >> 2) * kSpBlock + r * 128;
          // lanes of the second 64 dims write their second half first, or a quarter warp would meet half of the banks twice
          const int o = kHalves == 2 ? c >> 2 : 0, e = 2 * (c & 3);
          *reinterpret_cast<uint4 *>(block + (((e + o) ^ (r & 7)) << 4)) = o ? y[1] : y[0];
          *reinterpret_cast<uint4 *>(block + (((e + 1 - o) ^ (r & 7)) << 4)) = o ? y[0] : y[1];
        }
        if (v) {
          const float sc = *reinterpret_cast<const float *>(sp_smem + Cfg::kRawScale + (st * 128 + th) * 4);
          float *to = reinterpret_cast<float *>(sp_smem + Cfg::kScale + s * Cfg::kScaleFloats * 4);
          constexpr float kLog2 = (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f;
          if (th < 64) {
            to[th] = sc * kLog2;
          } else {
            to[th] = sc;
            to[th + 64] = piece_log2_scale(sc);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v ? v_full(s) : k_full(s));
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(raw_empty(st));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc<512>(tmem);
  if (a.late_wait) pdl_wait();
}

// The states of a row joined: thread = (row of a kv head, eight dims), lanes over rows, as the prefix's states lie.
constexpr int kSjRows = 32, kSjUnroll = 6;

template <int D>
__global__ void __launch_bounds__(128)
attn_join_kernel(const SpArgs a, const float *__restrict__ own_o, const float *__restrict__ own_ml, const int *__restrict__ ctx, uint16_t *__restrict__ out) {
  const int rho = blockIdx.x * kSjRows + (threadIdx.x & 31), chunk = blockIdx.y * 4 + (threadIdx.x >> 5), kvh = blockIdx.z;
  const int G = 1 << a.g_shift, t = rho >> a.g_shift;
  // A product whose weights are fetched in front of its wait gains 2.6 us a layer by starting here (an engine's step of 32 behind 4096 tokens, four layers: 520 ->
  // 509 us); the next call's first kernel only fills the SMs up while it waits (64 behind 8000, calls in a row: 50.9 -> 53.0)
  if (a.let_next) pdl_launch_dependents();
  pdl_wait();
  if (t >= a.T) return;
  const size_t head = ((size_t)t * a.n_kv + kvh) * G + (rho & (G - 1));
  const float2 ml = reinterpret_cast<const float2 *>(own_ml)[head];
  const float4 *x = reinterpret_cast<const float4 *>(own_o + head * D + chunk * 8);
  float M = ml.x, l = ml.y;
  float4 o0 = x[0], o1 = x[1];
  const int slices = ctx[t] < (a.prefix_at ? *a.prefix_at : a.prefix) ? 0 : a.slices;
  const size_t step = (size_t)a.n_kv * a.row_tiles;
  const size_t tile = (size_t)kvh * a.row_tiles + (rho >> 7);
  for (int s0 = 0; s0 < slices; s0 += kSjUnroll) {
    float2 y[kSjUnroll];
    float4 u[kSjUnroll], w[kSjUnroll];
#pragma unroll
    for (int j = 0; j < kSjUnroll; j++)
      if (s0 + j < slices) {
        const size_t at = tile + (s0 + j) * step;
        y[j] = reinterpret_cast<const float2 *>(a.state_ml)[at * 128 + (rho & 127)];
        const float4 *src = reinterpret_cast<const float4 *>(a.state_o) + (at * (D / 4) + 2 * chunk) * 128 + (rho & 127);
        u[j] = src[0];
        w[j] = src[128];
      }
#pragma unroll
    for (int j = 0; j < kSjUnroll; j++)
      if (s0 + j < slices) {
        const float m_new = fmaxf(M, y[j].x), f = piece_ex2(M - m_new), g = piece_ex2(y[j].x - m_new);
        M = m_new;
        l = l * f + y[j].y * g;
        o0.x = o0.x * f + u[j].x * g; o0.y = o0.y * f + u[j].y * g; o0.z = o0.z * f + u[j].z * g; o0.w = o0.w * f + u[j].w * g;
        o1.x = o1.x * f + w[j].x * g; o1.y = o1.y * f + w[j].y * g; o1.z = o1.z * f + w[j].z * g; o1.w = o1.w * f + w[j].w * g;
      }
  }
  uint32_t *to = reinterpret_cast<uint32_t *>(out + head * D + chunk * 8);
  const bool none = ctx[t] <= 0;
  to[0] = none ? 0u : float2_to_bf16x2(o0.x / l, o0.y / l);
  to[1] = none ? 0u : float2_to_bf16x2(o0.z / l, o0.w / l);
  to[2] = none ? 0u : float2_to_bf16x2(o1.x / l, o1.y / l);
  to[3] = none ? 0u : float2_to_bf16x2(o1.z / l, o1.w / l);
}

// ---------------------------------------------------------------------------------------- host
// Slices of the prefix: the number that ends soonest where a round of CTAs is 148 and a CTA's start and end cost as much as six tiles
static int shared_row_tiles(int T, int G) { return (int)(((long long)T * G + 127) / 128); }
static int shared_slice_limit(int blocks) { return std::min(kSpMaxSlices, std::max(1, 2 * kNumSMs / blocks)); }
static int shared_slices(int blocks, int tiles) {
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::min(shared_slice_limit(blocks), tiles); s++) {
    const double t = (double)(((long long)blocks * s + kNumSMs - 1) / kNumSMs) * ((tiles + s - 1) / s + 6);
    if (t < least) { least = t; best = s; }
  }
  return best;
}
static int shared_blocks(int T, int G, int n_kv) { const int rt = shared_row_tiles(T, G); return (rt > 1 ? (rt + 1) / 2 : 1) * n_kv; }

// Whether the prefix is read once, or every token goes alone (one kernel, to which the others' reads of the same pages are hits in L2): from 2^25 entries of T
// prefixes on the former is ahead; heads of 128 in two tiles of rows or more, and in 8 bits, each cross a quarter later.  From graphs, own parts of 100,
// together / alone, us, at 1 and 1.25 times 2^25 entries:
//   32 / 8 heads of 128, bf16   16 tokens 17.3 / 19.5, 16.8 / 22.2;  32: 18.5 / 19.6, 15.9 / 21.9;  64 (two tiles): 19.7 / 21.5, 20.2 / 23.8
//   the same in 8 bits          16: 18.8 / 19.2, 17.6 / 22.0;  32: 20.7 / 19.5, 17.1 / 21.7;  64: 21.3 / 21.3, 21.9 / 23.4
//   64 / 8 heads, 8 bits        16: 20.3 / 21.0, 18.8 / 23.8;  32 (two tiles): 25.2 / 21.2, 21.8 / 23.5;  64: 25.1 / 23.3, 24.0 / 25.5
//   32 / 4 heads of 64, 8 bits  16: 18.0 / 23.2, 18.6 / 25.9;  64 (four tiles): 19.8 / 21.5, 20.5 / 24.4
// A few tokens make little of a product's 128 rows: two or three over bf16 pages cross at 2 times 2^25 (2 tokens at 1, 1.5, 2, 4: 28.5 / 24.2, 35.0 / 32.3,
// 40.8 / 39.3, 63.5 / 87.1; 4 tokens at 1: 19.5 / 21.5).  Over 8-bit pages, which have to be turned to fp16 as well, fewer than six go alone at every length.  For two
// that is ahead to 131072 tokens of 8 heads of 128 at least (128.4 / 100.2).  A prefix read once passes three somewhere between 32768 and 131072 (45.9 / 42.0, 129 / 145), four
// near 25000 (8192 21.7 / 21.1, 32768 46.1 / 49.7), five before 8192 (21.7 / 23.9; 131072 130 / 211); of 4 heads of 64 four are level at 131072 (59.9 / 59.4): what so few
// could gain there the rule leaves aside.
bool attn_shared_pays(int T, int n_heads, int n_kv, int d, int prefix, bool int8) {
  if (T < (int8 ? 6 : 2) || n_kv < 1) return false;
  if (n_kv > 65535 || shared_row_tiles(T, std::max(n_heads / n_kv, 1)) > 65535) return false;  // (a grid's sides)
  const int quarters = (T < 4 ? 8 : 4) + (d == 128 ? (T > 128 / std::max(n_heads / n_kv, 1)) + int8 : 0);
  return (long long)T * prefix * n_kv * d >= (long long)quarters << 23;
}

int attn_shared_slices(int T, int n_heads, int n_kv, int d, int prefix, bool int8) {
  if (!attn_shared_pays(T, n_heads, n_kv, d, prefix, int8)) return 0;
  return shared_slices(shared_blocks(T, n_heads / n_kv, n_kv), (prefix + kSpTile - 1) / kSpTile);
}

size_t attn_shared_scratch_elems(int T, int n_heads, int n_kv, int d) {  // the stream's, its states, the slices' states
  if (T <= 0 || n_kv <= 0 || n_heads < n_kv || d <= 0) return 0;
  const int G = n_heads / n_kv, rt = shared_row_tiles(T, G);
  return (attn_stream_scratch_elems(n_heads, n_kv, d) + 3) / 4 * 4 + ((size_t)T * n_heads * (2 + (size_t)d) + 3) / 4 * 4 +
         (size_t)shared_slice_limit(shared_blocks(T, G, n_kv)) * n_kv * rt * 128 * (2 + (size_t)d);
}

template <int D, bool I8, bool kPair>
static cudaError_t prefix_launch(const TmaMap &map, const SpArgs &a, cudaStream_t st) {
  using Cfg = SpCfg<D, I8, kPair>;
  static_assert(Cfg::kSmem <= 227 * 1024 && Cfg::kRing <= 8, "");
  auto kern = attn_prefix_kernel<D, I8, kPair>;
  static DeviceOnce once;
  DIS_CUDA_TRY(once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem); }));
  return launch_k(kern, dim3(a.slices, kPair ? (a.row_tiles + 1) / 2 : a.row_tiles, a.n_kv), dim3(Cfg::kThreads), (size_t)Cfg::kSmem, st,
                  *reinterpret_cast<const CUtensorMap *>(&map), a);
}

cudaError_t launch_attn_shared(const uint16_t *q, const void *pool, const float *scale, long long n_pages, const int *page_table, int max_pages,
                               const int *pt_row, const int *ctx, int prefix, const int *prefix_at, uint16_t *out, float *scratch, int T, int n_heads, int n_kv,
                               int d, int page_size, bool chain, cudaStream_t st) {
  const int G = n_heads / n_kv;
  const int slices = attn_shared_slices(T, n_heads, n_kv, d, prefix, scale != nullptr);
  if (slices == 0)
    return launch_attn_stream(q, pool, scale, page_table, max_pages, pt_row, ctx, 0, nullptr, out, nullptr, nullptr, scratch, false, T, n_heads, n_kv, d, page_size, st);
  SpArgs a{};
  a.q = q; a.pool = static_cast<const int8_t *>(pool); a.scale = scale; a.page_table = page_table; a.pt_row = pt_row; a.max_pages = max_pages;
  while ((1 << a.page_shift) < page_size) a.page_shift++;
  while ((1 << a.g_shift) < G) a.g_shift++;
  a.T = T; a.n_kv = n_kv; a.prefix = prefix; a.prefix_at = prefix_at;
  a.row_tiles = shared_row_tiles(T, G);
  a.slices = slices;
  float *own_o = scratch + (attn_stream_scratch_elems(n_heads, n_kv, d) + 3) / 4 * 4, *own_ml = own_o + (size_t)T * n_heads * d;
  a.state_o = own_o + ((size_t)T * n_heads * (2 + (size_t)d) + 3) / 4 * 4;
  a.state_ml = a.state_o + (size_t)a.slices * n_kv * a.row_tiles * 128 * d;
  TmaMap map{};
  if (!scale) DIS_CUDA_TRY(make_kv_map(&map, static_cast<const uint16_t *>(pool), n_pages * 2 * n_kv * page_size, d, page_size));
  // The own parts first: their CTAs end one after the other, and the prefix's start as SMs come free
  DIS_CUDA_TRY(launch_attn_stream(q, pool, scale, page_table, max_pages, pt_row, ctx, prefix, prefix_at, nullptr, own_o, own_ml, scratch, true, T, n_heads, n_kv,
                                  d, page_size, st));
  // (chain, a call of the C ABI: the kernels behind the first overlap with the one in front of them even under capture, where the first may not with what is in
  // front of it)
  struct Pdl { const bool was = pdl_enabled(); ~Pdl() { pdl_enabled() = was; } } pdl;
  pdl_enabled() |= chain;
  a.let_next = !chain;
  a.late_wait = pdl_enabled();
  const bool pair = a.row_tiles > 1;
#define DIS_SP(DD, II, PP) DIS_CUDA_TRY((prefix_launch<DD, II, PP>(map, a, st)))
  if (d == 128) {
    if (scale) { if (pair) DIS_SP(128, true, true); else DIS_SP(128, true, false); }
    else { if (pair) DIS_SP(128, false, true); else DIS_SP(128, false, false); }
  } else {
    if (scale) { if (pair) DIS_SP(64, true, true); else DIS_SP(64, true, false); }
    else { if (pair) DIS_SP(64, false, true); else DIS_SP(64, false, false); }
  }
#undef DIS_SP
  const dim3 grid((unsigned)((T * G + kSjRows - 1) / kSjRows), d / 32, n_kv);
  if (d == 128) return launch_k(attn_join_kernel<128>, grid, dim3(128), 0, st, a, (const float *)own_o, (const float *)own_ml, ctx, out);
  return launch_k(attn_join_kernel<64>, grid, dim3(128), 0, st, a, (const float *)own_o, (const float *)own_ml, ctx, out);
}

}  // namespace dis
