// k_attn_stream.cu -- attention of single query tokens over paged keys and values, 8-bit (dis_k_attn_paged_i8) or bf16 (the own parts of
// dis_k_attn_shared): softmax(q K^T / sqrt d) V for all query heads of a kv head at once.
//
// 8-bit rows: k = ks k8, v = vs v8 with whole numbers k8, v8 and one fp32 factor per token and kv head.  The factors stay outside the products:
//   s_j = (q . k8_j) ks_j / sqrt d,   o = sum_j (p_j vs_j) v8_j / sum_j p_j,   p_j = 2^(s_j - m)
// so the operands are exact in fp16 or nearly: k8 and v8 by themselves, q after a power of two per head that brings its largest entry to
// [2^13, 2^14) (entries below 2^-28 of it lose bits), and p_j vs_j because m follows the largest s_j + log2 vs_j instead of the largest s_j, 2^7 below
// it: no product is above 2^15, and each loses 2^-11 of itself at most (bf16: 2^-8) or, below 2^-14, 2^-25, which is 2^-32 of the largest.  Which m a softmax
// is taken under cancels; vs below 2^-80 counts as that in m, so that sum p_j stays within fp32.  m, l, O and the scores are fp32.
//
// HBM-bound: 2 (d + 4) bytes (i8) or 4 d (bf16) per token and kv head, 4 G d operations on mma.sync m16n8k16 (tokens are its rows, the up to eight
// heads its columns: S^T = K Q^T, O^T = V^T P^T).  Operands go from shared memory to registers by 16-byte loads without ldmatrix: which dim is
// which k index of K Q^T is free as long as Q agrees, so a lane's 16 bytes of a K row are its operand of four k-steps; and a lane's 16 dims of two
// V rows, bytes interleaved, are its operand of eight m-tiles, the transposition being part of the conversion.
//
// Work: the histories of all (token, kv head) pairs laid end to end in tiles of 16 tokens, cut into equal shares, one per
// resident CTA, whatever the lengths are: lengths are read on the device, nothing depends on their maximum.  The CTA's four warps take its
// tiles in turn, each with a ring of its own filled by cp.async (no barrier of the block per tile, nothing to spin on), and merge their states at
// the end of a history's piece.  A history in several CTAs is finished by whichever of them ends last, which adds the pieces in the
// order of the history (more than eight of them in about sqrt(n) groups first, each added by the last CTA of the group): the result does not
// depend on who that is.
//
// Measured (B200, 8 bits, from graphs; time at 6.54 TB/s, a plain copy's rate, beside it): 32 histories to 6000 tokens, 32 / 8 heads of 128, 29.7 us
// (19.4); two to 60000, 64 / 8 heads, 37 (21.7); 64 to 3000, 32 / 4 heads of 64, 15.5 (5.3); four to 500 7.9 (0.3).  In the middle of a long
// launch rows come in at 6 to 6.9 TB/s.  The rest: 2.5 to 5 us until every ring has been filled once, 2 to 3 us from the last row to the
// result (states met in shared memory 0.5 to 1, count 0.9, join 1 a level), and CTAs of equal shares that end up to 15 % apart.  (Tiles taken
// as warps come free would even that out, and make the sums' order, so the result's last bits, differ from call to call.)
#include <algorithm>

#include <cuda_fp16.h>

#include "attn_piece.cuh"

namespace dis {

constexpr int kStWarps = 4;
constexpr int kStMaxT = 512;            // tokens of one launch
constexpr int kStCounters = 1 << 16;    // words kept for counters, of which two for each of a CTA's two pieces are used
constexpr int kStMinShare = kStWarps;   // tiles of a CTA, at least
constexpr int kSmSmem = 228 * 1024;     // shared memory of an SM, of which a CTA takes 1 KB besides its own, in units of 128 bytes
constexpr int kStStatic = (2 * kStWarps * 8 + kStWarps + 2) * 4;  // static shared memory of the kernel

template <int D, bool I8>
struct StCfg {
  static constexpr int kTok = 16;                         // tokens of a tile
  static constexpr int kRow = D * (I8 ? 1 : 2);           // bytes of a row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPart = kTok * kRow;               // K or V of a tile
  static constexpr int kStage = 2 * kPart + (I8 ? 2 * kTok * 4 : 0);
  static constexpr int kHead = 16 * (D / 16 + 1) + 4;     // floats between two heads' O in the merge: no bank twice in a half warp
  // Stages of a warp and CTAs of an SM, us of (8 bits) 32 histories to 6000, two of 60000, 64 of heads of 64; (bf16) 32 requests behind 6000 tokens: heads of
  // 128 in 8 bits 3, 3: 30.4, 39.4; 2, 4: 31.0, 39.0; 4, 2: 32.1, 38.2; heads of 64 4, 4: 16.4; 3, 3 (tiles of 32 tokens): 18.3; bf16 2, 3: 26.2; 3, 2: 27.4
  static constexpr int kStages = I8 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2);
  static constexpr int kCtas = I8 && D == 64 ? 4 : 3;
  static constexpr int kRing = kStWarps * kStages * kStage;
  static constexpr int meet(int G) { return G * D <= 512 ? G : 512 / D; }  // heads whose states meet in shared memory at a time
  static constexpr int fixed(int G) { return kRing + kStWarps * meet(G) * kHead * 4; }
};

// Where row r's 16-byte chunk c of a tile lies, in chunks: a quarter warp's loads (K: two rows, four chunks; V: two chunks of four rows, every
// second one) meet every bank once.
template <int D, bool I8>
__device__ __forceinline__ int st_k_chunk(int r, int c) {
  if (I8 && D == 64) return r * 4 + c;
  return r * StCfg<D, I8>::kChunks + (c ^ ((r & 1) << 2));
}
template <int D, bool I8>
__device__ __forceinline__ int st_v_chunk(int r, int c) {
  const int t = (r >> 1) & 3;
  if (I8 && D == 64) return (r ^ (t & 1)) * 4 + (c ^ (t & 2));
  if (!I8 && D == 128) return r * 16 + (c ^ ((t & 1) | ((t & 2) << 1)));
  return r * 8 + (c ^ (t << 1));
}

__device__ __forceinline__ void st_copy_16(uint32_t dst, const void *src, bool in) {  // zeros where the row is not visible
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void st_copy_4(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void st_copy_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void st_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 st_lds_16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 st_lds_8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float st_lds_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
template <bool I8>
__device__ __forceinline__ void st_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (I8)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t st_transpose(uint32_t v) {  // an 8x8 matrix of pairs across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// floats of a piece's (m, l): whole 16 bytes
__host__ __device__ constexpr int st_ml(int G) { return G < 2 ? 4 : 2 * G; }

__host__ __device__ constexpr size_t stream_slots() { return 2 * 4 * (size_t)kNumSMs; }  // two of each resident CTA

struct StArgs {
  const uint16_t *q;
  const void *pool;
  const float *scale;      // I8
  const int *page_table;
  int max_pages;
  const int *pt_row, *ctx;
  int first;               // keys in front of this position are somebody else's, for the tokens that reach it
  const int *first_at;     // where that position is instead (kAt), or nullptr
  uint16_t *out;           // the result, or nullptr: the states go to state_o, state_ml
  float *state_o, *state_ml;
  int *counters;           // [2][2 per CTA], zero between calls
  float *piece_o, *piece_ml;  // [2 per CTA][G][D], [2 per CTA][st_ml(G)]
  float *group_o, *group_ml;  // of pieces joined, likewise
  int T, n_kv, page_shift;
  int inputs_first;        // the kernel behind reads the same inputs and does not wait for them: it may start when they are complete
};

// A tile at a history's start or end, or over pages that end inside it, row by row: zeros where they are not visible.  (Not inlined: the kernel runs
// this seldom, and how long its code is counts in every launch.)
template <int D, bool I8>
__device__ __noinline__ void st_fetch_rows(uint32_t dst, const char *pool, const float *scale, const int *pt, int pos0, int first, int keys, int page_shift,
                                           int n_kv, int h) {
  using Cfg = StCfg<D, I8>;
  constexpr int kLaneRows = 32 / Cfg::kChunks;
  const int lane = threadIdx.x & 31, lc = lane % Cfg::kChunks;
  const long long v_rows = (long long)n_kv << page_shift;
#pragma unroll 1
  for (int r = lane / Cfg::kChunks; r < Cfg::kTok; r += kLaneRows) {
    const int pos = pos0 + r;
    const bool in = pos >= first && pos < keys;
    const int at = min(max(pos, first), keys - 1);
    const long long row = (((long long)pt[at >> page_shift] * 2 * n_kv + h) << page_shift) + (at & ((1 << page_shift) - 1));
    st_copy_16(dst + st_k_chunk<D, I8>(r, lc) * 16, pool + row * Cfg::kRow + lc * 16, in);
    st_copy_16(dst + Cfg::kPart + st_v_chunk<D, I8>(r, lc) * 16, pool + (row + v_rows) * Cfg::kRow + lc * 16, in);
    if (I8 && lc == 0) {
      st_copy_4(dst + 2 * Cfg::kPart + r * 4, scale + row, in);
      st_copy_4(dst + 2 * Cfg::kPart + (Cfg::kTok + r) * 4, scale + row + v_rows, in);
    }
  }
}

// kAt: `first` is read from a.first_at.  (As a branch of the one kernel 64 histories of heads of 64 take 15.5 us, not 15.2, four to 500 8.1, not 8.0)
template <int D, int G, bool I8, bool kAt>
__global__ void __launch_bounds__(kStWarps * 32, StCfg<D, I8>::kCtas)
attn_stream_kernel(const StArgs a) {
  using Cfg = StCfg<D, I8>;
  constexpr int KS = D / 16;
  constexpr int kPer = D / 8;                    // dims of a lane's V operand
  constexpr bool kTwice = !I8 && G <= 4;         // bf16 weights in two halves, the rest through columns of its own or (G = 8) a product of its own
  constexpr int kCols = kTwice ? 2 * G : G, kMeet = Cfg::meet(G);
  extern __shared__ __align__(16) uint8_t st_smem[];
  float *s_o = reinterpret_cast<float *>(st_smem + Cfg::kRing);  // [warp][kMeet heads][kHead]
  int *s_tiles = reinterpret_cast<int *>(s_o + kStWarps * kMeet * Cfg::kHead);  // [T + 1]: tiles of a kv head in front of token t
  int *s_keys = s_tiles + a.T + 1, *s_row = s_keys + a.T;                          // [T] keys, page-table rows
  __shared__ float s_m[kStWarps][8], s_l[kStWarps][8];
  __shared__ int s_scan[kStWarps], s_last[2];

  const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  pdl_wait();
  if (a.inputs_first) pdl_launch_dependents();
  const int n_heads = a.n_kv * G, page_size = 1 << a.page_shift, first_own = kAt ? *a.first_at : a.first, base0 = first_own / Cfg::kTok * Cfg::kTok;
  auto first_of = [&](int keys) { return keys < first_own ? 0 : first_own; };  // a history that ends in front of it is all this kernel's
  auto base_of = [&](int keys) { return keys < first_own ? 0 : base0; };

  // ---- tiles in front of each token; tokens without keys of their own get their result here
  for (int t0 = 0, sum = 0; t0 < a.T; t0 += kStWarps * 32) {
    const int t = t0 + threadIdx.x;
    int n = 0;
    if (t < a.T) {
      const int keys = min(a.ctx[t], a.max_pages << a.page_shift);
      s_row[t] = a.pt_row[t];
      s_keys[t] = keys;
      n = keys > first_of(keys) ? (keys - base_of(keys) + Cfg::kTok - 1) / Cfg::kTok : 0;
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
    for (int w = 0; w < kStWarps; w++) {
      if (w < warp) before += s_scan[w];
      sum += s_scan[w];
    }
    if (t < a.T) s_tiles[t + 1] = before + x;
    __syncthreads();
  }
  if (threadIdx.x == 0) s_tiles[0] = 0;
  __syncthreads();
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
    if (s_tiles[t + 1] > s_tiles[t]) continue;
    for (int i = threadIdx.x; i < n_heads * D; i += kStWarps * 32) {
      if (a.out) a.out[(size_t)t * n_heads * D + i] = 0;
      else a.state_o[(size_t)t * n_heads * D + i] = 0.f;
    }
    if (!a.out)
      for (int i = threadIdx.x; i < n_heads; i += kStWarps * 32) {
        a.state_ml[((size_t)t * n_heads + i) * 2] = kPieceNone;
        a.state_ml[((size_t)t * n_heads + i) * 2 + 1] = 0.f;
      }
  }

  const int total = s_tiles[a.T] * a.n_kv;
  const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kStMinShare);
  const int lo = (int)min((long long)total, (long long)blockIdx.x * share), hi = min(total, lo + share);

  // A walk over the (token, kv head) pairs; [u0, u1) are the pair's tiles
  struct Cursor { int t, h, u0, u1; };
  auto next_pair = [&](Cursor &c) {
    c.u0 = c.u1;
    if (++c.h == a.n_kv) {
      c.h = 0;
      do c.t++;
      while (s_tiles[c.t + 1] == s_tiles[c.t]);
    }
    c.u1 = c.u0 + s_tiles[c.t + 1] - s_tiles[c.t];
  };
  Cursor cur{0, 0, 0, 0};
  if (lo < hi) {
    int b = 0, e = a.T;  // the last token with s_tiles[t] * n_kv <= lo
    while (e - b > 1) {
      const int mid = (b + e) >> 1;
      if (s_tiles[mid] * a.n_kv <= lo) b = mid;
      else e = mid;
    }
    const int n = s_tiles[b + 1] - s_tiles[b], at = s_tiles[b] * a.n_kv;
    cur.t = b;
    cur.h = (lo - at) / n;
    cur.u0 = at + cur.h * n;
    cur.u1 = cur.u0 + n;
  }

  // ---- the ring: this warp's tiles lo + warp, lo + warp + 4, ..
  const uint32_t ring = smem_u32(st_smem) + warp * Cfg::kStages * Cfg::kStage;
  Cursor ahead = cur;
  int fetch = lo + warp, into = 0;                      // next tile to fetch, and its stage
  int a_t = -1, a_keys = 0, a_first = 0, a_base = 0, win_first = 0, win = 0;  // of token a_t; 32 page numbers, one in each lane
  const int *a_pt = nullptr;
  // A tile inside a page is one run of bytes: copy i of a lane is 512 bytes behind copy i - 1, there and (but for V's turn) here
  constexpr int kCopies = Cfg::kPart / 512, kLaneRows = 32 / Cfg::kChunks;
  const int lr = lane / Cfg::kChunks, lc = lane % Cfg::kChunks;
  const uint32_t k_to = st_k_chunk<D, I8>(lr, lc) * 16;
  uint32_t v_to[4];  // V's rows turn in eights
#pragma unroll
  for (int i = 0; i < 4; i++) v_to[i] = Cfg::kPart + st_v_chunk<D, I8>(i * kLaneRows % 8 + lr, lc) * 16 - i * kLaneRows % 8 * Cfg::kRow;
  const long long v_rows = (long long)a.n_kv << a.page_shift;
  const uint32_t lane_scale = (lane & 15) * 4 + (lane < 16 ? 0 : Cfg::kTok * 4) + 2 * Cfg::kPart;
  const long long lane_scale_row = (lane & 15) + (lane < 16 ? 0 : v_rows);
  auto page_of = [&](int pi, int last) {
    if (pi < win_first || pi - win_first >= 32) {
      win_first = pi;
      win = a_pt[min(pi + lane, last)];
    }
    return (long long)__shfl_sync(0xffffffffu, win, pi - win_first);
  };
  auto fetch_next = [&] {
    if (fetch < hi) {
      if (fetch >= ahead.u1) {
        do next_pair(ahead);
        while (fetch >= ahead.u1);
        // its queries, on their way to L1 while the tiles in front of its first are taken
        if (lane < G * D / 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.q + ((size_t)ahead.t * n_heads + ahead.h * G) * D + lane * 64));
      }
      if (ahead.t != a_t) {
        a_t = ahead.t;
        a_keys = s_keys[a_t];
        a_first = first_of(a_keys);
        a_base = base_of(a_keys);
        a_pt = a.page_table + (size_t)s_row[a_t] * a.max_pages;
        win_first = 1 << 30;
      }
      const int pos0 = a_base + (fetch - ahead.u0) * Cfg::kTok, last_page = (a_keys - 1) >> a.page_shift;
      const uint32_t dst = ring + into * Cfg::kStage;
      const char *pool = reinterpret_cast<const char *>(a.pool);
      if (pos0 >= a_first && pos0 + Cfg::kTok <= a_keys && page_size >= Cfg::kTok) {
        const long long row = ((page_of(pos0 >> a.page_shift, last_page) * 2 * a.n_kv + ahead.h) << a.page_shift) + (pos0 & (page_size - 1));
        const char *k_src = pool + row * Cfg::kRow + lane * 16, *v_src = k_src + v_rows * Cfg::kRow;
#pragma unroll
        for (int i = 0; i < kCopies; i++) {
          st_copy_16(dst + k_to + i * 512, k_src + i * 512, true);
          st_copy_16(dst + v_to[i & 3] + i * 512, v_src + i * 512, true);
        }
        if (I8) {
          st_copy_4(dst + lane_scale, a.scale + row + lane_scale_row, true);
        }
      } else {
        st_fetch_rows<D, I8>(dst, pool, a.scale, a_pt, pos0, a_first, a_keys, a.page_shift, a.n_kv, ahead.h);
      }
      fetch += kStWarps;
    }
    into = into + 1 == Cfg::kStages ? 0 : into + 1;
    st_copy_end();
  };

  constexpr float kScale = (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f;  // scores are kept in the log2 domain
  int tile = lo + warp, stage = 0;
  if (lo < hi) {
#pragma unroll 1
    for (int i = 0; i < Cfg::kStages - 1; i++) fetch_next();
  }
  auto put = [&](size_t head, int i, float4 o, float m, float l) {  // four dims of a token's head
    if (a.out) {
      uint32_t *to = reinterpret_cast<uint32_t *>(a.out + head * D + i);
      to[0] = float2_to_bf16x2(o.x / l, o.y / l);
      to[1] = float2_to_bf16x2(o.z / l, o.w / l);
    } else {
      *reinterpret_cast<float4 *>(a.state_o + head * D + i) = o;
      if (i == 0) *reinterpret_cast<float2 *>(a.state_ml + head * 2) = make_float2(m, l);
    }
  };
  size_t part_row[2] = {0, 0};
  int part_first[2] = {0, 0}, part_last[2] = {0, 0};
  while (lo < hi) {
    // ================= one piece: tiles [max(u0, lo), min(u1, hi)) of a pair
    float oacc[KS][4];  // O^T: dims g kPer + 2 m (+ 1) of columns 2 tq (+ 1): {dim, column}, {dim, column + 1}, {dim + 1, column}, ..
#pragma unroll
    for (int m = 0; m < KS; m++) { oacc[m][0] = 0.f; oacc[m][1] = 0.f; oacc[m][2] = 0.f; oacc[m][3] = 0.f; }
    float m_run[2] = {kPieceNone, kPieceNone}, l_run[2] = {0.f, 0.f};
    const int end = min(cur.u1, hi), keys = s_keys[cur.t], first = first_of(keys), base = base_of(keys);
    // Q as the B operand: column g is head g (kTwice: the next G columns repeat it)
    uint32_t qb[KS][2];
    float qf[2] = {kScale, kScale};  // factor of the scores of columns 2 tq, 2 tq + 1
    {
      const bool has = g < kCols;
      const uint4 *qp = reinterpret_cast<const uint4 *>(a.q + ((size_t)cur.t * n_heads + cur.h * G + (has ? g % G : 0)) * D);
      if constexpr (I8) {
        uint4 raw[D / 64][2];
#pragma unroll
        for (int i = 0; i < D / 64; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) raw[i][j] = has ? qp[(tq + 4 * i) * 2 + j] : make_uint4(0u, 0u, 0u, 0u);
        uint32_t big = 0;  // largest magnitude's bits (a NaN's are above infinity's)
#pragma unroll
        for (int i = 0; i < D / 64; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t w[4] = {raw[i][j].x, raw[i][j].y, raw[i][j].z, raw[i][j].w};
#pragma unroll
            for (int k = 0; k < 4; k++) big = max(big, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
          }
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // exponent of the factor, kept where the factor and its inverse are normal numbers; infinities and NaN go through as they are
        const int ex = min(max((int)(big >> 7) - 127 - 13, -100), 100);
        const float down = __int_as_float((127 - ex) << 23), up = __int_as_float((127 + ex) << 23);
#pragma unroll
        for (int i = 0; i < D / 64; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t w[4] = {raw[i][j].x, raw[i][j].y, raw[i][j].z, raw[i][j].w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float2 f = bf16x2_to_float2(w[k]);
              const __half2 h = __floats2half2_rn(f.x * down, f.y * down);
              qb[i * 4 + j * 2 + (k >> 1)][k & 1] = *reinterpret_cast<const uint32_t *>(&h);
            }
          }
        qf[0] *= __shfl_sync(0xffffffffu, up, tq * 8);
        qf[1] *= __shfl_sync(0xffffffffu, up, tq * 8 + 4);
      } else {
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const uint4 w = has ? qp[tq + 4 * i] : make_uint4(0u, 0u, 0u, 0u);
          qb[2 * i][0] = w.x; qb[2 * i][1] = w.y; qb[2 * i + 1][0] = w.z; qb[2 * i + 1][1] = w.w;
        }
      }
    }
    for (; tile < end; tile += kStWarps) {
      st_copy_wait<Cfg::kStages - 2>();
      __syncwarp();
      fetch_next();  // into the stage that was read last
      const uint32_t at = ring + stage * Cfg::kStage;
      stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
      const int pos0 = base + (tile - cur.u0) * Cfg::kTok;
      // ---- S^T = K Q^T: tokens g, g + 8, columns 2 tq (+ 1); two accumulators halve the chain
      float sa[2][4];
#pragma unroll
      for (int e = 0; e < 2; e++) { sa[e][0] = 0.f; sa[e][1] = 0.f; sa[e][2] = 0.f; sa[e][3] = 0.f; }
#pragma unroll
      for (int i = 0; i < Cfg::kChunks / 4; i++) {
        const uint4 x4 = st_lds_16(at + st_k_chunk<D, I8>(g, tq + 4 * i) * 16), y4 = st_lds_16(at + st_k_chunk<D, I8>(g + 8, tq + 4 * i) * 16);
        const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
        if constexpr (I8) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t a0, a1, a2, a3;
            bytes_to_half2(x[j] ^ 0x80808080u, a0, a2);
            bytes_to_half2(y[j] ^ 0x80808080u, a1, a3);
            st_mma<I8>(sa[j & 1], a0, a1, a2, a3, qb[i * 4 + j][0], qb[i * 4 + j][1]);
          }
        } else {
          st_mma<I8>(sa[0], x[0], y[0], x[1], y[1], qb[2 * i][0], qb[2 * i][1]);
          st_mma<I8>(sa[1], x[2], y[2], x[3], y[3], qb[2 * i + 1][0], qb[2 * i + 1][1]);
        }
      }
      // ---- the reference follows the maximum where that grows by more than kPieceLazy; the whole warp acts then
      float k_f[2] = {1.f, 1.f}, v_f[2] = {1.f, 1.f};
      if (I8) {
        const uint32_t sc = at + 2 * Cfg::kPart + g * 4;
        k_f[0] = st_lds_f(sc); k_f[1] = st_lds_f(sc + 32);
        v_f[0] = st_lds_f(sc + Cfg::kTok * 4); v_f[1] = st_lds_f(sc + Cfg::kTok * 4 + 32);
      }
      const float up0 = I8 ? piece_log2_scale(v_f[0]) : 0.f, up1 = I8 ? piece_log2_scale(v_f[1]) : 0.f;
      float p[4], mx[2];  // p: scores without the head's factor
#pragma unroll
      for (int e = 0; e < 2; e++) {
        p[e] = (sa[0][e] + sa[1][e]) * k_f[0];
        p[2 + e] = (sa[0][2 + e] + sa[1][2 + e]) * k_f[1];
      }
      if (pos0 < first || pos0 + Cfg::kTok > keys) {  // (uniform)
        const int p0 = pos0 + g, p1 = p0 + 8;
        if (p0 < first || p0 >= keys) p[0] = p[1] = -INFINITY;
        if (p1 < first || p1 >= keys) p[2] = p[3] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) mx[e] = fmaxf(fmaf(p[e], qf[e], up0), fmaf(p[2 + e], qf[e], up1));
      constexpr float kDown = I8 ? kPieceDown : 0.f, kRaise = kPieceLazy + kDown;
      if (__any_sync(0xffffffffu, mx[0] > m_run[0] + kRaise || mx[1] > m_run[1] + kRaise)) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float x = mx[e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float m_new = fmaxf(m_run[e], x - kDown);
          f[e] = piece_ex2(m_run[e] - m_new);
          l_run[e] *= f[e];
          m_run[e] = m_new;
        }
#pragma unroll
        for (int m = 0; m < KS; m++) { oacc[m][0] *= f[0]; oacc[m][1] *= f[1]; oacc[m][2] *= f[0]; oacc[m][3] *= f[1]; }
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        p[e] = piece_ex2(fmaf(p[e], qf[e], -m_run[e]));
        p[2 + e] = piece_ex2(fmaf(p[2 + e], qf[e], -m_run[e]));
        l_run[e] += p[e] + p[2 + e];
      }
      uint32_t pb0, pb1, pl0 = 0u, pl1 = 0u;
      if constexpr (I8) {
        const __half2 h0 = __floats2half2_rn(p[0] * v_f[0], p[1] * v_f[0]), h1 = __floats2half2_rn(p[2] * v_f[1], p[3] * v_f[1]);
        pb0 = st_transpose(*reinterpret_cast<const uint32_t *>(&h0));
        pb1 = st_transpose(*reinterpret_cast<const uint32_t *>(&h1));
      } else {
        const uint32_t p01 = float2_to_bf16x2(p[0], p[1]), p23 = float2_to_bf16x2(p[2], p[3]);
        const float2 r01 = bf16x2_to_float2(p01), r23 = bf16x2_to_float2(p23);
        const uint32_t q01 = float2_to_bf16x2(p[0] - r01.x, p[1] - r01.y), q23 = float2_to_bf16x2(p[2] - r23.x, p[3] - r23.y);
        const bool rest = kTwice && tq * 2 >= G;
        pb0 = st_transpose(G == 1 ? (p01 & 0xffffu) | (q01 & 0xffff0000u) : rest ? q01 : p01);
        pb1 = st_transpose(G == 1 ? (p23 & 0xffffu) | (q23 & 0xffff0000u) : rest ? q23 : p23);
        if (!kTwice) { pl0 = st_transpose(q01); pl1 = st_transpose(q23); }
      }
      // ---- O^T += V^T P^T: tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9, dims g kPer ..
      const uint32_t va = at + Cfg::kPart;
      const int t0 = 2 * tq;
      if constexpr (I8) {
        uint32_t v[4][kPer / 4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int r = t0 + (k & 1) + (k >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 w = st_lds_16(va + st_v_chunk<D, I8>(r, g) * 16);
            v[k][0] = w.x; v[k][1] = w.y; v[k][2] = w.z; v[k][3] = w.w;
          } else {
            const uint2 w = st_lds_8(va + st_v_chunk<D, I8>(r, g >> 1) * 16 + (g & 1) * 8);
            v[k][0] = w.x; v[k][1] = w.y;
          }
#pragma unroll
          for (int j = 0; j < kPer / 4; j++) v[k][j] ^= 0x80808080u;
        }
#pragma unroll
        for (int j = 0; j < kPer / 4; j++) {
#pragma unroll
          for (int hf = 0; hf < 2; hf++) {
            uint32_t a0, a1, a2, a3;
            bytes_to_half2(__byte_perm(v[0][j], v[1][j], hf ? 0x7362 : 0x5140), a0, a1);
            bytes_to_half2(__byte_perm(v[2][j], v[3][j], hf ? 0x7362 : 0x5140), a2, a3);
            st_mma<I8>(oacc[2 * j + hf], a0, a1, a2, a3, pb0, pb1);
          }
        }
      } else {
#pragma unroll
        for (int cc = 0; cc < kPer / 8; cc++) {
          uint4 w[4];
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = st_lds_16(va + st_v_chunk<D, I8>(t0 + (k & 1) + (k >> 1) * 8, g * (kPer / 8) + cc) * 16);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            auto el = [&](int k) { return j == 0 ? w[k].x : j == 1 ? w[k].y : j == 2 ? w[k].z : w[k].w; };
            const uint32_t a0 = __byte_perm(el(0), el(1), 0x5410), a1 = __byte_perm(el(0), el(1), 0x7632);
            const uint32_t a2 = __byte_perm(el(2), el(3), 0x5410), a3 = __byte_perm(el(2), el(3), 0x7632);
            st_mma<I8>(oacc[4 * cc + j], a0, a1, a2, a3, pb0, pb1);
            if (!kTwice) st_mma<I8>(oacc[4 * cc + j], a0, a1, a2, a3, pl0, pl1);
          }
        }
      }
    }

    // ================= the warps' states meet in shared memory, kMeet heads at a time
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 4);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 8);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 16);
    }
    if constexpr (kTwice) {  // the weights' halves: columns h and h + G
#pragma unroll
      for (int m = 0; m < KS; m++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          if (G == 1) { if (!(k & 1)) oacc[m][k] += oacc[m][k + 1]; }
          else oacc[m][k] += __shfl_xor_sync(0xffffffffu, oacc[m][k], G / 2);
        }
    }
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < 2; e++) { s_m[warp][2 * tq + e] = m_run[e]; s_l[warp][2 * tq + e] = l_run[e]; }
    }
    const size_t row = (size_t)cur.t * n_heads + cur.h * G;             // of the pair's first head in the result
    const int c_first = cur.u0 / share, c_last = (cur.u1 - 1) / share;  // the CTAs that have a piece of this history
    const int side = cur.u0 >= lo ? 1 : 0;  // (of the histories that others have pieces of too, one was begun before, one goes on)
    const size_t slot = 2 * (size_t)blockIdx.x + side;
#pragma unroll
    for (int h0 = 0; h0 < G; h0 += kMeet) {
      if (h0) __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = 2 * tq + e - h0;
        if (col >= 0 && col < kMeet) {
          float2 *o = reinterpret_cast<float2 *>(s_o + (warp * kMeet + col) * Cfg::kHead + g * (kPer + 2));
#pragma unroll
          for (int m = 0; m < KS; m++) o[m] = make_float2(oacc[m][e], oacc[m][2 + e]);
        }
      }
      __syncthreads();
      const int hh = threadIdx.x / (D / 4), h = h0 + hh, i = threadIdx.x % (D / 4) * 4;  // four dims of a head
      if (hh < kMeet) {
        const int off = i / kPer * (kPer + 2) + i % kPer;
        float M = kPieceNone, l = 0.f;
#pragma unroll
        for (int w = 0; w < kStWarps; w++) M = fmaxf(M, s_m[w][h]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kStWarps; w++) {
          const float f = piece_ex2(s_m[w][h] - M);
          const float2 *x = reinterpret_cast<const float2 *>(s_o + (w * kMeet + hh) * Cfg::kHead + off), y = x[0], z = x[1];
          o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y); o.z = fmaf(z.x, f, o.z); o.w = fmaf(z.y, f, o.w);
          l = fmaf(s_l[w][h], f, l);
        }
        if (c_first == c_last) {
          put(row + h, i, o, M, l);
        } else {
          __stcg(reinterpret_cast<float4 *>(a.piece_o + (slot * G + h) * D + i), o);
          if (i == 0) __stcg(reinterpret_cast<float2 *>(a.piece_ml + slot * st_ml(G) + 2 * h), make_float2(M, l));
        }
      }
    }
    if (c_first != c_last) {
      if (side) { part_row[1] = row; part_first[1] = c_first; part_last[1] = c_last; }
      else { part_row[0] = row; part_first[0] = c_first; part_last[0] = c_last; }
    }
    if (cur.u1 >= hi) break;
    next_pair(cur);
    __syncthreads();  // the next piece's states may come
  }
  st_copy_wait<0>();
  st_copy_wait<0>();

  // (Not at the start: CTAs of the next kernel that wait on the SMs cost calls in a row 0.4 us, 64 of heads of 64 17.2 -> 16.8, 32 to 6000 30.6 -> 30.2)
  if (!a.inputs_first) pdl_launch_dependents();
  // ================= histories in several CTAs: the one that ends last joins the pieces, in the order of the history.  More than eight are joined in
  // about as many groups as a group has pieces, and then the groups: what one CTA reads at the end stays short however long the history is.  The
  // barriers and one thread's atomic, a release and an acquire, order all threads' writes and reads (with fences on both sides of a relaxed one
  // 0.4 us more a level); both histories' first counts share them
  if (part_first[0] != part_last[0] || part_first[1] != part_last[1]) {
    auto fan_of = [&](int parts) { return parts <= 8 ? parts : (int)ceilf(sqrtf((float)parts)); };
    auto arrive = [&](int level, size_t slot, int n) {
      int *count = a.counters + level * stream_slots() + slot;
      int before;
      asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
      const bool last = before == n - 1;
      if (last) *count = 0;  // as the next call wants it
      return last;
    };
    __syncthreads();
    if (threadIdx.x < 2) {
      const int c_first = threadIdx.x ? part_first[1] : part_first[0], c_last = threadIdx.x ? part_last[1] : part_last[0];
      bool last = false;
      if (c_first != c_last) {
        const int fan = fan_of(c_last - c_first + 1), lead = c_first + ((int)blockIdx.x - c_first) / fan * fan;  // the group's first CTA
        last = arrive(0, 2 * (size_t)lead + (lead == c_first ? 1 : 0), min(fan, c_last + 1 - lead));
      }
      s_last[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int side = 0; side < 2; side++) {
      if (!s_last[side]) continue;
      const size_t row = side ? part_row[1] : part_row[0];
      const int c_first = side ? part_first[1] : part_first[0], c_last = side ? part_last[1] : part_last[0];
      const int parts = c_last - c_first + 1, fan = fan_of(parts), groups = (parts + fan - 1) / fan;
      const int lead = c_first + ((int)blockIdx.x - c_first) / fan * fan;
      auto slot_of = [&](int c) { return 2 * (size_t)c + (c == c_first ? 1 : 0); };
      int n = min(fan, c_last + 1 - lead);
#pragma unroll 1
      for (int level = 0;; level++) {
        if (level) {
          __syncthreads();
          if (threadIdx.x == 0) s_last[side] = arrive(1, slot_of(c_first), n);
          __syncthreads();
          if (!s_last[side]) break;
        }
        const bool whole = level || groups == 1;
        const float *src_o = level ? a.group_o : a.piece_o, *src_ml = level ? a.group_ml : a.piece_ml;
        // four dims of a head to a thread (groups of eight: of two heads), kAhead pieces' on their way.  (Both heads at once: two histories of 60000 in 28
        // pieces 40.1 -> 37.7 us; eight pieces at once are no faster and cost a short call 0.5 us: code is fetched anew at every launch)
        constexpr int kQuads = G * D / 4, kAhead = 4;
        constexpr int kMine = (kQuads + kStWarps * 32 - 1) / (kStWarps * 32);
        if (threadIdx.x < kQuads) {
          float M[kMine], l[kMine];
          float4 o[kMine];
#pragma unroll
          for (int q = 0; q < kMine; q++) { M[q] = kPieceNone; l[q] = 0.f; o[q] = make_float4(0.f, 0.f, 0.f, 0.f); }
#pragma unroll 1
          for (int k = 0; k < n; k += kAhead) {
            float2 ml[kAhead][kMine];
            float4 x[kAhead][kMine];
#pragma unroll
            for (int j = 0; j < kAhead; j++)
              if (k + j < n) {
                const size_t sl = slot_of(level ? c_first + (k + j) * fan : lead + k + j);
#pragma unroll
                for (int q = 0; q < kMine; q++) {
                  const int quad = threadIdx.x + q * kStWarps * 32;
                  ml[j][q] = __ldcg(reinterpret_cast<const float2 *>(src_ml + sl * st_ml(G)) + quad / (D / 4));
                  x[j][q] = __ldcg(reinterpret_cast<const float4 *>(src_o) + sl * kQuads + quad);
                }
              }
#pragma unroll
            for (int j = 0; j < kAhead; j++)
              if (k + j < n) {
#pragma unroll
                for (int q = 0; q < kMine; q++) {
                  const float m_new = fmaxf(M[q], ml[j][q].x), f = piece_ex2(M[q] - m_new), fn = piece_ex2(ml[j][q].x - m_new);
                  M[q] = m_new;
                  l[q] = l[q] * f + ml[j][q].y * fn;
                  o[q].x = o[q].x * f + x[j][q].x * fn;
                  o[q].y = o[q].y * f + x[j][q].y * fn;
                  o[q].z = o[q].z * f + x[j][q].z * fn;
                  o[q].w = o[q].w * f + x[j][q].w * fn;
                }
              }
          }
#pragma unroll
          for (int q = 0; q < kMine; q++) {
            const int quad = threadIdx.x + q * kStWarps * 32, h = quad / (D / 4), i = quad % (D / 4) * 4;
            if (whole) {
              put(row + h, i, o[q], M[q], l[q]);
            } else {
              __stcg(reinterpret_cast<float4 *>(a.group_o) + slot_of(lead) * kQuads + quad, o[q]);
              if (i == 0) __stcg(reinterpret_cast<float2 *>(a.group_ml + slot_of(lead) * st_ml(G)) + h, make_float2(M[q], l[q]));
            }
          }
        }
        if (whole) break;
        n = groups;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------- host
size_t attn_stream_scratch_elems(int n_heads, int n_kv, int d) {  // counters, then the pieces of every resident CTA
  if (n_kv <= 0 || n_heads <= 0 || d <= 0) return 0;
  return kStCounters + 2 * stream_slots() * ((size_t)(n_heads / n_kv) * d + st_ml(n_heads / n_kv));
}

template <int D, int G, bool I8, bool kAt>
static cudaError_t stream_launch(const StArgs &a, cudaStream_t st) {
  using Cfg = StCfg<D, I8>;
  auto kern = attn_stream_kernel<D, G, I8, kAt>;
  constexpr int kFixed = Cfg::fixed(G);
  static DeviceOnce once;
  DIS_CUDA_TRY(once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + (3 * kStMaxT + 1) * 4); }));
  // A share for each CTA that is resident, so that all of them run at once: the tokens' lengths take shared memory too, and from 126 tokens on bf16 heads of 128
  // have room for two CTAs of an SM, not three.  (Shares for three: 126 tokens to 600 40.7 us, for two 31.9; 200 to 2100 127.8, 108.6; 500 to 900 160, 137)
  const int smem = kFixed + (3 * a.T + 1) * 4, ctas = std::min(Cfg::kCtas, kSmSmem / ((smem + kStStatic + 127) / 128 * 128 + 1024));
  return launch_k(kern, dim3(kNumSMs * ctas), dim3(kStWarps * 32), (size_t)smem, st, a);
}

template <bool I8>
static cudaError_t stream_dispatch(const StArgs &a, int G, int d, cudaStream_t st) {
#define DIS_ST_CASE(DD, GG) \
  if (d == DD && G == GG) return a.first_at ? stream_launch<DD, GG, I8, true>(a, st) : stream_launch<DD, GG, I8, false>(a, st);
  DIS_ST_CASE(128, 8) DIS_ST_CASE(128, 4) DIS_ST_CASE(128, 2) DIS_ST_CASE(128, 1)
  DIS_ST_CASE(64, 8) DIS_ST_CASE(64, 4) DIS_ST_CASE(64, 2) DIS_ST_CASE(64, 1)
#undef DIS_ST_CASE
  set_last_error("attention over pieces: head_dim must be 64 or 128 and the GQA group 1, 2, 4 or 8");
  return cudaErrorInvalidValue;
}

cudaError_t launch_attn_stream(const uint16_t *q, const void *pool, const float *scale, const int *page_table, int max_pages, const int *pt_row,
                               const int *ctx, int first, const int *first_at, uint16_t *out, float *state_o, float *state_ml, float *scratch,
                               bool inputs_first, int T, int n_heads, int n_kv, int d, int page_size, cudaStream_t st) {
  // a launch's tiles are counted in 32 bits
  const long long most = ((long long)max_pages * page_size / 16 + 2) * n_kv;
  const int G = n_heads / n_kv, step = (int)std::max(1ll, std::min({(long long)kStMaxT, 0x7fffffffll / most}));
  StArgs a{};
  a.pool = pool; a.scale = scale; a.page_table = page_table; a.max_pages = max_pages; a.first = first; a.first_at = first_at;
  a.counters = reinterpret_cast<int *>(scratch);
  a.piece_o = scratch + kStCounters;
  a.group_o = a.piece_o + stream_slots() * (size_t)G * d;
  a.piece_ml = a.group_o + stream_slots() * (size_t)G * d;
  a.group_ml = a.piece_ml + stream_slots() * (size_t)st_ml(G);
  a.n_kv = n_kv;
  while ((1 << a.page_shift) < page_size) a.page_shift++;
  for (int t = 0; t < T; t += step) {
    a.T = std::min(step, T - t);
    a.inputs_first = inputs_first;
    a.q = q + (size_t)t * n_heads * d;
    a.pt_row = pt_row + t;
    a.ctx = ctx + t;
    a.out = out ? out + (size_t)t * n_heads * d : nullptr;
    a.state_o = state_o ? state_o + (size_t)t * n_heads * d : nullptr;
    a.state_ml = state_ml ? state_ml + (size_t)t * n_heads * 2 : nullptr;
    DIS_CUDA_TRY(scale ? stream_dispatch<true>(a, G, d, st) : stream_dispatch<false>(a, G, d, st));
  }
  return cudaSuccess;
}

}  // namespace dis
