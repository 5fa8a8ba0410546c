// k_attn_shared.cu -- decode attention of a batch whose requests share the first `prefix` positions of their histories.
#include "attn_piece.cuh"

namespace dis {

size_t attn_shared_scratch_elems(int T, int n_heads, int n_kv, int d) { return attn_stream_scratch_elems(n_heads, n_kv, d); }

cudaError_t launch_attn_shared(const uint16_t *q, const void *pool, const float *scale, long long n_pages, const int *page_table, int max_pages,
                               const int *pt_row, const int *ctx, int prefix, uint16_t *out, float *scratch, int T, int n_heads, int n_kv, int d,
                               int page_size, cudaStream_t st) {
  return launch_attn_stream(q, pool, scale, page_table, max_pages, pt_row, ctx, 0, out, nullptr, nullptr, scratch, false, T, n_heads, n_kv, d, page_size, st);
}

}  // namespace dis
