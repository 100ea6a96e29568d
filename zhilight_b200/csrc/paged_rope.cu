// Rotation of fused query / key / value rows by positions on several axes, and their append to a paged cache of 16 bits (paged_rope.cuh).
#include "paged_rope.cuh"

using namespace zl;

extern "C" int zl_qkv_axes_rope_append(const void* qkv, long long ldq, const int32_t* pos, long long ld_pos, int axes, const double* inv_freq,
                                       const int32_t* axis, int half, int layout, float mscale, const int32_t* token_seq, const int32_t* placement,
                                       const int32_t* page_table, int ld_table, int max_pages, int seqs, void* k_cache, void* v_cache,
                                       long long num_pages, int page_size, long long page_stride, long long row_stride, long long head_stride,
                                       void* q_out, int T, int heads, int kv_heads, int dim, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(qkv && pos && token_seq && placement && q_out && T > 0 && heads > 0 && kv_heads > 0);
    ZL_CHECK_ARG(half >= 0 && 2 * half <= dim && axes > 0 && ld_pos >= T && (half == 0 || (inv_freq && axis)));
    ZL_CHECK_ARG(layout == ZL_ROT_HALVES || layout == ZL_ROT_ADJACENT);
    ZL_CHECK_PAGED(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, seqs);
    ZL_CHECK_SUPPORTED(dim > 0 && dim % 8 == 0 && dim <= 1024 && dtype != ZL_F32);
    ZL_CHECK_ARG(ldq >= (long long)(heads + 2 * kv_heads) * dim);
    ZL_CHECK_SUPPORTED(ldq % 8 == 0 && ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) == 0);
    ZL_CHECK_SUPPORTED((heads + 2ll * kv_heads) * dim <= kRopeSmem / 2);   // a row in shared memory
    const PagedCache c = {k_cache, v_cache, num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, page_size, seqs, paged_divisor(page_size)};
    return axes_rope_append<false>(qkv, ldq, pos, ld_pos, axes, inv_freq, axis, half, layout, mscale, token_seq, placement, c, q_out, T, heads, kv_heads, dim, dtype,
                                   pdl != 0, stream);
}
