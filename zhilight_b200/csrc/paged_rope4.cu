// The append of paged_rope.cuh to a paged cache of 4 bits, and what such a cache stands for (int4_cache.cuh).
#include "paged_rope.cuh"

namespace zl {

struct Int4Values {
    const void *k, *v;
    void *k_out, *v_out;
    const int32_t* pages;   // nullptr: page i is number i
    long long num_pages, page_stride, row_stride, head_stride;   // bytes
    int page_size, kv_heads, rows;   // rows: of heads, page_size * kv_heads a page
    PagedDivisor by_heads, by_page;
};

constexpr int kValuesThreads = 256, kValuesAhead = 4;

// grid (ctas, caches): a thread for 16 columns of kValuesAhead rows: where a row lies is most of the work.  Two lanes have a group of 32 columns; they change the codes of 8 of them, so that
// each store of theirs is 32 bytes behind one another.  36000 rows of 8 heads of 64, 97 MB of which four fifths are written: 8 columns a thread 18 us, 16 without the change 26, so 17.
template <typename T, int D>
__global__ void __launch_bounds__(kValuesThreads) k_int4_values(const Int4Values p) {
    constexpr int kPieces = D / 16, kRows = kValuesThreads / kPieces;
    pdl_trigger();
    pdl_wait();
    const uint8_t* from = static_cast<const uint8_t*>(blockIdx.y ? p.v : p.k);
    uint4* out = static_cast<uint4*>(blockIdx.y ? p.v_out : p.k_out);
    const int piece = threadIdx.x % kPieces, row0 = (int)blockIdx.x * (kRows * kValuesAhead) + threadIdx.x / kPieces;
    uint2 codes[kValuesAhead];
    uint32_t meta[kValuesAhead];
#pragma unroll
    for (int u = 0; u < kValuesAhead; ++u) {
        const int i = row0 + u * kRows;
        codes[u] = make_uint2(0u, 0u), meta[u] = 0;
        if (i >= p.rows) continue;
        const int row = p.by_heads(i), head = i - row * p.kv_heads, page = p.by_page(row), id = p.pages ? p.pages[page] : page;
        if (id < 0 || id >= p.num_pages) continue;
        const uint8_t* at = from + (long long)id * p.page_stride + (long long)(row - page * p.page_size) * p.row_stride + (long long)head * p.head_stride;
        codes[u] = *reinterpret_cast<const uint2*>(at + piece * 8);
        meta[u] = *reinterpret_cast<const uint32_t*>(at + D / 2 + piece / 2 * 4);
    }
#pragma unroll
    for (int u = 0; u < kValuesAhead; ++u) {
        const int i = row0 + u * kRows;
        const bool odd = piece & 1;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? codes[u].x : codes[u].y, 1);
        if (i >= p.rows) continue;
        uint32_t step, low;
        int4_meta<T>(meta[u], step, low);
        uint4* to = out + ((size_t)i * kPieces + piece) * 2 - odd;
        to[0] = int4_eight<T>(odd ? other : codes[u].x, step, low);
        to[2] = int4_eight<T>(odd ? codes[u].y : other, step, low);
    }
}

template <typename T, int D>
static int int4_values(const Int4Values& p, int caches, bool pdl, zl_stream_t stream) {
    const int each = kValuesThreads / (D / 16) * kValuesAhead;
    ZL_CHECK_CUDA(launch(k_int4_values<T, D>, dim3((p.rows - 1) / each + 1, caches), dim3(kValuesThreads), 0, stream, pdl, p));
    return ZL_OK;
}

}  // namespace zl

using namespace zl;

extern "C" int zl_qkv_axes_rope_append_int4(const void* qkv, long long ldq, const int32_t* pos, long long ld_pos, int axes, const double* inv_freq,
                                            const int32_t* axis, int half, int layout, float mscale, const int32_t* token_seq, const int32_t* placement,
                                            const int32_t* page_table, int ld_table, int max_pages, int seqs, void* k_cache, void* v_cache,
                                            long long num_pages, int page_size, long long page_stride, long long row_stride, long long head_stride,
                                            void* q_out, int T, int heads, int kv_heads, int dim, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(qkv && pos && token_seq && placement && q_out && T > 0 && heads > 0 && kv_heads > 0);
    ZL_CHECK_ARG(half >= 0 && 2 * half <= dim && axes > 0 && ld_pos >= T && (half == 0 || (inv_freq && axis)));
    ZL_CHECK_ARG(layout == ZL_ROT_HALVES || layout == ZL_ROT_ADJACENT);
    ZL_CHECK_PAGED_INT4(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, dim);
    ZL_CHECK_ARG(page_table && max_pages > 0 && ld_table >= max_pages && seqs > 0);
    ZL_CHECK_SUPPORTED(dtype == ZL_F16 || dtype == ZL_BF16);
    ZL_CHECK_ARG(ldq >= (long long)(heads + 2 * kv_heads) * dim);
    ZL_CHECK_SUPPORTED(ldq % 8 == 0 && ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) == 0);
    ZL_CHECK_SUPPORTED((heads + 2ll * kv_heads) * dim <= kRopeSmem / 4);   // two rows in shared memory; what stands beside them there is seen to in axes_rope_append
    const PagedCache c = {k_cache, v_cache, num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, page_size, seqs, paged_divisor(page_size)};
    return axes_rope_append<true>(qkv, ldq, pos, ld_pos, axes, inv_freq, axis, half, layout, mscale, token_seq, placement, c, q_out, T, heads, kv_heads, dim, dtype,
                                  pdl != 0, stream);
}

extern "C" int zl_int4_cache_values(const void* k_cache, const void* v_cache, long long num_pages, int page_size, long long page_stride, long long row_stride,
                                    long long head_stride, const int32_t* pages, long long n, void* k_out, void* v_out, int kv_heads, int dim, int dtype, int pdl,
                                    zl_stream_t stream) {
    ZL_CHECK_ARG(k_out && (v_cache ? v_out != nullptr : true) && kv_heads > 0 && n > 0 && (pages || n <= num_pages));
    ZL_CHECK_PAGED_INT4(k_cache, v_cache ? v_cache : k_cache, num_pages, page_size, page_stride, row_stride, head_stride, dim);
    ZL_CHECK_SUPPORTED(dtype == ZL_F16 || dtype == ZL_BF16);
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0);
    ZL_CHECK_SUPPORTED(n <= 0x7fff0000ll / page_size / kv_heads);   // rows are counted in 32 bits, with room for a CTA's more
    const Int4Values p = {k_cache, v_cache, k_out, v_out, pages, num_pages, page_stride, row_stride, head_stride, page_size, kv_heads, (int)(n * page_size * kv_heads),
                          paged_divisor(kv_heads), paged_divisor(page_size)};
    const int caches = v_cache ? 2 : 1;
    if (dtype == ZL_F16) return dim == 64 ? int4_values<__half, 64>(p, caches, pdl != 0, stream) : int4_values<__half, 128>(p, caches, pdl != 0, stream);
    return dim == 64 ? int4_values<__nv_bfloat16, 64>(p, caches, pdl != 0, stream) : int4_values<__nv_bfloat16, 128>(p, caches, pdl != 0, stream);
}
