// Attention of the new tokens of every sequence over its pages.  Row i of the n_b new rows of sequence b stands at place p = len_b - n_b + i of the
// sequence and sees the keys j <= p, with a window w those with j > p - w too: o = sum_j softmax_j(scale q k_j) v_j, zeros where it sees none.
#include "paged.cuh"

namespace zl {

struct PagedAttn {
    const void* q;
    void* out;
    const int32_t *lens, *starts;
    int rows, heads, kv_heads, window;
    float scale;   // times log2(e)
};

// first sequence whose rows end behind t, from starts[0 .. seqs]; -1: row of no sequence
__device__ __forceinline__ int paged_seq_of(const int32_t* starts, int seqs, int t) {
    if (t < starts[0] || t >= starts[seqs]) return -1;
    int lo = 0, hi = seqs;
    while (lo + 1 < hi) {
        const int m = (lo + hi) >> 1;
        if (starts[m] <= t) lo = m;
        else hi = m;
    }
    while (lo + 1 < seqs && starts[lo + 1] <= t) ++lo;
    return lo;
}

// grid (rows, heads): a row and a head by 128 threads, a warp for every fourth key
template <typename T, int D>
__global__ void __launch_bounds__(128) k_paged_attn_rows(const PagedAttn p, const PagedCache c) {
    constexpr int E = D / 32;
    __shared__ float s_m[4], s_l[4], s_o[4][D];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = paged_seq_of(p.starts, c.seqs, t);
    if (b < 0) return;
    const int len = min(max(p.lens[b], 0), c.room());
    const int at = p.lens[b] - p.starts[b + 1] + t;
    const int last = min(at, len - 1), first = p.window ? max(0, at - p.window + 1) : 0;
    const long long head = (long long)(h / (p.heads / p.kv_heads)) * c.head_stride;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = to_f32<T>(static_cast<const T*>(p.q)[((size_t)t * p.heads + h) * D + e * 32 + lane]);
    for (int j = first + warp; j <= last; j += 4) {
        const long long r = c.row_at(b, j);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (r >= 0) s = fmaf(q[e], to_f32<T>(static_cast<const T*>(c.k)[r + head + e * 32 + lane]), s);
        s = warp_sum(s) * p.scale;
        const float up = fmaxf(m, s), f = up == -INFINITY ? 1.f : exp2f(m - up), w = up == -INFINITY ? 0.f : exp2f(s - up);
        m = up;
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + (r >= 0 ? w * to_f32<T>(static_cast<const T*>(c.v)[r + head + e * 32 + lane]) : 0.f);
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][e * 32 + lane] = o[e];
    __syncthreads();
    m = -INFINITY;
    for (int w = 0; w < 4; ++w) m = fmaxf(m, s_m[w]);
    for (int d = threadIdx.x; d < D; d += 128) {
        float sum = 0.f, v = 0.f;
        for (int w = 0; w < 4; ++w) {
            const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - m);
            sum = fmaf(s_l[w], f, sum);
            v = fmaf(s_o[w][d], f, v);
        }
        static_cast<T*>(p.out)[((size_t)t * p.heads + h) * D + d] = from_f32<T>(sum != 0.f ? v / sum : 0.f);
    }
}

}  // namespace zl

using namespace zl;

extern "C" size_t zl_paged_attention_workspace_bytes(int rows, int max_new, int seqs, int heads, int kv_heads, int dim) {
    (void)rows, (void)max_new, (void)seqs, (void)heads, (void)kv_heads, (void)dim;
    return 0;
}

extern "C" int zl_paged_attention(const void* q, const void* k_cache, const void* v_cache, long long num_pages, int page_size, long long page_stride,
                                  long long row_stride, long long head_stride, const int32_t* page_table, int ld_table, int max_pages,
                                  const int32_t* seq_lens, const int32_t* q_starts, int seqs, float scale, int window, void* out, int rows, int max_new,
                                  int heads, int kv_heads, int dim, void* workspace, size_t workspace_bytes, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(q && seq_lens && q_starts && out && rows > 0 && max_new > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0);
    ZL_CHECK_ARG(scale > 0.f && scale < INFINITY && window >= 0);
    ZL_CHECK_PAGED(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, seqs);
    ZL_CHECK_SUPPORTED((dim == 64 || dim == 128) && (dtype == ZL_F16 || dtype == ZL_BF16));
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 && heads <= 65535);
    const size_t need = zl_paged_attention_workspace_bytes(rows, max_new, seqs, heads, kv_heads, dim);
    ZL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need));
    const PagedCache c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages,
                          page_size, seqs, paged_divisor(page_size)};
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, kv_heads, window, scale * 1.4426950408889634f};
    auto kernel = dtype == ZL_F16 ? (dim == 64 ? k_paged_attn_rows<__half, 64> : k_paged_attn_rows<__half, 128>)
                                  : (dim == 64 ? k_paged_attn_rows<__nv_bfloat16, 64> : k_paged_attn_rows<__nv_bfloat16, 128>);
    ZL_CHECK_CUDA(launch(kernel, dim3(rows, heads), dim3(128), 0, stream, pdl != 0, p, c));
    return ZL_OK;
}
