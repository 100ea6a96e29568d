// Attention of the new tokens of every sequence over its pages.  Row i of the n_b new rows of sequence b stands at place p = len_b - n_b + i of the
// sequence and sees the keys j <= p, with a window w those with j > p - w too: o = sum_j softmax_j(scale q k_j) v_j, zeros where it sees none.
#include "paged_attn_tc.cuh"

#include <climits>

namespace zl {

// sequence that has row t of q, from starts[0 .. seqs]; -1: none
__device__ __forceinline__ int paged_seq_of(const int32_t* starts, int seqs, int t) {
    if (t < starts[0] || t >= starts[seqs]) return -1;
    int lo = 0, hi = seqs;   // starts[lo] <= t < starts[hi]
    while (lo + 1 < hi) {
        const int m = (lo + hi) >> 1;
        if (starts[m] <= t) lo = m;
        else hi = m;
    }
    return lo;
}

// grid (rows, heads): a row and a head by 128 threads, a warp for every fourth key; of sequences of up to p.few rows
template <typename T, int D>
__global__ void __launch_bounds__(128) k_paged_attn_rows(const PagedAttn p, const PagedCache c) {
    constexpr int E = D / 32;
    __shared__ float s_m[4], s_l[4], s_o[4][D];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = paged_seq_of(p.starts, c.seqs, t);
    if (b < 0 || (p.starts[b + 1] - p.starts[b]) * p.group > p.few) return;
    const int len = min(max(p.lens[b], 0), c.room());
    const int at = p.lens[b] - p.starts[b + 1] + t;
    const int last = min(at, len - 1), first = p.window ? max(0, at - p.window + 1) : 0;
    const long long head = (long long)(h / p.group) * c.head_stride;
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

constexpr int kFewRows = 16;   // (token, head) rows of a kv head that a sequence brings to the kernel for few rows

struct PagedPlan {
    bool tiles, few;        // which kernels run
    int blocks, splits;     // of the tiles
    size_t ml_bytes, bytes;
};

static PagedPlan paged_plan(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    PagedPlan s = {};
    const int group = heads / kv_heads;
    s.tiles = (long long)max_new * group > kFewRows;
    s.few = !s.tiles || seqs > 1;
    if (!s.tiles) return s;
    // every sequence adds less than one block to those of the rows, and only those of more than kFewRows rows have any
    const long long all = (long long)rows * group, more = seqs > 1 ? all / (kFewRows + 1) : 1;
    s.blocks = (int)(all / kPtRows + (more < seqs ? more : seqs));
    const int tiles = cdiv(max_keys, kPtKeys), sms = device_sm_count();
    s.splits = 1;
    while (s.splits < 16 && 2ll * s.splits * s.blocks * kv_heads <= sms && tiles >= 8 * s.splits) s.splits *= 2;
    if (s.splits > 1) {
        const size_t parts = (size_t)s.blocks * s.splits * kv_heads * kPtRows;
        s.ml_bytes = parts * sizeof(float2);
        s.bytes = s.ml_bytes + parts * dim * sizeof(float);
    }
    return s;
}

template <typename T, int D>
static int paged_attention(PagedAttn p, const PagedCache& c, const PagedPlan& s, int kv_heads, int pdl, zl_stream_t stream) {
    unsigned* words = nullptr;
    if (s.tiles) {
        ZL_CHECK_WAITS();
        words = wait_words();
        ZL_CHECK_CUDA(words ? cudaSuccess : cudaErrorMemoryAllocation);
        static bool attr_set[64] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !attr_set[dev]) {
            ZL_CHECK_CUDA(cudaFuncSetAttribute(k_paged_attn_tiles<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PtCfg<D>::kBytes));
            if (dev >= 0 && dev < 64) attr_set[dev] = true;
        }
    }
    p.few = !s.tiles ? INT_MAX : s.few ? kFewRows : 0;
    if (s.few) ZL_CHECK_CUDA(launch(k_paged_attn_rows<T, D>, dim3(p.rows, p.heads), dim3(128), 0, stream, pdl != 0, p, c));
    if (s.tiles) {
        ZL_CHECK_CUDA(launch(k_paged_attn_tiles<T, D>, dim3(s.blocks * s.splits, kv_heads), dim3(kPtThreads), PtCfg<D>::kBytes, stream, pdl != 0, p, c, words + kWaitAttnPaged));
        if (s.splits > 1) ZL_CHECK_CUDA(launch(k_paged_attn_join<T, D>, dim3(s.blocks, kv_heads), dim3(256), 0, stream, true, p, c));
    }
    return ZL_OK;
}

}  // namespace zl

using namespace zl;

extern "C" size_t zl_paged_attention_workspace_bytes(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    if (rows <= 0 || max_new <= 0 || seqs <= 0 || max_keys <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0) return 0;
    return paged_plan(rows, max_new, seqs, max_keys, heads, kv_heads, dim).bytes;
}

extern "C" int zl_paged_attention(const void* q, const void* k_cache, const void* v_cache, long long num_pages, int page_size, long long page_stride,
                                  long long row_stride, long long head_stride, const int32_t* page_table, int ld_table, int max_pages,
                                  const int32_t* seq_lens, const int32_t* q_starts, int seqs, float scale, int window, void* out, int rows, int max_new,
                                  int heads, int kv_heads, int dim, void* workspace, size_t workspace_bytes, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(q && seq_lens && q_starts && out && rows > 0 && max_new > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0);
    ZL_CHECK_ARG(scale > 0.f && scale < INFINITY && window >= 0);
    ZL_CHECK_PAGED(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, seqs);
    ZL_CHECK_SUPPORTED((dim == 64 || dim == 128) && (dtype == ZL_F16 || dtype == ZL_BF16));
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0);
    ZL_CHECK_SUPPORTED(heads <= 65535 && (long long)rows * heads < INT_MAX);
    const long long room = (long long)max_pages * page_size;
    const PagedPlan s = paged_plan(rows, max_new, seqs, (int)(room < INT_MAX - 255 ? room : INT_MAX - 255), heads, kv_heads, dim);
    ZL_CHECK_ARG(s.bytes == 0 || (workspace && workspace_bytes >= s.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0));
    const PagedCache c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages,
                          page_size, seqs, paged_divisor(page_size)};
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, heads / kv_heads, window, scale * 1.4426950408889634f, 0, s.splits ? s.splits : 1,
                         static_cast<float2*>(workspace), s.bytes ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + s.ml_bytes) : nullptr};
    if (dtype == ZL_F16) return dim == 64 ? paged_attention<__half, 64>(p, c, s, kv_heads, pdl, stream) : paged_attention<__half, 128>(p, c, s, kv_heads, pdl, stream);
    return dim == 64 ? paged_attention<__nv_bfloat16, 64>(p, c, s, kv_heads, pdl, stream) : paged_attention<__nv_bfloat16, 128>(p, c, s, kv_heads, pdl, stream);
}
