// Attention of the new tokens of every sequence over its pages.  Row i of the n_b new rows of sequence b stands at place p = len_b - n_b + i of the
// sequence and sees the keys j <= p, with a window w those with j > p - w too: o = sum_j softmax_j(scale q k_j) v_j, zeros where it sees none.
#include "paged_attn_few.cuh"
#include "paged_attn_tc.cuh"

#include <climits>

namespace zl {

constexpr int kFewRows = 32;   // (token, head) rows of a kv head that a sequence brings to the kernel for few rows

struct PagedPlan {
    bool tiles, few;                        // which kernels run
    int blocks, splits;                     // of the tiles
    int ctas, few_rows;                     // of the few rows; rows of their blocks
    size_t ml, part, few_ml, few_part, bytes;   // places in the workspace
};

static PagedPlan paged_plan(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    PagedPlan s = {};
    const int group = heads / kv_heads, sms = device_sm_count();
    const long long all = (long long)rows * group, most = (long long)max_new * group;
    s.tiles = most > kFewRows;
    s.few = !s.tiles || seqs > 1;
    auto take = [&](size_t bytes) {
        const size_t at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    if (s.tiles) {
        // every sequence adds less than one block to those of the rows, and only those of more than kFewRows rows have any
        const long long more = seqs > 1 ? all / (kFewRows + 1) : 1;
        s.blocks = (int)(all / kPtRows + (more < seqs ? more : seqs));
        const int tiles = cdiv(max_keys, kPtKeys);
        s.splits = 1;
        while (s.splits < 16 && 2ll * s.splits * s.blocks * kv_heads <= sms && tiles >= 8 * s.splits) s.splits *= 2;
        if (s.splits > 1) {
            const size_t parts = (size_t)s.blocks * s.splits * kv_heads * kPtRows;
            s.ml = take(parts * sizeof(float2)), s.part = take(parts * dim * sizeof(float));
        }
    }
    if (s.few) {
        s.few_rows = most <= 16 ? 16 : 32;
        // no more CTAs than there can be tiles: every block has the pool's rows of its sequence at the most
        const long long blocks = all / s.few_rows + seqs, tiles = blocks * cdiv(max_keys, kPfKeys) * kv_heads;
        s.ctas = (int)(tiles < kPfPerSm * sms ? tiles : kPfPerSm * sms);
        const size_t parts = (size_t)s.ctas * 2 * s.few_rows;
        s.few_ml = take(parts * sizeof(float2)), s.few_part = take(parts * dim * sizeof(float));
    }
    return s;
}

template <typename T, int D, int MT>
static int paged_few(PagedAttn p, const PagedCache& c, const PagedPlan& s, int kv_heads, bool pdl, zl_stream_t stream) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        ZL_CHECK_CUDA(cudaFuncSetAttribute(k_paged_attn_few<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, PfCfg<D>::kBytes));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    ZL_CHECK_CUDA(launch(k_paged_attn_few<T, D, MT>, dim3(s.ctas), dim3(kPfWarps * 32), PfCfg<D>::kBytes, stream, pdl, p, c, kv_heads));
    if (s.ctas > 1) ZL_CHECK_CUDA(launch(k_paged_few_join<T, D, MT>, dim3(s.ctas), dim3(kPfWarps * 32), 0, stream, true, p, c, kv_heads));
    return ZL_OK;
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
    uint8_t* ws = reinterpret_cast<uint8_t*>(p.ml);
    p.few = !s.tiles ? INT_MAX : s.few ? kFewRows : 0;
    if (s.few) {
        p.ml = reinterpret_cast<float2*>(ws + s.few_ml), p.part = reinterpret_cast<float*>(ws + s.few_part);
        const int rc = s.few_rows == 16 ? paged_few<T, D, 1>(p, c, s, kv_heads, pdl != 0, stream) : paged_few<T, D, 2>(p, c, s, kv_heads, pdl != 0, stream);
        if (rc) return rc;
    }
    if (s.tiles) {
        p.ml = reinterpret_cast<float2*>(ws + s.ml), p.part = reinterpret_cast<float*>(ws + s.part);
        // behind the other kernels of this call it may be launched early whatever the caller's chain allows: it waits for them to end
        ZL_CHECK_CUDA(launch(k_paged_attn_tiles<T, D>, dim3(s.blocks * s.splits, kv_heads), dim3(kPtThreads), PtCfg<D>::kBytes, stream, pdl != 0 || s.few, p, c,
                             words + kWaitAttnPaged));
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
    // the kernels count tiles in 32 bits
    ZL_CHECK_SUPPORTED(((long long)rows * (heads / kv_heads) / 16 + seqs) * (room / kPfKeys + 1) < INT_MAX / kv_heads);
    ZL_CHECK_ARG(s.bytes == 0 || (workspace && workspace_bytes >= s.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0));
    const PagedCache c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages,
                          page_size, seqs, paged_divisor(page_size)};
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, heads / kv_heads, window, scale * 1.4426950408889634f, 0, s.splits ? s.splits : 1,
                         static_cast<float2*>(workspace), nullptr};
    if (dtype == ZL_F16) return dim == 64 ? paged_attention<__half, 64>(p, c, s, kv_heads, pdl, stream) : paged_attention<__half, 128>(p, c, s, kv_heads, pdl, stream);
    return dim == 64 ? paged_attention<__nv_bfloat16, 64>(p, c, s, kv_heads, pdl, stream) : paged_attention<__nv_bfloat16, 128>(p, c, s, kv_heads, pdl, stream);
}
