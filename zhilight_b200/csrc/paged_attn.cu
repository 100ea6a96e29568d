// Attention of the new tokens of every sequence over its pages.  Row i of the n_b new rows of sequence b stands at place p = len_b - n_b + i of the
// sequence and sees the keys j <= p, with a window w those with j > p - w too: o = sum_j softmax_j(scale q k_j) v_j, zeros where it sees none.
#include "paged_attn_few.cuh"
#include "paged_attn_tc.cuh"

#include <climits>

namespace zl {

constexpr int kFewRows = 32;   // (token, head) rows of a kv head that a sequence brings to the kernel for few rows

struct PagedPlan {
    bool tiles, few;              // which kernels run
    int ctas, few_ctas, few_rows; // their CTAs; rows of a block of the few
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
    // no more CTAs than the line can be long: every sequence adds less than one block to those of the rows, each of all the keys there is room for
    if (s.tiles) {
        const long long turns = (all / kPtRows + seqs) * cdiv(max_keys, kPtKeys) * kv_heads;
        s.ctas = (int)(turns < sms ? turns : sms);
        const size_t parts = (size_t)s.ctas * 2 * kPtRows;
        s.ml = take(parts * sizeof(float2)), s.part = take(parts * dim * sizeof(float));
    }
    if (s.few) {
        s.few_rows = most <= 16 ? 16 : 32;
        const long long tiles = (all / s.few_rows + seqs) * cdiv(max_keys, kPfKeys) * kv_heads;
        s.few_ctas = (int)(tiles < kPfPerSm * sms ? tiles : kPfPerSm * sms);
        const size_t parts = (size_t)s.few_ctas * 2 * s.few_rows;
        s.few_ml = take(parts * sizeof(float2)), s.few_part = take(parts * dim * sizeof(float));
    }
    return s;
}

// once for every device: `done` remembers
template <typename... KArgs>
static cudaError_t allow_smem(void (*kernel)(KArgs...), int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return e;
}

template <typename T, int D, int MT>
static int paged_few(PagedAttn p, const PagedCache& c, const PagedPlan& s, void* ws, bool pdl, zl_stream_t stream) {
    static bool done[64] = {};
    ZL_CHECK_CUDA(allow_smem(k_paged_attn_few<T, D, MT>, PfCfg<D>::kBytes, done));
    p.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws) + s.few_ml), p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + s.few_part);
    ZL_CHECK_CUDA(launch(k_paged_attn_few<T, D, MT>, dim3(s.few_ctas), dim3(kPfWarps * 32), PfCfg<D>::kBytes, stream, pdl, p, c));
    if (s.few_ctas > 1)
        ZL_CHECK_CUDA(launch(k_paged_join<T, D, PfKind<16 * MT>, false>, dim3(s.few_ctas, MT), dim3(kJoinThreads), 0, stream, true, p, c, 0, p.few));
    return ZL_OK;
}

template <typename T, int D>
static int paged_tiles(PagedAttn p, const PagedCache& c, const PagedPlan& s, void* ws, bool pdl, zl_stream_t stream) {
    static bool done[64] = {};
    ZL_CHECK_WAITS();
    unsigned* words = wait_words();
    ZL_CHECK_CUDA(words ? cudaSuccess : cudaErrorMemoryAllocation);
    ZL_CHECK_CUDA(allow_smem(k_paged_attn_tiles<T, D>, PtCfg<D>::kBytes, done));
    p.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ws) + s.ml), p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + s.part);
    // boxes: the rows that a tile and a page have in common wherever they meet
    int box = 1;
    while (box < kPtKeys && c.page_size % (2 * box) == 0) box *= 2;
    CUtensorMap maps[2] = {};
    if (box >= 8) {
        const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        auto step = [](long long elements, int n) { return n > 1 ? (uint64_t)elements * 2 : (uint64_t)(D * 2); };   // of one alone none is taken
        const uint64_t dims[4] = {(uint64_t)D, (uint64_t)c.page_size, (uint64_t)p.kv_heads, (uint64_t)c.num_pages};
        const uint64_t strides[3] = {step(c.row_stride, c.page_size), step(c.head_stride, p.kv_heads), step(c.page_stride, c.num_pages > 1 ? 2 : 1)};
        const uint32_t rows[4] = {64, (uint32_t)box, 1, 1};
        for (int i = 0; i < 2; ++i)
            if (!tc_make_map_nd(&maps[i], i ? c.v : c.k, dt, 4, dims, strides, rows, CU_TENSOR_MAP_SWIZZLE_128B)) box = 0;
    } else {
        box = 0;
    }
    ZL_CHECK_CUDA(launch(k_paged_attn_tiles<T, D>, dim3(s.ctas), dim3(kPtThreads), PtCfg<D>::kBytes, stream, pdl, p, c, maps[0], maps[1], box, words + kWaitAttnPaged));
    if (s.ctas > 1)
        ZL_CHECK_CUDA(launch(k_paged_join<T, D, PtKind, true>, dim3(s.ctas, kPtRows / kJoinRows), dim3(kJoinThreads), 0, stream, true, p, c, p.few, INT_MAX));
    return ZL_OK;
}

template <typename T, int D>
static int paged_attention(PagedAttn p, const PagedCache& c, const PagedPlan& s, void* ws, bool pdl, zl_stream_t stream) {
    p.few = !s.tiles ? INT_MAX : s.few ? kFewRows : 0;
    int rc = ZL_OK;
    if (s.few) rc = s.few_rows == 16 ? paged_few<T, D, 1>(p, c, s, ws, pdl, stream) : paged_few<T, D, 2>(p, c, s, ws, pdl, stream);
    // behind the other kernels of this call it may be launched early whatever the caller's chain allows: it waits for them to end
    if (rc == ZL_OK && s.tiles) rc = paged_tiles<T, D>(p, c, s, ws, pdl || s.few, stream);
    return rc;
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
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, heads / kv_heads, window, paged_divisor(heads / kv_heads), scale * 1.4426950408889634f, 0, kv_heads, nullptr, nullptr};
    if (dtype == ZL_F16)
        return dim == 64 ? paged_attention<__half, 64>(p, c, s, workspace, pdl != 0, stream) : paged_attention<__half, 128>(p, c, s, workspace, pdl != 0, stream);
    return dim == 64 ? paged_attention<__nv_bfloat16, 64>(p, c, s, workspace, pdl != 0, stream)
                     : paged_attention<__nv_bfloat16, 128>(p, c, s, workspace, pdl != 0, stream);
}
