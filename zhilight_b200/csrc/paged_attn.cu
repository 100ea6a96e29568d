// Attention of the new tokens of every sequence over its pages.  Row i of the n_b new rows of sequence b stands at place p = len_b - n_b + i of the
// sequence and sees the keys j <= p, with a window w those with j > p - w too: o = sum_j softmax_j(scale q k_j) v_j, zeros where it sees none.
#include "paged_attn_few.cuh"
#include "paged_attn_tc.cuh"

#include <climits>

namespace zl {

// Calls whose sequences bring at most so many (token, head) rows of a kv head each go to the kernel for few rows, as do groups that no tile holds a token of.
// us in a graph, it / the tiles, 32 heads on 8, 2000 keys: 16 sequences with 4 rows 35 / 48, with 16 rows 37 / 49; two with 16 rows 16 / 24; one with 16 rows on 30000
// keys 41 / 54.  A variant for 32 rows took 58 to 60 where the tiles took 53 (16 sequences; 26 / 28 for two, 66 / 70 for one on 30000 keys) and was left out.
// The line is drawn for groups of 4 and 8.  Single tokens of wider ones, in blocks of 16 rows here: 16 sequences of 2000 keys with 20 or 32 heads on one 19 / 25,
// 64 heads 25 / 25, 128 heads 39 / 24; one sequence of 30000 keys 34 to 38 for all of these, 76 to 84 on the tiles, to which these calls go.
constexpr int kFewRows = kPfRows;

struct PagedPlan {
    bool tiles;                       // on the 5th-generation tensor cores
    int ctas, block_rows, tile_rows, places;   // rows of a place in the workspace
    size_t ml, part, cuts, bytes;     // what lies where in it
};

static PagedPlan paged_plan(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    PagedPlan s = {};
    const int group = heads / kv_heads, sms = device_sm_count();
    const long long all = (long long)rows * group, most = (long long)max_new * group;
    s.tiles = most > kFewRows && group <= kPaRows;
    s.tile_rows = s.tiles ? kPaRows / group * group : 0;
    s.block_rows = s.tiles ? 2 * s.tile_rows : kPfRows;
    s.places = s.tiles ? kPtRows : kPfRows;
    // no more CTAs than the line can be long: every sequence adds less than one block to those of the rows, each of all the keys there is room for
    const long long units = (all / s.block_rows + seqs) * (s.tiles ? PtKind::kSetup + cdiv(max_keys, kPtKeys) : PfKind::kSetup + cdiv(max_keys, kPfKeys)) * kv_heads;
    const int most_ctas = s.tiles ? sms : kPfPerSm * sms;
    s.ctas = (int)(units < most_ctas ? units : most_ctas);
    const size_t parts = (size_t)s.ctas * 2 * s.places;
    auto take = [&](size_t bytes) {
        const size_t at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    s.ml = take(parts * sizeof(float2)), s.part = take(parts * dim * sizeof(float)), s.cuts = take((size_t)s.ctas * sizeof(PagedCut));
    return s;
}

template <typename T, int D>
static int paged_few(const PagedAttn& p, const PagedCache& c, int ctas, bool pdl, zl_stream_t stream) {
    static bool done[64] = {};
    ZL_CHECK_CUDA(allow_smem(k_paged_attn_few<T, D>, PfCfg<D>::kBytes, done));
    ZL_CHECK_CUDA(launch(k_paged_attn_few<T, D>, dim3(ctas), dim3(kPfWarps * 32), PfCfg<D>::kBytes, stream, pdl, p, c));
    if (ctas > 1) ZL_CHECK_CUDA(launch(k_paged_join<T, D, kPfRows>, dim3(ctas), dim3(kJoinWarps * 32), 0, stream, true, p));
    return ZL_OK;
}

template <typename T, int D>
static int paged_tiles(const PagedAttn& p, const PagedCache& c, int ctas, bool pdl, zl_stream_t stream) {
    static bool done[64] = {};
    ZL_CHECK_WAITS();
    unsigned* words = wait_words();
    ZL_CHECK_CUDA(words ? cudaSuccess : cudaErrorMemoryAllocation);
    ZL_CHECK_CUDA(allow_smem(k_paged_attn_tiles<T, D>, PtCfg<D>::kBytes, done));
    const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap maps[3] = {};
    ZL_CHECK_CUDA(pt_q_map<D>(&maps[0], p, dt) ? cudaSuccess : cudaErrorInvalidValue);
    // boxes of K and V: the rows that a tile and a page have in common wherever they meet
    int box = 1;
    while (box < kPtHalf && c.page_size % (2 * box) == 0) box *= 2;
    if (box < 4 || c.page_size < 8) box = 0;   // a turn's 256 keys in the 32 pages that a warp's lanes know; smaller boxes are more copies than 16 bytes at a time save
    if (box) {
        auto step = [](long long elements, bool more) { return more ? (uint64_t)elements * 2 : (uint64_t)(D * 2); };   // of one alone none is taken
        const uint64_t dims[4] = {(uint64_t)D, (uint64_t)c.page_size, (uint64_t)p.kv_heads, (uint64_t)c.num_pages};
        const uint64_t strides[3] = {step(c.row_stride, c.page_size > 1), step(c.head_stride, p.kv_heads > 1), step(c.page_stride, c.num_pages > 1)};
        const uint32_t rows[4] = {64, (uint32_t)box, 1, 1};
        for (int i = 0; i < 2; ++i)
            if (!tc_make_map_nd(&maps[1 + i], i ? c.v : c.k, dt, 4, dims, strides, rows, CU_TENSOR_MAP_SWIZZLE_128B)) box = 0;
    }
    ZL_CHECK_CUDA(launch(k_paged_attn_tiles<T, D>, dim3(ctas), dim3(kPtThreads<false>), PtCfg<D>::kBytes, stream, pdl, p, c, maps[0], maps[1], maps[2], box,
                         words + kWaitAttnPaged));
    if (ctas > 1) ZL_CHECK_CUDA(launch(k_paged_join_tiles<T, D>, dim3(ctas, kPtRows / 32), dim3(256), 0, stream, true, p));
    return ZL_OK;
}

int paged_tiles(const PagedAttn& p, const PagedCache& c, int ctas, int dim, int dtype, bool pdl, zl_stream_t stream) {
    if (dtype == ZL_F16) return dim == 64 ? paged_tiles<__half, 64>(p, c, ctas, pdl, stream) : paged_tiles<__half, 128>(p, c, ctas, pdl, stream);
    return dim == 64 ? paged_tiles<__nv_bfloat16, 64>(p, c, ctas, pdl, stream) : paged_tiles<__nv_bfloat16, 128>(p, c, ctas, pdl, stream);
}

template <typename T, int D>
static int paged_attention(const PagedAttn& p, const PagedCache& c, const PagedPlan& s, bool pdl, zl_stream_t stream) {
    return s.tiles ? paged_tiles<T, D>(p, c, s.ctas, pdl, stream) : paged_few<T, D>(p, c, s.ctas, pdl, stream);
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
    ZL_CHECK_SUPPORTED(((long long)rows * (heads / kv_heads) / 16 + seqs) * (room / kPfKeys + 4) < (INT_MAX - (1 << 16)) / kv_heads);   // with room for a stretch more
    ZL_CHECK_ARG(workspace && workspace_bytes >= s.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0);
    const PagedCache c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages,
                          page_size, seqs, paged_divisor(page_size)};
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, heads / kv_heads, window, paged_divisor(heads / kv_heads), scale * 1.4426950408889634f, kv_heads,
                         s.block_rows, s.tile_rows, reinterpret_cast<float2*>(ws + s.ml), reinterpret_cast<float*>(ws + s.part), reinterpret_cast<PagedCut*>(ws + s.cuts)};
    if (dtype == ZL_F16) return dim == 64 ? paged_attention<__half, 64>(p, c, s, pdl != 0, stream) : paged_attention<__half, 128>(p, c, s, pdl != 0, stream);
    return dim == 64 ? paged_attention<__nv_bfloat16, 64>(p, c, s, pdl != 0, stream) : paged_attention<__nv_bfloat16, 128>(p, c, s, pdl != 0, stream);
}
