// Attention of the new tokens of every sequence over pages of 4 bits (int4_cache.cuh): what paged_attn.cu does over pages of 16.
#include "paged_attn4_few.cuh"
#include "paged_attn_tc.cuh"

#include <climits>

namespace zl {

// Calls whose sequences bring at most so many (token, head) rows of a kv head go to the kernel for few rows, and all where groups have more heads than a tile has rows.
// Drafts of 16 sequences, 48 rows, up to 6000 keys: 49 us there, in three blocks, 87 on the tiles, whose blocks of up to 128 rows cost the same.
// Few rows / tiles in us, by the rows of a kv head (groups of 8, bf16, heads of 128, 8 kv heads; fp16 and heads of 64 have their borders within 16 rows of these):
//   keys        1 x 1000   1 x 8000   1 x 60000   4 x 6000   16 x 1000   16 x 6000   64 x 300   64 x 2000
//   32 rows     12 / 17    22 / 30    58 / 85     32 / 48    26 / 35      84 / 136   39 / 76    113 / 213
//   48          13 / 18    24 / 30    79 / 90     41 / 50    35 / 36     119 / 138   51 / 78    163 / 217
//   64          15 / 18    26 / 30    97 / 86     50 / 50    41 / 36     151 / 138   66 / 76    213 / 213
//   80          15 / 19    28 / 30   118 / 91     56 / 51    52 / 36     188 / 138   95 / 78    279 / 221
// Of other calls, those sequences go there that bring a token or two of a group of up to 8 heads, or up to 16 rows: portions of prompts beside 20 single tokens (24 sequences, keys in a
// window of 1024) 71 us, 95 with all on the tiles.
// Few keys are not worth two launches more.  By the room that the page table has (lengths are the device's), us with both kernels / the tiles alone, a portion beside single tokens: two
// sequences of 740 keys 29 / 21, four of 2000 36 / 35, eight of 1000 28 / 28, eight of 4500 51 / 77, two of 30000 47 / 81, eight of 30000 97 / 249.
constexpr int kFewRows4 = 64, kFewBeside = 16, kBesideKeys = 8192;

// what lies where in the workspace, for one of the two kernels
struct Paged4Plan {
    int ctas, block_rows, tile_rows;   // ctas 0: it is not launched
    size_t ml, part, cuts;
};
struct Paged4Plans {
    Paged4Plan few, tiles;
    int split;                         // rows of a sequence for the kernel for few
    int wide_pages;                    // pages of 64 rows a sequence, of keys and values in 16 bits for the tiles; 0: the tiles make codes numbers by themselves
    size_t k, v, table, bytes;
};

// The tiles make every key's codes numbers once for each block of rows, which bounds them: 2048 tokens of 32 heads on 8 behind 6000 302 us.  Made numbers once, beforehand, in the workspace, they
// are read like a cache of 16 bits: 242.  The workspace has room for all that the page table has room for, so that is done up to this size of it; what is
// written there are only the keys that portions see.  And only from some blocks of rows on, by the rows / beforehand: 64 tokens behind 4000 27 / 30 us, 300 behind 300 23 / 25,
// 100 of four sequences behind 1000 40 / 39, 1000 behind 1000 61 / 53, 200 behind 30000 242 / 192.
constexpr size_t kWideBytes = 256u << 20;
constexpr int kWidePage = 64, kWideShares = 4, kWideRows = 512;

static Paged4Plans paged4_plan(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    Paged4Plans s = {};
    const int group = heads / kv_heads;
    const long long all = (long long)rows * group, most = (long long)max_new * group;
    const bool tiles = most > kFewRows4 && group <= kPaRows;
    auto take = [&](size_t bytes) {
        const size_t at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    auto plan = [&](Paged4Plan& p, int block_rows, int places, int block_units, int most_ctas) {
        // no more CTAs than the line can be long: every sequence adds less than one block to those of the rows, each of all the keys there is room for
        const long long units = (all / block_rows + seqs) * block_units * kv_heads;
        p.block_rows = block_rows;
        p.ctas = (int)(units < most_ctas ? units : most_ctas);
        const size_t parts = (size_t)p.ctas * 2 * places;
        p.ml = take(parts * sizeof(float2)), p.part = take(parts * dim * sizeof(float)), p.cuts = take((size_t)p.ctas * sizeof(PagedCut));
    };
    if (tiles) {
        s.tiles.tile_rows = kPaRows / group * group;
        plan(s.tiles, 2 * s.tiles.tile_rows, kPtRows, PtKind::kSetup + cdiv(max_keys, kPtKeys), device_sm_count());
    }
    if (tiles) {
        const long long pages = ((long long)max_keys + kWidePage - 1) / kWidePage;
        const size_t each = (size_t)kv_heads * kWidePage * dim * 2;
        if (most > kWideRows && (unsigned long long)seqs * pages * each * 2 <= kWideBytes) {
            s.wide_pages = (int)pages;
            s.k = take(seqs * pages * each), s.v = take(seqs * pages * each), s.table = take(seqs * pages * sizeof(int32_t));
        }
    }
    if (!tiles || (seqs > 1 && (long long)seqs * max_keys >= kBesideKeys && group <= kFewBeside)) {   // wider groups are no few rows
        const bool eight = (tiles ? group : most) <= 8;   // beside the tiles: single tokens, mostly
        s.split = !tiles ? INT_MAX : eight ? 8 : kFewBeside;
        plan(s.few, eight ? 8 : 16, eight ? 8 : 16, P4Kind::kSetup + cdiv(max_keys, kP4Keys), kP4PerSm * device_sm_count());
    }
    return s;
}

// Boxes of 16 rows of K and of V (int4_box), as words of 32 bits: -> kInt4Copies where there are none
template <int D>
static int p4_maps(CUtensorMap (&maps)[2], const PagedAttn& p, const PagedCache& c) {
    constexpr int kRow = int4_row_bytes(D), kWords = kRow / 4;
    if (c.page_size % 16 != 0) return kInt4Copies;
    const bool run = D == 128 || c.row_stride == kRow, wide = !run && (p.kv_heads == 1 || c.head_stride == kRow);
    if (!run && !wide) return kInt4Copies;
    auto step = [](long long bytes, bool more) { return more ? (uint64_t)bytes : 16u; };   // of one alone none is taken
    const bool rows = D == 128 || wide;
    const uint64_t dims[4] = {(uint64_t)(D == 128 ? kWords : wide ? p.kv_heads * kWords : c.page_size * kWords), (uint64_t)(rows ? c.page_size : 1), (uint64_t)(wide ? 1 : p.kv_heads),
                              (uint64_t)c.num_pages};
    const uint64_t strides[3] = {step(c.row_stride, rows), step(c.head_stride, !wide && p.kv_heads > 1), step(c.page_stride, c.num_pages > 1)};
    const uint32_t box[4] = {(uint32_t)(D == 128 ? kWords : wide ? 12 : 16 * kWords), rows ? 16u : 1u, 1, 1};
    for (int i = 0; i < 2; ++i)
        if (!tc_make_map_nd(&maps[i], i ? c.v : c.k, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return kInt4Copies;
    return wide ? kInt4Wide : kInt4Run;
}

template <typename T, int D, int NT>
static int paged4_few(const PagedAttn& p, const PagedCache& c, int ctas, bool pdl, zl_stream_t stream) {
    using C = P4Cfg<D, NT>;
    static bool done[64] = {};
    ZL_CHECK_CUDA(allow_smem(k_paged_attn4_few<T, D, NT>, C::kBytes, done));
    CUtensorMap maps[2] = {};
    const int form = p4_maps<D>(maps, p, c);
    ZL_CHECK_CUDA(launch(k_paged_attn4_few<T, D, NT>, dim3(ctas), dim3(kP4Warps * 32), C::kBytes, stream, pdl, p, c, maps[0], maps[1], form, wait_words() + kWaitAttnPaged));
    if (ctas > 1) ZL_CHECK_CUDA(launch(k_paged_join<T, D, 8 * NT>, dim3(ctas), dim3(kJoinWarps * 32), 0, stream, true, p));
    return ZL_OK;
}

template <typename T, int D>
static int paged4_tiles(const PagedAttn& p, const PagedCache& c, int ctas, bool pdl, zl_stream_t stream) {
    using C = PtCfg<D, true>;
    static bool done[64] = {};
    ZL_CHECK_CUDA(allow_smem(k_paged_attn_tiles<T, D, true>, C::kBytes, done));
    CUtensorMap q_map = {}, maps[2] = {};
    const int form = p4_maps<D>(maps, p, c);
    const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    ZL_CHECK_CUDA(pt_q_map<D>(&q_map, p, dt) ? cudaSuccess : cudaErrorInvalidValue);
    ZL_CHECK_CUDA(launch(k_paged_attn_tiles<T, D, true>, dim3(ctas), dim3(kPtThreads<true>), C::kBytes, stream, pdl, p, c, q_map, maps[0], maps[1], form, wait_words() + kWaitAttnPaged));
    if (ctas > 1) ZL_CHECK_CUDA(launch(k_paged_join_tiles<T, D>, dim3(ctas, kPtRows / 32), dim3(256), 0, stream, true, p));
    return ZL_OK;
}

// Keys and values of a tile of 64 rows of a sequence as numbers: grid (tiles, sequences, shares of the work).  Tiles that no row of the kernel for tiles sees, and sequences of few rows, are left out.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_paged4_wide(const PagedAttn p, const PagedCache c, T* __restrict__ k_out, T* __restrict__ v_out, int32_t* table) {
    constexpr int kPieces = D / 16, kAhead = 4;
    __shared__ long long s_off[kWidePage];
    const int tid = threadIdx.x, b = blockIdx.y, row0 = blockIdx.x * kWidePage, page = b * gridDim.x + blockIdx.x;
    pdl_trigger();
    pdl_wait();
    if (tid == 0 && blockIdx.z == 0) table[page] = page;
    const int from = max(p.starts[b], 0), tokens = max(min(p.starts[b + 1], p.rows), from) - from, len = p.lens[b], place0 = len - p.starts[b + 1] + from, have = min(max(len, 0), c.room());
    const int hi = min(place0 + tokens - 1, have - 1), lo = paged_from(p, place0) / kPtKeys * kPtKeys;
    if (!PtKind::takes(p, tokens * p.group) || row0 > hi || row0 + kWidePage <= lo) return;
    if (tid < kWidePage) s_off[tid] = row0 + tid <= hi ? c.row_at(b, row0 + tid) : -1;
    __syncthreads();
    const int half = p.kv_heads * kWidePage * kPieces, items = 2 * half;   // a cache's page; both
    for (int i0 = (int)blockIdx.z * (kAhead * 256) + tid; i0 < items; i0 += (int)gridDim.z * (kAhead * 256)) {
        uint2 codes[kAhead];
        uint32_t meta[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * 256, piece = i % kPieces, row = i / kPieces % kWidePage, head = i / (kPieces * kWidePage), is_v = head >= p.kv_heads;
            codes[u] = make_uint2(0u, 0u), meta[u] = 0;
            if (i >= items || s_off[row] < 0) continue;
            const uint8_t* at = static_cast<const uint8_t*>(is_v ? c.v : c.k) + s_off[row] + (long long)(head - (is_v ? p.kv_heads : 0)) * c.head_stride;
            codes[u] = *reinterpret_cast<const uint2*>(at + piece * 8);
            meta[u] = *reinterpret_cast<const uint32_t*>(at + D / 2 + piece / 2 * 4);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * 256;
            const bool odd = i & 1, is_v = i >= half;
            const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? codes[u].x : codes[u].y, 1);   // two lanes have a group of 32 columns (int4 values)
            if (i >= items) continue;
            uint32_t step, low;
            int4_meta<T>(meta[u], step, low);
            uint4* to = reinterpret_cast<uint4*>(is_v ? v_out : k_out) + ((size_t)page * half + i - (is_v ? half : 0)) * 2 - odd;
            to[0] = int4_eight<T>(odd ? other : codes[u].x, step, low);
            to[2] = int4_eight<T>(odd ? codes[u].y : other, step, low);
        }
    }
}

template <typename T, int D>
static int paged4(PagedAttn p, const PagedCache& c, const Paged4Plans& s, uint8_t* ws, bool pdl, zl_stream_t stream) {
    ZL_CHECK_WAITS();
    ZL_CHECK_CUDA(wait_words() ? cudaSuccess : cudaErrorMemoryAllocation);
    auto with = [&](const Paged4Plan& plan) {
        p.block_rows = plan.block_rows, p.tile_rows = plan.tile_rows;
        p.ml = reinterpret_cast<float2*>(ws + plan.ml), p.part = reinterpret_cast<float*>(ws + plan.part), p.cuts = reinterpret_cast<PagedCut*>(ws + plan.cuts);
    };
    const bool both = s.few.ctas && s.tiles.ctas;
    p.split = s.split;
    if (s.few.ctas) {
        with(s.few);
        const int rc = s.few.block_rows == 8 ? paged4_few<T, D, 1>(p, c, s.few.ctas, pdl, stream) : paged4_few<T, D, 2>(p, c, s.few.ctas, pdl, stream);
        if (rc || !both) return rc;
    }
    with(s.tiles);
    if (!both) p.split = 0;
    if (s.wide_pages == 0) return paged4_tiles<T, D>(p, c, s.tiles.ctas, pdl || both, stream);
    T *k = reinterpret_cast<T*>(ws + s.k), *v = reinterpret_cast<T*>(ws + s.v);
    int32_t* table = reinterpret_cast<int32_t*>(ws + s.table);
    ZL_CHECK_CUDA(launch(k_paged4_wide<T, D>, dim3(s.wide_pages, c.seqs, kWideShares), dim3(256), 0, stream, pdl || both, p, c, k, v, table));
    const long long rows = (long long)c.max_pages * c.page_size;   // below 2^31, or the workspace would be larger
    const PagedCache wide = {k, v, (long long)c.seqs * s.wide_pages, (long long)p.kv_heads * kWidePage * D, D, kWidePage * D, table, s.wide_pages, s.wide_pages, kWidePage, c.seqs,
                             paged_divisor(kWidePage), (int)rows};
    return paged_tiles(p, wide, s.tiles.ctas, D, std::is_same<T, __half>::value ? ZL_F16 : ZL_BF16, true, stream);
}

}  // namespace zl

using namespace zl;

extern "C" size_t zl_paged_attention_int4_workspace_bytes(int rows, int max_new, int seqs, int max_keys, int heads, int kv_heads, int dim) {
    if (rows <= 0 || max_new <= 0 || seqs <= 0 || max_keys <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0) return 0;
    return paged4_plan(rows, max_new, seqs, max_keys, heads, kv_heads, dim).bytes;
}

extern "C" int zl_paged_attention_int4(const void* q, const void* k_cache, const void* v_cache, long long num_pages, int page_size, long long page_stride,
                                       long long row_stride, long long head_stride, const int32_t* page_table, int ld_table, int max_pages,
                                       const int32_t* seq_lens, const int32_t* q_starts, int seqs, float scale, int window, void* out, int rows, int max_new,
                                       int heads, int kv_heads, int dim, void* workspace, size_t workspace_bytes, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(q && seq_lens && q_starts && out && rows > 0 && max_new > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0);
    ZL_CHECK_ARG(scale > 0.f && scale < INFINITY && window >= 0);
    ZL_CHECK_PAGED_INT4(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, dim);
    ZL_CHECK_ARG(page_table && max_pages > 0 && ld_table >= max_pages && seqs > 0);
    ZL_CHECK_SUPPORTED(dtype == ZL_F16 || dtype == ZL_BF16);
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0);
    ZL_CHECK_SUPPORTED(dtype == ZL_F16 || scale <= 0x1p64f);   // products with bf16 keys carry 2^-20 (Int4Codes), which the scale takes away: neither that nor the smallest sums may leave 32 bits
    ZL_CHECK_SUPPORTED(heads <= 65535 && (long long)rows * heads < INT_MAX);
    const long long room = (long long)max_pages * page_size;
    const Paged4Plans s = paged4_plan(rows, max_new, seqs, (int)(room < INT_MAX - 255 ? room : INT_MAX - 255), heads, kv_heads, dim);
    // the kernels count tiles in 32 bits
    const int least_rows = s.few.ctas ? s.few.block_rows : kPaRows / 2;   // of a block
    ZL_CHECK_SUPPORTED(((long long)rows * (heads / kv_heads) / least_rows + seqs) * (room / kP4Keys + 2 + P4Kind::kSetup) < (INT_MAX - (1 << 16)) / kv_heads);
    ZL_CHECK_ARG(workspace && workspace_bytes >= s.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0);
    const PagedCache c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages,
                          page_size, seqs, paged_divisor(page_size)};
    const PagedAttn p = {q, out, seq_lens, q_starts, rows, heads, heads / kv_heads, window, paged_divisor(heads / kv_heads), scale * 1.4426950408889634f, kv_heads};
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (dtype == ZL_F16) return dim == 64 ? paged4<__half, 64>(p, c, s, ws, pdl != 0, stream) : paged4<__half, 128>(p, c, s, ws, pdl != 0, stream);
    return dim == 64 ? paged4<__nv_bfloat16, 64>(p, c, s, ws, pdl != 0, stream) : paged4<__nv_bfloat16, 128>(p, c, s, ws, pdl != 0, stream);
}
