// Attention of few (token, head) rows of a kv head over pages of 4 bits (int4_cache.cuh).  Work is shared out as in paged_attn_few.cuh: tiles of 128 keys of all
// blocks stand in one line, a CTA takes an equal stretch, a warp has 32 keys of a tile and a ring of its own.
//
// What 4 bits take off the memory they put on the instructions: a key and its value are 160 bytes instead of 512, and every code costs more than one of them.
// So the products are turned around, S^T = K Q^T and O^T += V^T P^T by mma.sync with the keys' and values' 16 rows as the first operand and 8 rows of queries as the
// second: blocks of 8 rows (one token of a group of 8, two of 4) take half the products, exponentials and registers that 16 rows would.
//   K: columns may be summed in any order as long as Q's are in the same one, so lane (g, t) takes a quarter of the columns of keys g and g + 8 in one piece,
//      one 16-byte load and one pair (step, lowest) each.
//   V: the operand wants two keys in a register; codes of two keys come together by one byte permutation per four columns, before they become numbers, so
//      that this costs an eighth of an instruction a value.  Output columns may lie anywhere: lane g takes D / 8 neighbouring ones.
//   P: the scores' accumulators, rounded to 16 bits, are the second operand once 8 x 8 of them are transposed (movmatrix).
// Probabilities are rounded to the rows' type once (half a step each, of random sign: beside the output's own rounding), sums are in 32 bits: errors of 2.3e-3 against 64 bits, 1.7e-3
// with probabilities of two 16-bit values, for which a long sequence takes 8 % longer and drafts 14: the cache's own steps are far coarser.
//
// One token over 131072 keys, 32 heads on 8: 48 us a call in a graph, 51 in a row of eager ones (168 MB; with 16 bits 103), 45 of them in this kernel under ncu: bound by instructions, of which
// an SM's schedulers issue one in 55 % of the cycles (396 for 16 keys of a warp), while HBM is busy 46 %.  32 sequences
// with up to 4096 keys, fp16, whose codes take more instructions: 27 us.  On the way, a long sequence in us: copies of 16 bytes by all lanes, with their addresses, 69;
// boxes and one fma for two codes 55; 32 keys of a warp at a time, so that what a tile costs beside its products is there half as often, 49; three CTAs an SM 48.
//
// Codes of bf16 rows become numbers by one `and` and one fma for two (Int4Codes).  16 rows of a head come by one TMA box where a page holds whole 16s of them, else by copies
// (kInt4Copies ...).
#pragma once
#include "int4_cache.cuh"
#include "paged_attn_few.cuh"
#include "paged_attn_tc.cuh"

namespace zl {

constexpr int kP4Warps = 4, kP4Each = 32, kP4Keys = kP4Each * kP4Warps, kP4Stages = 2, kP4PerSm = 3;   // four CTAs of 128 registers an SM: decoding 28.2 us, a long sequence 48.8; three 26.9 and 48.0

template <int D, int NT>
struct P4Cfg {
    static constexpr int kChunk = D / 8;                             // bytes copied at once; of a row, four chunks of codes and one of pairs
    static constexpr int kV = kP4Each * kInt4Pitch<D>, kStage = 2 * kV;   // rows of K, then of V
    static constexpr int kWarp = kP4Stages * kStage;
    static constexpr int kBytes = kP4Warps * kWarp;
    static constexpr int kPitch = D + 8;                             // floats; of a row of a warp's output in its ring
    static_assert(8 * NT * kPitch * 4 <= kWarp, "a warp's output, where its ring was");
};

// tiles of 128 keys; at least one: a block that sees nothing is written too
struct P4Kind {
    static constexpr int kSetup = 2;
    static __device__ __forceinline__ bool takes(const PagedAttn& p, int rows) { return rows <= p.split; }
    static __device__ __forceinline__ int turns(const PagedAttn&, const PagedBlock& k) { return k.hi >= 0 ? k.hi / kP4Keys - k.lo / kP4Keys + 1 : 1; }
};

template <int BYTES>
__device__ __forceinline__ void p4_copy(uint32_t dst, const void* src, int bytes) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t p4_transpose(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// N words in one load
template <int N>
__device__ __forceinline__ void p4_words(uint32_t (&w)[N], const uint8_t* at) {
    if constexpr (N == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        w[0] = x.x, w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(at);
    }
}

// grid: CTAs that share the line; blocks of up to 8 NT rows.  tma: one of kInt4Copies ...
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kP4Warps * 32, kP4PerSm)
k_paged_attn4_few(const PagedAttn p, const PagedCache c, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, int tma, unsigned* err) {
    using C = P4Cfg<D, NT>;
    constexpr bool kHalf = std::is_same<T, __half>::value, kScaled = Int4Codes<T, false>::kScaled;
    constexpr int R = 8 * NT, KS = D / 16, MT = D / 16, KW = D / 32, VW = D / 64;
    // Values times 2^-20 take probabilities of 2^20 more: products and the sums that become parts are those of PagedExp, and the probabilities' sum follows at the end.
    constexpr float kTau = PagedExp<kHalf>::kTau, kUp = PagedExp<kHalf>::kUp + (kScaled ? 20.f : 0.f);
    extern __shared__ __align__(128) uint8_t p4_smem[];
    __shared__ float2 s_ml[kP4Warps][R];
    __shared__ uint64_t full[kP4Warps][kP4Stages];
    __shared__ int s_gave_up;
    volatile int* s_abort = &s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    uint8_t* ring = p4_smem + warp * C::kWarp;
    const uint32_t ring_at = smem_u32(ring);
    if (lane == 0)
        for (int i = 0; i < kP4Stages; ++i) mbar_init(&full[warp][i], 1);
    if (tid == 0) s_gave_up = 0;
    mbar_fence_init();
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    if (tid == 0) p.cuts[blockIdx.x].parts = 0;
    int used = 0;   // tiles of this warp so far: of its ring
    PagedWalk<P4Kind> walk;
    const PagedBlock& k = walk.k;
    const PagedPlace& at = walk.place;
    walk.find(p, c, -1);
    for (; walk.w < walk.end; walk.go(p, c)) {
        int first, count;
        walk.share(first, count);
        if (count == 0) continue;
        const int pitch = int4_pitch<D>(tma), skip = int4_skip<D>(tma, at.hk);
        const int key0 = ((k.hi >= 0 ? k.lo / kP4Keys : 0) + first) * kP4Keys + warp * kP4Each;
        // The lanes ask for the page numbers of the rows a stage ahead; where pages hold whole 16s lanes 0 and 1 do
        auto find = [&](int j) {
            const int row = key0 + j * kP4Keys + (tma ? (lane & 1) * 16 : lane), pg = c.by_page(row);
            return j < count && row <= k.hi && pg < c.max_pages ? c.table[(size_t)k.seq * c.ld_table + pg] : -1;
        };
        auto copy = [&](int j, int id) {
            const int stage = (used + j) % kP4Stages, row0 = key0 + j * kP4Keys;
            if (tma) {
                if (lane == 0) mbar_expect_tx(&full[warp][stage], 2 * kP4Each * pitch);
                __syncwarp();
                if (lane < 2) {
                    const int row16 = row0 + lane * 16, row = row16 - c.by_page(row16) * c.page_size, page = id >= 0 && id < c.num_pages ? id : -1;   // -1: reads as zeros
                    const uint32_t to = ring_at + (uint32_t)(stage * C::kStage + lane * 16 * pitch);
                    int4_box<D>(to, &k_map, tma, at.hk, row, page, &full[warp][stage]);
                    int4_box<D>(to + C::kV, &v_map, tma, at.hk, row, page, &full[warp][stage]);
                }
            } else {
                const int mine = row0 + lane;
                const long long off = id >= 0 && id < c.num_pages
                                          ? (long long)id * c.page_stride + (long long)(mine - c.by_page(mine) * c.page_size) * c.row_stride + (long long)at.hk * c.head_stride : -1;
#pragma unroll 1
                for (int x = lane; x < 10 * kP4Each; x += 32) {
                    const int is_v = x >= 5 * kP4Each, r = (x - 5 * kP4Each * is_v) / 5, ch = (x - 5 * kP4Each * is_v) % 5;
                    const long long o = __shfl_sync(0xffffffffu, off, r);
                    p4_copy<C::kChunk>(ring_at + (uint32_t)(stage * C::kStage + is_v * C::kV + (x - 5 * kP4Each * is_v) * C::kChunk), static_cast<const uint8_t*>(is_v ? c.v : c.k) + (o < 0 ? 0 : o + ch * C::kChunk),
                                       o < 0 ? 0 : C::kChunk);
                }
            }
        };
        // rows of q: row g of each 8, as the columns of the second operand; what rows 2t and 2t + 1 see
        uint32_t qb[NT][KS][2];
        int hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + g;
            const bool in = r < k.rows;
            const int row = k.row0 + (in ? r : 0), t = p.by_group(row);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + ((size_t)(k.first + t) * p.heads + at.hk * p.group + row - t * p.group) * D) + t4 * (D / 8);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint2 x = make_uint2(0u, 0u);
                if (in) x = *reinterpret_cast<const uint2*>(src + 2 * s);
                qb[n][s][0] = x.x, qb[n][s][1] = x.y;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row_e = n * 8 + t4 * 2 + e;
                const bool is = row_e < k.rows;
                const int at_place = k.place0 + p.by_group(k.row0 + (is ? row_e : 0));
                hi[n][e] = is ? min(at_place, k.have - 1) : -1;
                lo[n][e] = paged_from(p, at_place);
            }
        }
        // keys that all rows of the block see; rows that are none may see them too
        const int all_hi = min(k.place0 + p.by_group(k.row0), k.have - 1), all_lo = paged_from(p, k.place0 + p.by_group(k.row0 + k.rows - 1));
        float o[MT][NT][4], l[NT][2], m_ref[NT][2];
        uint32_t track = 0;
        // The block's keys, one way or the other: -> whether there was a pair that the fast one does not serve.  A masked probability is exactly zero, but zero times NaN, which a
        // broken group of a row's values reads as, is NaN in its sum: of 16 keys with such a group SLOW takes the product key by key, of those that a row sees.
        auto pass = [&](auto slow) {
            constexpr bool SLOW = decltype(slow)::value;
            int id = find(0);
#pragma unroll 1
            for (int j = 0; j < kP4Stages - 1; ++j) {
                const int next = find(j + 1);
                if (j < count) copy(j, id);
                if (!tma) asm volatile("cp.async.commit_group;" ::: "memory");
                id = next;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int m = 0; m < MT; ++m) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
                l[n][0] = l[n][1] = 0.f, m_ref[n][0] = m_ref[n][1] = kPagedNone;
            }
#pragma unroll 1
            for (int j = 0; j < count; ++j) {
                const int stage = (used + j) % kP4Stages, kb = key0 + j * kP4Keys;
                uint8_t* st = ring + stage * C::kStage;
                if (tma) pt_wait(&full[warp][stage], (uint32_t)((used + j) / kP4Stages) & 1u, s_abort, err, 0x5c00 + warp);
                else asm volatile("cp.async.wait_group %0;" ::"n"(kP4Stages - 2) : "memory");
                __syncwarp();
                const int next = find(j + kP4Stages);
                if (j + kP4Stages - 1 < count) copy(j + kP4Stages - 1, id);
                if (!tma) asm volatile("cp.async.commit_group;" ::: "memory");
                id = next;
                if (kb > k.hi || kb + kP4Each - 1 < k.lo) continue;
                if (tma && kb + kP4Each - 1 > k.hi) {   // what a page holds behind the last key may be anything
                    if (kb + lane > k.hi)
#pragma unroll
                        for (int i = 0; i < D / kInt4Group; ++i) {
                            *reinterpret_cast<uint32_t*>(st + lane * pitch + skip + D / 2 + i * 4) = 0;
                            *reinterpret_cast<uint32_t*>(st + C::kV + lane * pitch + skip + D / 2 + i * 4) = 0;
                        }
                    pa_fence_async();
                    __syncwarp();
                }
                float s[2][NT][4] = {};   // keys kb + 16 h + {g, g + 8}, rows 8 n + 2t + {0, 1}
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t x[2][KW];
                    Int4Codes<T, SLOW> k_code[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint8_t* row = st + (16 * h + g + u * 8) * pitch + skip;
                        p4_words<KW>(x[u], row + t4 * C::kChunk);
                        const uint32_t pair = Int4Codes<T, SLOW>::pair(*reinterpret_cast<const uint32_t*>(row + D / 2 + t4 * (D / 4) / kInt4Group * 4), track);
                        k_code[u].set(__byte_perm(pair, 0, 0x1010), __byte_perm(pair, 0, 0x3232));
                    }
#pragma unroll
                    for (int w = 0; w < KW; ++w) {
                        const uint32_t a[4] = {k_code[0].template two<0>(x[0][w]), k_code[1].template two<0>(x[1][w]), k_code[0].template two<1>(x[0][w]), k_code[1].template two<1>(x[1][w])};
                        const uint32_t b[4] = {k_code[0].template two<2>(x[0][w]), k_code[1].template two<2>(x[1][w]), k_code[0].template two<3>(x[0][w]), k_code[1].template two<3>(x[1][w])};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            pf_mma<T>(s[h][n], a, qb[n][2 * w][0], qb[n][2 * w][1]);
                            pf_mma<T>(s[h][n], b, qb[n][2 * w + 1][0], qb[n][2 * w + 1][1]);
                        }
                    }
                }
                const float scale = p.scale * Int4Codes<T, SLOW>::kScale;
                const bool masks = kb + kP4Each - 1 > all_hi || kb < all_lo;
                bool up = false;
                float top[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float& x = s[i >> 1][n][(i & 1) * 2 + e];
                            x *= scale;
                            const int key = kb + g + 8 * i;
                            if (masks && (key > hi[n][e] || key < lo[n][e])) x = -INFINITY;
                        }
                        top[n][e] = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                        up |= top[n][e] - m_ref[n][e] > kTau;
                    }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], x));
                            const float f = top[n][e] > m_ref[n][e] ? pa_exp2(m_ref[n][e] - top[n][e]) : 1.f;
                            m_ref[n][e] = fmaxf(m_ref[n][e], top[n][e]);
                            l[n][e] *= f;
#pragma unroll
                            for (int m = 0; m < MT; ++m) o[m][n][e] *= f, o[m][n][2 + e] *= f;
                        }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t* values = st + C::kV + 16 * h * pitch + skip;
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {   // the difference first: it is as exact as the scores, whatever their size is
                            float &x = s[h][n][2 * u], &y = s[h][n][2 * u + 1];
                            x = pa_exp2((x - m_ref[n][0]) + kUp), y = pa_exp2((y - m_ref[n][1]) + kUp);
                            l[n][0] += x, l[n][1] += y;
                            pb[n][u] = p4_transpose(pf_pack<T>(x, y));
                        }
                    if constexpr (SLOW) {
                        bool whole = true;
                        for (int x = lane; x < D / 2; x += 32) whole = whole && int4_finite<T>(*reinterpret_cast<const uint32_t*>(values + x % 16 * pitch + D / 2 + x / 16 * 4));
                        if (__any_sync(0xffffffffu, !whole)) {   // the product key by key
#pragma unroll 1
                            for (int key = 0; key < 16; ++key) {
                                const uint8_t* row = values + key * pitch;
                                const uint32_t meta = *reinterpret_cast<const uint32_t*>(row + D / 2 + g * (D / 8) / kInt4Group * 4);
                                uint32_t x[VW];
                                p4_words<VW>(x, row + g * (D / 16));
                                const T* two = reinterpret_cast<const T*>(&meta);
                                float v[D / 8];
#pragma unroll
                                for (int i = 0; i < D / 8; ++i)
                                    v[i] = round_to<T>(fmaf((float)(x[i >> 3] >> ((i & 1) * 16 + (i & 6) * 2) & 15u), to_f32<T>(two[0]), to_f32<T>(two[1]))) / Int4Codes<T, SLOW>::kScale;
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const float w = __shfl_sync(0xffffffffu, key & 8 ? s[h][n][2 + e] : s[h][n][e], (key & 7) << 2 | t4);
                                        if (kb + 16 * h + key <= hi[n][e] && kb + 16 * h + key >= lo[n][e])
#pragma unroll
                                            for (int i = 0; i < D / 8; ++i) o[i >> 1][n][(i & 1) * 2 + e] = fmaf(w, v[i], o[i >> 1][n][(i & 1) * 2 + e]);
                                    }
                            }
                            continue;
                        }
                    }
                    uint32_t x[4][VW], pair[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {   // keys 2t + {0, 1, 8, 9}
                        const uint8_t* row = values + (2 * t4 + (u & 1) + (u >> 1) * 8) * pitch;
                        p4_words<VW>(x[u], row + g * (D / 16));
                        pair[u] = Int4Codes<T, SLOW>::pair(*reinterpret_cast<const uint32_t*>(row + D / 2 + g * (D / 8) / kInt4Group * 4), track);
                    }
                    Int4Codes<T, SLOW> v_code[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) v_code[u].set(__byte_perm(pair[2 * u], pair[2 * u + 1], 0x5410), __byte_perm(pair[2 * u], pair[2 * u + 1], 0x7632));
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        uint32_t even[2], odd[2];   // columns 0 2 4 6 and 1 3 5 7 of two keys
#pragma unroll
                        for (int u = 0; u < 2; ++u) even[u] = __byte_perm(x[2 * u][w], x[2 * u + 1][w], 0x5410), odd[u] = __byte_perm(x[2 * u][w], x[2 * u + 1][w], 0x7632);
                        auto product = [&](auto index) {
                            constexpr int J = decltype(index)::value;
                            const uint32_t a[4] = {v_code[0].template two<J>(even[0]), v_code[0].template two<J>(odd[0]), v_code[1].template two<J>(even[1]), v_code[1].template two<J>(odd[1])};
#pragma unroll
                            for (int n = 0; n < NT; ++n) pf_mma<T>(o[w * 4 + J][n], a, pb[n][0], pb[n][1]);
                        };
                        product(std::integral_constant<int, 0>{}), product(std::integral_constant<int, 1>{});
                        product(std::integral_constant<int, 2>{}), product(std::integral_constant<int, 3>{});
                    }
                }
            }
            used += count;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
        };
        pass(std::false_type{});
        bool again = false;
        if constexpr (kScaled) {
            again = !Int4Codes<T, false>::served(track);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    bool none = false;
#pragma unroll
                    for (int m = 0; m < MT; ++m) none |= o[m][n][e] != o[m][n][e] || o[m][n][2 + e] != o[m][n][2 + e];
                    again |= none && l[n][e] == l[n][e] && n * 8 + t4 * 2 + e < k.rows;
                }
        }
        if (__any_sync(0xffffffffu, again)) {
            __syncwarp();
            pass(std::true_type{});
        }
        // the warps' parts, in their rings
        if (!tma) asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = n * 8 + t4 * 2 + e;
                if (g == 0) s_ml[warp][r] = make_float2(m_ref[n][e], l[n][e] / Int4Codes<T, false>::kScale);
#pragma unroll
                for (int m = 0; m < MT; ++m) *reinterpret_cast<float2*>(mine + r * C::kPitch + g * (D / 8) + 2 * m) = make_float2(o[m][n][e], o[m][n][2 + e]);
            }
        __syncthreads();
        const bool whole = walk.whole(count);
        const size_t part = ((size_t)blockIdx.x * 2 + (first > 0 ? 0 : 1)) * R;
        for (int r = warp; r < k.rows; r += kP4Warps) {
            constexpr int E = D / 32;
            float m = s_ml[0][r].x, sum = 0.f, v[E] = {};
#pragma unroll
            for (int x = 1; x < kP4Warps; ++x) m = fmaxf(m, s_ml[x][r].x);
#pragma unroll
            for (int x = 0; x < kP4Warps; ++x) {
                const float f = pa_exp2(s_ml[x][r].x - m);
                sum = fmaf(s_ml[x][r].y, f, sum);
                const float* from = reinterpret_cast<const float*>(p4_smem + x * C::kWarp) + r * C::kPitch + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fmaf(from[e], f, v[e]);
            }
            if (whole) {
                paged_row_out<T, D>(p, k, at.hk, r, sum, v);
            } else {
                if (lane == 0) p.ml[part + r] = make_float2(m, sum);
                float* dst = p.part + (part + r) * D + lane * E;
                if constexpr (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                else *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[1]);
            }
        }
        if (tid == 0) walk.cut(p, first, count);
        pa_fence_async();   // TMA writes where the parts were
        __syncthreads();    // the rings are the next block's
    }
    tc2_drain(s_abort);
}

}  // namespace zl
