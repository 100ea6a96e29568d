// Attention of few (token, head) rows of a kv head -- single tokens, drafts of small groups -- over pages: bound by the bytes of K and V, which the CTAs
// of the grid share out evenly, whatever the sequences' lengths are.  All tiles of 64 keys of all blocks (up to 16 rows of one kv head of one sequence)
// stand in one line; a CTA takes an equal stretch of it.  A block that lies in one stretch is written at once, the parts of one that is cut go to the
// workspace, its first part to the CTA's place 1, others to its place 0, and k_paged_join puts them together.
//
// A warp has 16 keys of a tile to itself, in a ring of its own (16-byte cp.async; no barrier between the warps until a block's end):
// S = Q K^T and O += P V by mma.sync with Q as the 16-row operand, whose accumulators are the next product's operand as they stand.  The probabilities are
// carried as a 16-bit value and the rest of it as another, their sum in 32 bits; the reference maximum of a row follows lazily as in paged_attn_tc.cuh.
//
// One token over 131072 keys, 32 heads on 8: 99 us a call in a graph, 103 to 105 in a row of eager ones (537 MB: 5.1 TB/s or more of the 6.45 that a copy reaches), 96 of
// them in this kernel under ncu; errors of 1.7e-3 against 64 bits, 2.3e-3 with probabilities of 16 bits alone, which takes 2 to 3 us off.  28 of 32 sequences with up to 4096 keys:
// 41 us for 174 MB, bound by the first loads of every block, whose setup stands in the line as two tiles.  Two CTAs share an SM (167 or 238 registers), one's
// first loads and joins come under the other's stream.  Taken when these calls took 101 and 49 us: 64 where the setup did not count; Q by way of shared memory, for fewer
// registers, 108 and 57; one warp that finds the way for all 53.
#pragma once
#include "attn_ptx.cuh"
#include "paged_attn.cuh"

#include <type_traits>

namespace zl {

constexpr int kPfWarps = 4, kPfKeys = 16 * kPfWarps, kPfStages = 3, kPfPerSm = 2, kPfRows = 16;

template <int D>
struct PfCfg {
    static constexpr int kStage = 16 * D * 2 * 2;                    // 16 rows of K, then of V
    static constexpr int kWarp = kPfStages * kStage;
    static constexpr int kBytes = kPfWarps * kWarp;
    static constexpr int kPitch = D + 8;                             // floats; of a row of a warp's output in its ring
};

// tiles of 64 keys; at least one: a block that sees nothing is written too
struct PfKind {
    static constexpr int kSetup = 2;
    static __device__ __forceinline__ int turns(const PagedAttn&, const PagedBlock& k) { return k.hi >= 0 ? k.hi / kPfKeys - k.lo / kPfKeys + 1 : 1; }
};

__device__ __forceinline__ void pf_ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pf_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void pf_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) mma_16816_f16(d, a, b0, b1, d);
    else mma_16816_bf16(d, a, b0, b1, d);
}
template <typename T>
__device__ __forceinline__ uint32_t pf_pack(float a, float b) {
    T two[2] = {from_f32<T>(a), from_f32<T>(b)};
    return *reinterpret_cast<const uint32_t*>(two);
}

// grid: CTAs that share the line
template <typename T, int D>
__global__ void __launch_bounds__(kPfWarps * 32, kPfPerSm) k_paged_attn_few(const PagedAttn p, const PagedCache c) {
    using C = PfCfg<D>;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int R = kPfRows, CH = D / 8, KS = D / 16;
    constexpr float kTau = PagedExp<kHalf>::kTau, kUp = PagedExp<kHalf>::kUp;
    extern __shared__ __align__(128) uint8_t pf_smem[];
    __shared__ float2 s_ml[kPfWarps][R];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    uint8_t* ring = pf_smem + warp * C::kWarp;
    const uint32_t ring_at = smem_u32(ring);
    pdl_wait();
    pdl_trigger();
    if (tid == 0) p.cuts[blockIdx.x].parts = 0;
    PagedWalk<PfKind> walk;
    const PagedBlock& k = walk.k;
    const PagedPlace& at = walk.place;
    walk.find(p, c, -1);
    for (; walk.w < walk.end; walk.go(p, c)) {
        int first, count;
        walk.share(first, count);
        if (count == 0) continue;
        const int key0 = ((k.hi >= 0 ? k.lo / kPfKeys : 0) + first) * kPfKeys + warp * 16;
        const long long head = (long long)at.hk * c.head_stride;
        // Copies of a stage: each lane has a chunk of some rows.  Lanes 0 - 15 ask for the page numbers of the 16 rows a stage ahead; where pages hold whole
        // 16s these are one page.
        const bool one_page = c.page_size % 16 == 0;
        auto find = [&](int j) {
            const int row = key0 + j * kPfKeys + (lane & 15), pg = c.by_page(row);
            return j < count && row <= k.hi && pg < c.max_pages ? c.table[(size_t)k.seq * c.ld_table + pg] : -1;
        };
        auto copy = [&](int j, int id) {
            const uint32_t to = ring_at + (uint32_t)(j % kPfStages) * C::kStage;
            const int ch = lane % CH, row0 = key0 + j * kPfKeys, mine = row0 + (one_page ? 0 : lane & 15);
            long long off = id >= 0 && id < c.num_pages ? (long long)id * c.page_stride + (long long)(mine - c.by_page(mine) * c.page_size) * c.row_stride : -1;
            if (one_page) off = __shfl_sync(0xffffffffu, off, 0);
#pragma unroll
            for (int i = 0; i < 16 * CH / 32; ++i) {
                const int r = lane / CH + i * (32 / CH);
                long long o = off;
                if (!one_page) o = __shfl_sync(0xffffffffu, off, r);
                else if (row0 + r > k.hi) o = -1;
                else if (o >= 0) o += r * c.row_stride;
                const long long from = o < 0 ? 0 : o + head + ch * 8;
                const int bytes = o < 0 ? 0 : 16;
                const uint32_t dst = to + (uint32_t)(r * (D * 2) + ((ch ^ (r & 7)) << 4));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(static_cast<const T*>(c.k) + from), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 16 * D * 2), "l"(static_cast<const T*>(c.v) + from), "r"(bytes) : "memory");
            }
        };
        // rows of q: (g, g + 8) of each 16
        uint32_t qa[KS][4];
        int hi[2], lo[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = g + u * 8;
            const bool in = r < k.rows;
            const int row = k.row0 + (in ? r : 0), t = p.by_group(row), place = k.place0 + t;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + ((size_t)(k.first + t) * p.heads + at.hk * p.group + row - t * p.group) * D);
            hi[u] = in ? min(place, k.have - 1) : -1;
            lo[u] = paged_from(p, place);
#pragma unroll
            for (int s = 0; s < KS; ++s) qa[s][u] = in ? src[s * 8 + t4] : 0u, qa[s][2 + u] = in ? src[s * 8 + 4 + t4] : 0u;
        }
        float o[D / 8][4], l[2], m_ref[2];
        // Once, mostly.  A masked probability is exactly zero, but zero times an infinity or NaN that a row must not see is NaN in its sum (and the rest of a
        // probability times an infinity may be one too).  Where the warp's sums hold a NaN that no score explains, it goes over its keys once more and looks at the
        // values: of 16 keys that are not all numbers it takes the product key by key, of those that a row sees.
        for (bool again = false;; again = true) {
            int id = find(0);
#pragma unroll 1
            for (int j = 0; j < kPfStages - 1; ++j) {
                const int next = find(j + 1);
                if (j < count) copy(j, id);
                asm volatile("cp.async.commit_group;" ::: "memory");
                id = next;
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
            l[0] = l[1] = 0.f, m_ref[0] = m_ref[1] = kPagedNone;
            for (int j = 0; j < count; ++j) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kPfStages - 2) : "memory");
                __syncwarp();
                const int next = find(j + kPfStages);
                if (j + kPfStages - 1 < count) copy(j + kPfStages - 1, id);
                asm volatile("cp.async.commit_group;" ::: "memory");
                id = next;
                const int kb = key0 + j * kPfKeys;
                if (kb > k.hi || kb + 15 < k.lo) continue;
                const uint32_t st = ring_at + (uint32_t)(j % kPfStages) * C::kStage;
                float s[2][4] = {};
                {
                    // matrices of 8 keys x 8 columns: (keys 0-7, first 8), (0-7, next 8), (8-15, first 8), (8-15, next 8)
                    const int r = (lane & 7) + ((lane >> 4) << 3), ch0 = (lane >> 3) & 1;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        uint32_t b[4];
                        pf_ldsm(b, st + (uint32_t)(r * (D * 2) + (((2 * i + ch0) ^ (r & 7)) << 4)));
                        pf_mma<T>(s[0], qa[i], b[0], b[1]), pf_mma<T>(s[1], qa[i], b[2], b[3]);
                    }
                }
                uint32_t pa[4], pb[4];   // probabilities, and what their rounding left of them
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = kb + n * 8 + t4 * 2 + (e & 1);
                        s[n][e] = key <= hi[e >> 1] && key >= lo[e >> 1] ? s[n][e] * p.scale : -INFINITY;
                    }
                bool up = false;
                float top[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    top[u] = fmaxf(fmaxf(s[0][2 * u], s[0][2 * u + 1]), fmaxf(s[1][2 * u], s[1][2 * u + 1]));
                    up |= top[u] - m_ref[u] > kTau;
                }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 1));
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 2));
                        const float f = top[u] > m_ref[u] ? pa_exp2(m_ref[u] - top[u]) : 1.f;
                        m_ref[u] = fmaxf(m_ref[u], top[u]);
                        l[u] *= f;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) o[n][2 * u] *= f, o[n][2 * u + 1] *= f;
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {   // the difference first: it is as exact as the scores, whatever their size is
                        const float x = pa_exp2((s[n][2 * u] - m_ref[u]) + kUp), y = pa_exp2((s[n][2 * u + 1] - m_ref[u]) + kUp);
                        l[u] += x + y;
                        s[n][2 * u] = x, s[n][2 * u + 1] = y;
                        pa[2 * n + u] = pf_pack<T>(x, y);
                        const T* two = reinterpret_cast<const T*>(&pa[2 * n + u]);
                        pb[2 * n + u] = pf_pack<T>(x - to_f32<T>(two[0]), y - to_f32<T>(two[1]));
                    }
                bool apart = false;   // the product key by key
                if (again) {
                    const uint4* v = reinterpret_cast<const uint4*>(ring + (j % kPfStages) * C::kStage + 16 * D * 2);
                    uint32_t top = 0;
                    for (int x = lane; x < 16 * CH; x += 32) {
                        const uint4 w = v[x];
                        top = __vmaxu2(__vmaxu2(top, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
                    }
                    constexpr uint32_t kInf = kHalf ? 0x7c00 : 0x7f80;
                    apart = __any_sync(0xffffffffu, (top & 0xffffu) >= kInf || top >> 16 >= kInf);
                }
                if (apart) {
#pragma unroll 1
                    for (int key = 0; key < 16; ++key) {
                        const T* v = reinterpret_cast<const T*>(ring + (j % kPfStages) * C::kStage + 16 * D * 2 + key * (D * 2));
                        float w[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            w[u] = __shfl_sync(0xffffffffu, key & 1 ? (key & 8 ? s[1][2 * u + 1] : s[0][2 * u + 1]) : (key & 8 ? s[1][2 * u] : s[0][2 * u]),
                                               (lane & ~3) | (key >> 1 & 3));
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (kb + key <= hi[u] && kb + key >= lo[u])
#pragma unroll
                                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) o[n][2 * u + e] = fmaf(w[u], to_f32<T>(v[((n ^ (key & 7)) << 3) + t4 * 2 + e]), o[n][2 * u + e]);
                    }
                } else {
                    // transposed: (keys 0-7, first 8 columns), (keys 8-15, first 8), (0-7, next 8), (8-15, next 8)
                    const int r = (lane & 7) + (((lane >> 3) & 1) << 3), ch0 = lane >> 4;
#pragma unroll
                    for (int n = 0; n < D / 8; n += 2) {
                        uint32_t b[4];
                        pf_ldsm_t(b, st + (uint32_t)(16 * D * 2 + r * (D * 2) + (((n + ch0) ^ (r & 7)) << 4)));
                        pf_mma<T>(o[n], pa, b[0], b[1]), pf_mma<T>(o[n + 1], pa, b[2], b[3]);
                        pf_mma<T>(o[n], pb, b[0], b[1]), pf_mma<T>(o[n + 1], pb, b[2], b[3]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            }
            if (again) break;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                bool none = false;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) none |= o[n][2 * u] != o[n][2 * u] || o[n][2 * u + 1] != o[n][2 * u + 1];
                again |= none && l[u] == l[u] && g + u * 8 < k.rows;
            }
            if (!__any_sync(0xffffffffu, again)) break;
            __syncwarp();
        }
        // the warps' parts, in their rings
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = g + u * 8;
            if (t4 == 0) s_ml[warp][r] = make_float2(m_ref[u], l[u]);
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(mine + r * C::kPitch + n * 8 + t4 * 2) = make_float2(o[n][2 * u], o[n][2 * u + 1]);
        }
        __syncthreads();
        const bool whole = walk.whole(count);
        const size_t part = ((size_t)blockIdx.x * 2 + (first > 0 ? 0 : 1)) * R;
        for (int r = warp; r < k.rows; r += kPfWarps) {
            constexpr int E = D / 32;
            float m = s_ml[0][r].x, sum = 0.f, v[E] = {};
#pragma unroll
            for (int x = 1; x < kPfWarps; ++x) m = fmaxf(m, s_ml[x][r].x);
#pragma unroll
            for (int x = 0; x < kPfWarps; ++x) {
                const float f = pa_exp2(s_ml[x][r].x - m);
                sum = fmaf(s_ml[x][r].y, f, sum);
                const float* from = reinterpret_cast<const float*>(pf_smem + x * C::kWarp) + r * C::kPitch + lane * E;
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
        __syncthreads();   // the rings are the next block's
    }
}

}  // namespace zl
