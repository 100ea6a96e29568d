// Attention of many new tokens over pages on the 5th-generation tensor cores.  A CTA owns up to 256 (token, head) rows of one kv head of one sequence,
// all heads of the group beside one another, as two tiles of 128, and walks the keys 128 at a time:
//
//   warps 0-3, 4-7  softmax of a tile each: thread = row = lane of tensor memory; running maximum and sum in 32 bits; probabilities go back over the scores
//   warp 8          one thread issues S = Q K^T and O += P V (P from tensor memory, V as it lies: rows of keys, the B operand along n) of both tiles
//   warps 10, 11    K and V tiles from the pages into a ring of buffers, 16 bytes a copy into the swizzled layout; rows that no row of the CTA sees
//                   and rows behind a page number outside the pool are zero-filled, so whatever lies there never meets a product
//
// Tensor memory: scores of the two tiles (128 columns each, probabilities over their first half), then their outputs.  Probabilities are rounded to the
// rows' type once (half a step each, of random sign: beside the output's own rounding), the sums that divide them are not.  A row's reference maximum
// follows the true one only once that has grown by 2^5 (fp16, whose probabilities carry 2^10) or 2^8: any reference gives the same quotient.
//
// A masked probability is exactly zero, but zero times an infinity or NaN that a row must not see (a later token's value) is NaN in its sum.  A row that
// comes out as NaN is therefore done once more from the definition, key by key (paged_row_exact); numbers never take that path.
#pragma once
#include "attn_ptx.cuh"
#include "paged_attn.cuh"

#include <type_traits>

namespace zl {

constexpr int kPtRows = 256, kPtKeys = 128, kPtThreads = 384, kPtWarpMma = 8, kPtWarpLoad = 10, kPtLoaders = 64;

template <int D>
struct PtCfg {
    static constexpr int kAtoms = D / 64;
    static constexpr int kQ = kAtoms * kPaRows * 128;       // a tile of Q: [64 of d][128 rows][128 B]
    static constexpr int kTile = kAtoms * kPtKeys * 128;    // K or V: [64 of d][128 keys][128 B]
    static constexpr int kRing = D == 128 ? 5 : 8;
    static constexpr int kRingOff = 2 * kQ, kOffs = kRingOff + kRing * kTile;
    static constexpr int kBytes = kOffs + kPtKeys * 8 + 1024;   // + slack for the manual 1024-byte alignment
    static_assert(tmem_alone(kBytes) && kBytes + 1024 <= 227 * 1024, "all of tensor memory, an SM to itself");
    static constexpr int kO = 256;                          // TMEM columns: scores 0, 128; outputs from here
};

// grid (row blocks * splits, kv heads)
template <typename T, int D>
__global__ void __launch_bounds__(kPtThreads, 1) k_paged_attn_tiles(const PagedAttn p, const PagedCache c, unsigned* err) {
    using C = PtCfg<D>;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int CH = D / 8;
    extern __shared__ uint8_t pt_smem[];
    uint8_t* smem = pt_smem + ((1024u - (smem_u32(pt_smem) & 1023u)) & 1023u);
    __shared__ uint64_t full[C::kRing], empty[C::kRing], s_full[2], p_full[2], o_done[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    volatile int* s_abort = &s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hk = blockIdx.y;
    if (tid == 0) {
        for (int i = 0; i < C::kRing; ++i) mbar_init(&full[i], kPtLoaders), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&o_done[i], 1);
        s_gave_up = 0;
        mbar_fence_init();
    }
    if (warp == kPtWarpMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    pdl_wait();
    const uint32_t tmem = s_tmem;
    const int item = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    PagedBlock k = {};
    const bool any = paged_block(p, c, item, kPtRows, k);
    if (any) {
        const int tiles_m = k.rows > kPaRows ? 2 : 1;
        const int have = k.hi >= 0 ? k.hi / kPtKeys + 1 - k.lo / kPtKeys : 0, per = cdiv(have, p.splits);
        const int t0 = k.lo / kPtKeys + min(have, split * per), count = min(have, (split + 1) * per) - min(have, split * per);
        if (warp < kPtWarpMma) {
            // rows of q, [64 of d][row][128 B] with the chunks xor the row; rows behind the last one are zeros
            const int ch = tid % CH;
#pragma unroll
            for (int i = 0; i < kPtRows * CH / 256; ++i) {
                const int r = tid / CH + i * (256 / CH), rr = r & (kPaRows - 1);
                const bool in = r < k.rows;
                const int row = k.row0 + (in ? r : 0), t = row / p.group;
                const T* src = static_cast<const T*>(p.q) + ((size_t)(k.first + t) * p.heads + hk * p.group + row - t * p.group) * D + ch * 8;
                pa_cp16(smem_u32(smem) + (uint32_t)((r >> 7) * C::kQ + (ch >> 3) * (kPaRows * 128) + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)), src, in);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            pa_fence_async();
            asm volatile("bar.sync 1, 288;" ::: "memory");
        }
        if (warp == kPtWarpMma) {
            asm volatile("bar.sync 1, 288;" ::: "memory");
            if (tc_elect_one()) {
                const uint32_t id_s = pa_idesc(!kHalf, kPtKeys, false), id_o = pa_idesc(!kHalf, D, true);
                bool ok = true;
                auto scores = [&](int m, int j) {
                    const int it = 2 * j, slot = it % C::kRing;
                    ok = ok && tc2_wait1(&full[slot], (uint32_t)(it / C::kRing) & 1u, s_abort, err, 0x5100 + slot);
                    if (!ok) return;
                    pa_fence_async();
                    tc_fence_after();
                    const uint64_t qd = tc_desc_sw128(smem_u32(smem + m * C::kQ)), kd = tc_desc_sw128(smem_u32(smem + C::kRingOff + slot * C::kTile));
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        pa_mma_ss(tmem + (uint32_t)(m * 128), qd + (uint64_t)((i >> 2) * (kPaRows * 128 / 16) + (i & 3) * 2),
                                  kd + (uint64_t)((i >> 2) * (kPtKeys * 128 / 16) + (i & 3) * 2), id_s, i > 0 ? 1u : 0u);
                    tc_commit(&s_full[m]);
                    if (m == tiles_m - 1) tc_commit(&empty[slot]);
                };
                auto values = [&](int m, int j) {
                    const int it = 2 * j + 1, slot = it % C::kRing;
                    ok = ok && tc2_wait1(&full[slot], (uint32_t)(it / C::kRing) & 1u, s_abort, err, 0x5200 + slot);
                    ok = ok && tc2_wait1(&p_full[m], (uint32_t)j & 1u, s_abort, err, 0x5300 + m);
                    if (!ok) return;
                    pa_fence_async();
                    tc_fence_after();
                    const uint64_t vd = pa_desc_mn(smem_u32(smem + C::kRingOff + slot * C::kTile), kPtKeys * 128);
#pragma unroll
                    for (int i = 0; i < kPtKeys / 16; ++i)
                        pa_mma_ts(tmem + (uint32_t)(C::kO + m * D), tmem + (uint32_t)(m * 128 + i * 8), vd + (uint64_t)(i * (16 * 128 / 16)), id_o,
                                  (j > 0 || i > 0) ? 1u : 0u);
                    tc_commit(&o_done[m]);
                    if (m == tiles_m - 1) tc_commit(&empty[slot]);
                };
                if (count > 0)
                    for (int m = 0; m < tiles_m; ++m) scores(m, 0);
                for (int j = 0; j < count && ok; ++j)
                    for (int m = 0; m < tiles_m && ok; ++m) {
                        values(m, j);
                        if (j + 1 < count) {   // over the probabilities that P V has read
                            ok = ok && tc2_wait1(&o_done[m], (uint32_t)j & 1u, s_abort, err, 0x5400 + m);
                            scores(m, j + 1);
                        }
                    }
            }
            __syncwarp();
        } else if (warp >= kPtWarpLoad) {
            const int t = tid - kPtWarpLoad * 32, ch = t % CH;
            long long* offs = reinterpret_cast<long long*>(smem + C::kOffs);
            const long long head = (long long)hk * c.head_stride + ch * 8;
            const T *kp = static_cast<const T*>(c.k) + head, *vp = static_cast<const T*>(c.v) + head;
            const uint32_t at = smem_u32(smem) + (uint32_t)(C::kRingOff + (ch >> 3) * (kPtKeys * 128));
            bool ok = true;   // after a wait that gave up the loop goes on without copies: its barriers want both warps
            for (int j = 0; j < count; ++j) {
#pragma unroll
                for (int u = 0; u < kPtKeys; u += kPtLoaders) {
                    const int row = (t0 + j) * kPtKeys + t + u;
                    offs[t + u] = row <= k.hi ? c.row_at(k.seq, row) : -1;
                }
                asm volatile("bar.sync 2, %0;" ::"n"(kPtLoaders) : "memory");
#pragma unroll 1
                for (int is_v = 0; is_v < 2; ++is_v) {
                    const int it = 2 * j + is_v, slot = it % C::kRing;
                    if (it >= C::kRing) ok = ok && tc2_wait(&empty[slot], (uint32_t)(it / C::kRing - 1) & 1u, s_abort, err, 0x5500 + slot);
                    if (!ok) break;
                    const T* from = is_v ? vp : kp;
                    const uint32_t to = at + (uint32_t)(slot * C::kTile);
#pragma unroll 8
                    for (int i = 0; i < kPtKeys * CH / kPtLoaders; ++i) {
                        const int r = t / CH + i * (kPtLoaders / CH);
                        const long long off = offs[r];
                        pa_cp16(to + (uint32_t)(r * 128 + (((ch & 7) ^ (r & 7)) << 4)), from + (off < 0 ? 0 : off), off >= 0);
                    }
                    pa_landed(&full[slot]);
                }
                asm volatile("bar.sync 2, %0;" ::"n"(kPtLoaders) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (warp < kPtWarpMma) {
            const int m = warp >> 2, r = tid;   // of the CTA's rows
            if (m < tiles_m) {
                const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = taddr + (uint32_t)(m * 128), to = taddr + (uint32_t)(C::kO + m * D);
                constexpr float kTau = kHalf ? 5.f : 8.f, kUp = kHalf ? 10.f : 0.f;
                const float cs = p.scale;
                const int row = k.row0 + r, t = row / p.group, place = k.place0 + t;
                const int hi = r < k.rows ? min(place, k.have - 1) : -1, lo = r < k.rows && p.window ? max(0, place - p.window + 1) : 0;
                float l = 0.f, m_ref = -1.4426950e20f;
                for (int j = 0; j < count; ++j) {
                    const int h = hi - (t0 + j) * kPtKeys, w = lo - (t0 + j) * kPtKeys;   // this row sees w .. h of the tile
                    if (!tc2_wait(&s_full[m], (uint32_t)j & 1u, s_abort, err, 0x5600 + m)) break;
                    tc_fence_after();
                    uint32_t raw[kPtKeys];
#pragma unroll
                    for (int i = 0; i < kPtKeys; i += 32) pa_ld32(ts + i, raw + i);
                    pa_wait_ld();
                    if (!__all_sync(0xffffffffu, h >= kPtKeys - 1 && w <= 0)) {
                        const unsigned span = h >= w ? (unsigned)(h - w) : 0u, from = h >= w ? (unsigned)w : 0x40000000u;
#pragma unroll
                        for (int i = 0; i < kPtKeys; ++i)
                            if ((unsigned)i - from > span) raw[i] = 0xff800000u;
                    }
                    float mx[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(raw[i]);
#pragma unroll
                    for (int i = 4; i < kPtKeys - 4; i += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u) mx[u] = pa_max3(mx[u], __uint_as_float(raw[i + 2 * u]), __uint_as_float(raw[i + 2 * u + 1]));
                    mx[0] = pa_max3(mx[0], __uint_as_float(raw[kPtKeys - 4]), __uint_as_float(raw[kPtKeys - 3]));
                    mx[1] = pa_max3(mx[1], __uint_as_float(raw[kPtKeys - 2]), __uint_as_float(raw[kPtKeys - 1]));
                    const float m_tile = pa_max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * cs;
                    const bool up = m_tile > m_ref + kTau;
                    if (__any_sync(0xffffffffu, up)) {
                        const float f = up ? pa_exp2(m_ref - m_tile) : 1.f;
                        if (up) m_ref = m_tile;
                        l *= f;
                        if (j > 0) {   // P V of the tile before has ended: these scores were issued behind it
#pragma unroll 1
                            for (int d0 = 0; d0 < D; d0 += 16) {
                                float v[16];
                                uint32_t x[16];
                                tc_ld16(to + (uint32_t)d0, v);
#pragma unroll
                                for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(v[i] * f);
                                tc_st16(to + (uint32_t)d0, x);
                            }
                        }
                    }
                    const uint64_t c2 = pa_two(cs, cs), m2 = pa_two(kUp - m_ref, kUp - m_ref);
                    uint64_t sum[2] = {0, 0};
#pragma unroll
                    for (int part = 0; part < kPtKeys; part += 32) {
                        uint32_t x[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float a, b;
                            pa_split(pa_fma2(pa_two(__uint_as_float(raw[part + 2 * i]), __uint_as_float(raw[part + 2 * i + 1])), c2, m2), a, b);
                            a = pa_exp2(a);
                            b = pa_exp2(b);
                            sum[i & 1] = pa_add2(sum[i & 1], pa_two(a, b));
                            if constexpr (kHalf) {
                                const __half2 y = __floats2half2_rn(a, b);
                                x[i] = *reinterpret_cast<const uint32_t*>(&y);
                            } else {
                                const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
                                x[i] = *reinterpret_cast<const uint32_t*>(&y);
                            }
                        }
                        tc_st16(ts + (uint32_t)(part / 2), x);
                    }
                    float s0, s1;
                    pa_split(pa_add2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[m]);
                }
                if (count > 0) tc2_wait(&o_done[m], (uint32_t)(count - 1) & 1u, s_abort, err, 0x5700 + m);
                tc_fence_after();
                if (p.splits == 1) {
                    const int head = hk * p.group + row - t * p.group;
                    T* dst = static_cast<T*>(p.out) + ((size_t)(k.first + t) * p.heads + head) * D;
                    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                    bool broken = false;
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += 16) {
                        float v[16];
                        tc_ld16(to + (uint32_t)d0, v);
                        if (r < k.rows) {
                            float f[2][8];
#pragma unroll
                            for (int i = 0; i < 16; ++i) f[i >> 3][i & 7] = count > 0 ? v[i] * inv : 0.f, broken |= f[i >> 3][i & 7] != f[i >> 3][i & 7];
                            *reinterpret_cast<uint4*>(dst + d0) = pack8<T>(f[0]);
                            *reinterpret_cast<uint4*>(dst + d0 + 8) = pack8<T>(f[1]);
                        }
                    }
                    for (unsigned left = __ballot_sync(0xffffffffu, broken); left; left &= left - 1) {
                        const int src = __ffs(left) - 1;
                        paged_row_exact<T, D>(p, c, k.seq, __shfl_sync(0xffffffffu, k.first + t, src), __shfl_sync(0xffffffffu, head, src),
                                              __shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, hi, src));
                    }
                } else {
                    // the part of these keys: {maximum, sum}, then the output as it stands
                    const size_t part = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * kPtRows + r;
                    if (r < k.rows) p.ml[part] = make_float2(count > 0 ? m_ref : -INFINITY, count > 0 ? l : 0.f);
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += 16) {
                        float v[16];
                        if (count > 0) tc_ld16(to + (uint32_t)d0, v);
                        if (r < k.rows && count > 0)
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(p.part + part * D + d0 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                }
            }
        }
    }
    __syncwarp();
    tc2_drain(s_abort);
    tc_fence_before();
    __syncthreads();
    if (warp == kPtWarpMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
    }
}

// Joins the parts of the key ranges: grid (row blocks, kv heads), a warp for every eighth row
template <typename T, int D>
__global__ void __launch_bounds__(256) k_paged_attn_join(const PagedAttn p, const PagedCache c) {
    constexpr int E = D / 32;
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y;
    PagedBlock k = {};
    if (!paged_block(p, c, blockIdx.x, kPtRows, k)) return;
    for (int r = warp; r < k.rows; r += 8) {
        const int row = k.row0 + r, t = row / p.group, head = hk * p.group + row - t * p.group, place = k.place0 + t;
        const size_t at = ((size_t)hk * gridDim.x + blockIdx.x) * p.splits * kPtRows + r;
        float m = -INFINITY, l = 0.f, o[E] = {};
        for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.ml[at + (size_t)s * kPtRows].x);
        for (int s = 0; s < p.splits; ++s) {
            const float2 x = p.ml[at + (size_t)s * kPtRows];
            if (x.x == -INFINITY) continue;   // no keys in this range: nothing was written
            const float f = pa_exp2(x.x - m);
            l = fmaf(x.y, f, l);
            const float* from = p.part + (at + (size_t)s * kPtRows) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(from[e], f, o[e]);
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        T two[E];
        bool broken = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = l == 0.f ? 0.f : o[e] * inv;
            broken |= v != v;
            two[e] = from_f32<T>(v);
        }
        T* dst = static_cast<T*>(p.out) + ((size_t)(k.first + t) * p.heads + head) * D + lane * E;
        if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(two);
        else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<uint32_t*>(two);
        if (__any_sync(0xffffffffu, broken))
            paged_row_exact<T, D>(p, c, k.seq, k.first + t, head, p.window ? max(0, place - p.window + 1) : 0, min(place, k.have - 1));
    }
}

}  // namespace zl
