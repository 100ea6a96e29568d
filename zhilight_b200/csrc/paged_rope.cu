// Rotation of fused query / key / value rows by positions on several axes, and their append to a paged cache: the counterpart of zl_qkv_rope_append
// for pictures and video, whose tokens have a place in time, height and width, each turning frequencies of its own.
//
//   angle[t][i] = pos[axis[i]][t] * inv_freq[i];   (a, b) -> (a cos - b sin, b cos + a sin) * mscale for the pair i of every query and key head
//
// A CTA serves tokens in turn.  Bulk copies bring their rows into a ring in shared memory, one ahead; the threads turn queries and keys there, in
// place, and bulk copies take them on to q and to the pages (values go by untouched).  One thread for each frequency works out the next token's cosine and
// sine meanwhile.  Angle and reduction are in 64 bits (at position 4e6 a 32-bit angle is off by 0.25 rad): the angle in turns, less the nearest whole
// number, is exact to 1e-9 of a turn, and what is left of it goes through CUDA's 32-bit functions (within 2e-7).  Products and sums are in 32 bits,
// rounded once.  Bound by bytes, a row is read once and written once: 4525 rows of 32 + 2 * 8 heads of 128 (111 MB) 21.5 to 23 us by the GPU it ran on, 4.8 to 5.2 TB/s,
// where an elementwise product of as many bytes takes 19.5; through registers, a row ahead, 25 to 31.  A third row ahead gives nothing (22.5).
#include "attn_ptx.cuh"
#include "paged.cuh"

#include <type_traits>

namespace zl {

enum { kRopePairs, kRopeAdjacent, kRopeAny };   // halves of whole 16 bytes, a piece of the first with its partner of the second; adjacent; other halves
constexpr int kRopeMaxStages = 4;

// two neighbouring elements as two 32-bit numbers, and back
template <typename T>
__device__ __forceinline__ uint64_t rope_unpack(uint32_t x) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
        return pa_two(f.x, f.y);
    } else {
        return pa_two(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
}
template <typename T>
__device__ __forceinline__ uint32_t rope_pack(uint64_t v) {
    float a, b;
    pa_split(v, a, b);
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 y = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&y);
    } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&y);
    }
}
__device__ __forceinline__ void rope_turn(uint64_t& f, uint64_t& g, uint64_t c, uint64_t s) {
    uint64_t fs, gs;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(fs) : "l"(f), "l"(s));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(gs) : "l"(g), "l"(s));
    f = pa_fma2(f, c, gs ^ 0x8000000080000000ull);
    g = pa_fma2(g, c, fs);
}

struct AxesRope {
    const void* qkv;
    void* q;
    const int32_t *pos, *axis, *token_seq, *placement;
    const double* inv_freq;
    long long ldq, ld_pos;
    int axes, half, heads, kv_heads, dim;
    float mscale;
    int rows, stages, row_bytes;
};

__device__ __forceinline__ void rope_s2g(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}

// grid: CTAs that share the tokens; dynamic shared memory: `stages` rows, then cosines and sines of two tokens
template <typename T, int FORM>
__global__ void __launch_bounds__(256, 4) k_axes_rope_append(const AxesRope p, const PagedCache c, unsigned* err) {
    extern __shared__ __align__(128) uint8_t rope_smem[];
    __shared__ uint64_t full[kRopeMaxStages];
    __shared__ int s_gave_up;
    volatile int* s_abort = &s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = blockDim.x, step = (int)gridDim.x;
    // As (cos, cos, sin, sin) of two frequencies.  A piece of 16 bytes takes `per` of them: its pair k stands at [k][piece], so that neighbouring lanes read
    // neighbouring 16 bytes.
    constexpr int per = FORM == kRopePairs ? 8 : FORM == kRopeAdjacent ? 4 : 2;
    const int pieces = (p.half + per - 1) / per, room = 2 * pieces * per;
    float* turns = reinterpret_cast<float*>(rope_smem + p.stages * p.row_bytes);
    auto slot = [&](int i) { return (i % per / 2 * pieces + i / per) * 4 + (i & 1); };
    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
        s_gave_up = 0;
        mbar_fence_init();
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    auto fetch = [&](int i) {   // the CTA's token i, by one thread
        const int t = (int)blockIdx.x + i * step, s = i % p.stages;
        if (t >= p.rows) return;
        mbar_expect_tx(&full[s], (uint32_t)p.row_bytes);
        bulk_g2s(rope_smem + s * p.row_bytes, static_cast<const T*>(p.qkv) + (size_t)t * p.ldq, (uint32_t)p.row_bytes, &full[s]);
    };
    if (tid == 0)
        for (int i = 0; i < p.stages; ++i) fetch(i);
    // this thread's first frequency; further ones are looked up again
    const int ax = tid < p.half ? p.axis[tid] : -1, my_slot = slot(tid);
    const double freq = tid < p.half ? p.inv_freq[tid] * 0.15915494309189533577 : 0.0;
    auto pos_of = [&](int axis, int t) { return (unsigned)axis < (unsigned)p.axes && t < p.rows ? p.pos[(size_t)axis * p.ld_pos + t] : 0; };
    auto angle = [&](float* to, int pos, double f) {
        const double x = (double)pos * f;
        float sn, cs;
        sincospif(2.0f * (float)(x - rint(x)), &sn, &cs);
        to[0] = cs * p.mscale, to[2] = sn * p.mscale;
    };
    auto angles = [&](float* turn, int t, int pos) {
        if (tid < p.half) angle(turn + my_slot, pos, freq);
        if (t < p.rows)
            for (int i = tid + threads; i < p.half; i += threads) angle(turn + slot(i), pos_of(p.axis[i], t), p.inv_freq[i] * 0.15915494309189533577);
    };
    int t = blockIdx.x, pos = pos_of(ax, t + step), seq = p.token_seq[t], pl = p.placement[t];
    angles(turns, t, pos_of(ax, t));
    __syncthreads();
    bool ok = true;
    for (int i = 0; t < p.rows; ++i, t += step) {
        const int s = i % p.stages;
        uint8_t* row = rope_smem + s * p.row_bytes;
        const float4* w4 = reinterpret_cast<const float4*>(turns + (i & 1) * room);
        int id = -1, in_page = 0;   // of the token's place
        if (warp == 0) {
            const int pg = pl >= 0 ? c.by_page(pl) : 0;
            in_page = pl - pg * c.page_size;
            if (pl >= 0 && (unsigned)seq < (unsigned)c.seqs && pg < c.max_pages) id = c.table[(size_t)seq * c.ld_table + pg];
            if (t + step < p.rows) seq = p.token_seq[t + step], pl = p.placement[t + step];
        }
        ok = ok && tc2_wait1(&full[s], (uint32_t)(i / p.stages) & 1u, s_abort, err, 0x6100 + s);
        if (ok) {
            if constexpr (FORM == kRopePairs) {
                const int h8 = p.half >> 3, d8 = p.dim >> 3;
                for (int it = tid; it < (p.heads + p.kv_heads) * h8; it += threads) {
                    const int head = it / h8, at = it - head * h8;
                    uint4* x = reinterpret_cast<uint4*>(row) + head * d8 + at;
                    const uint4 a = x[0], b = x[h8];
                    uint32_t xs[4] = {a.x, a.y, a.z, a.w}, ys[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float4 w = w4[u * pieces + at];
                        uint64_t f = rope_unpack<T>(xs[u]), g = rope_unpack<T>(ys[u]);
                        rope_turn(f, g, pa_two(w.x, w.y), pa_two(w.z, w.w));
                        xs[u] = rope_pack<T>(f), ys[u] = rope_pack<T>(g);
                    }
                    x[0] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
                    x[h8] = make_uint4(ys[0], ys[1], ys[2], ys[3]);
                }
            } else if constexpr (FORM == kRopeAdjacent) {
                const int d8 = p.dim >> 3;
                for (int it = tid; it < (p.heads + p.kv_heads) * pieces; it += threads) {
                    const int head = it / pieces, at = it - head * pieces;
                    uint4* x = reinterpret_cast<uint4*>(row) + head * d8 + at;
                    const uint4 a = x[0];
                    uint32_t xs[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        if (at * 4 + u >= p.half) continue;
                        const float4 w = w4[u / 2 * pieces + at];
                        const uint32_t second = xs[u + 1];
                        float f0, f1, g0, g1;
                        pa_split(rope_unpack<T>(xs[u]), f0, g0);
                        pa_split(rope_unpack<T>(second), f1, g1);
                        uint64_t f = pa_two(f0, f1), g = pa_two(g0, g1);
                        rope_turn(f, g, pa_two(w.x, w.y), pa_two(w.z, w.w));
                        pa_split(f, f0, f1);
                        pa_split(g, g0, g1);
                        xs[u] = rope_pack<T>(pa_two(f0, g0));
                        xs[u + 1] = at * 4 + u + 1 < p.half ? rope_pack<T>(pa_two(f1, g1)) : second;
                    }
                    x[0] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
                }
            } else {
                const float* w = reinterpret_cast<const float*>(w4);
                for (int it = tid; it < (p.heads + p.kv_heads) * p.half; it += threads) {
                    const int head = it / p.half, k = it - head * p.half;
                    T* x = reinterpret_cast<T*>(row) + head * p.dim + k;
                    const float cs = w[k / 2 * 4 + (k & 1)], sn = w[k / 2 * 4 + 2 + (k & 1)], f = to_f32<T>(x[0]), g = to_f32<T>(x[p.half]);
                    x[0] = from_f32<T>(fmaf(f, cs, -(g * sn)));
                    x[p.half] = from_f32<T>(fmaf(g, cs, f * sn));
                }
            }
        }
        angles(turns + ((i + 1) & 1) * room, t + step, pos);   // the readers of that half are a barrier behind
        pos = pos_of(ax, t + 2 * step);
        pa_fence_async();
        __syncthreads();
        if (warp == 0 && ok) {
            // queries in one piece; keys and values a head a lane, or in one piece too where a page holds them so
            const uint32_t head_bytes = (uint32_t)p.dim * 2, kv = (uint32_t)p.kv_heads * head_bytes;
            const uint8_t* from = row + p.heads * head_bytes;
            if (lane == 0) rope_s2g(static_cast<T*>(p.q) + (size_t)t * p.heads * p.dim, row, p.heads * head_bytes);
            if (id >= 0 && id < c.num_pages) {
                const long long at = (long long)id * c.page_stride + (long long)in_page * c.row_stride;
                T *k = static_cast<T*>(c.k) + at, *v = static_cast<T*>(c.v) + at;
                if (c.head_stride == p.dim || p.kv_heads == 1) {
                    if (lane == 0) rope_s2g(k, from, kv), rope_s2g(v, from + kv, kv);
                } else {
                    for (int h = lane; h < p.kv_heads; h += 32) {
                        rope_s2g(k + h * c.head_stride, from + h * head_bytes, head_bytes);
                        rope_s2g(v + h * c.head_stride, from + kv + h * head_bytes, head_bytes);
                    }
                }
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            // the row before this one has left the ring: its place takes the next one
            if (p.stages > 1) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            const int next = p.stages > 1 ? i - 1 + p.stages : i + 1;
            if (lane == 0 && (i > 0 || p.stages == 1)) fetch(next);
        }
    }
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // shared memory may go
    tc2_drain(s_abort);
}

constexpr int kRopeSmem = 220 * 1024;   // most that a CTA asks for

template <typename T, int FORM>
static int axes_rope(const AxesRope& p, const PagedCache& c, int ctas, int threads, int smem, bool pdl, zl_stream_t stream) {
    ZL_CHECK_WAITS();
    unsigned* words = wait_words();
    ZL_CHECK_CUDA(words ? cudaSuccess : cudaErrorMemoryAllocation);
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        ZL_CHECK_CUDA(cudaFuncSetAttribute(k_axes_rope_append<T, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRopeSmem));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    ZL_CHECK_CUDA(launch(k_axes_rope_append<T, FORM>, dim3(ctas), dim3(threads), smem, stream, pdl, p, c, words + kWaitRopePaged));
    return ZL_OK;
}

}  // namespace zl

using namespace zl;

extern "C" int zl_qkv_axes_rope_append(const void* qkv, long long ldq, const int32_t* pos, long long ld_pos, int axes, const double* inv_freq,
                                       const int32_t* axis, int half, int layout, float mscale, const int32_t* token_seq, const int32_t* placement,
                                       const int32_t* page_table, int ld_table, int max_pages, int seqs, void* k_cache, void* v_cache,
                                       long long num_pages, int page_size, long long page_stride, long long row_stride, long long head_stride,
                                       void* q_out, int T, int heads, int kv_heads, int dim, int dtype, int pdl, zl_stream_t stream) {
    ZL_CHECK_ARG(qkv && pos && token_seq && placement && q_out && T > 0 && heads > 0 && kv_heads > 0);
    ZL_CHECK_ARG(half >= 0 && 2 * half <= dim && axes > 0 && ld_pos >= T && (half == 0 || (inv_freq && axis)));
    ZL_CHECK_ARG(layout == ZL_ROT_HALVES || layout == ZL_ROT_ADJACENT);
    ZL_CHECK_PAGED(k_cache, v_cache, num_pages, page_size, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, seqs);
    ZL_CHECK_SUPPORTED(dim > 0 && dim % 8 == 0 && dim <= 1024 && dtype != ZL_F32);
    ZL_CHECK_ARG(ldq >= (long long)(heads + 2 * kv_heads) * dim);
    ZL_CHECK_SUPPORTED(ldq % 8 == 0 && ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) == 0);
    ZL_CHECK_SUPPORTED((heads + 2ll * kv_heads) * dim <= kRopeSmem / 2);   // a row in shared memory
    const PagedCache c = {k_cache, v_cache, num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, page_size, seqs, paged_divisor(page_size)};
    const int form = layout == ZL_ROT_ADJACENT ? kRopeAdjacent : half % 8 == 0 ? kRopePairs : kRopeAny;
    // a thread for every two pieces to turn; as many CTAs as the SMs hold threads of 64 registers, and rows in shared memory
    const int row_bytes = (heads + 2 * kv_heads) * dim * 2, turns = 2 * 8 * (half + 7);
    const int items = (heads + kv_heads) * (form == kRopePairs ? half / 8 : form == kRopeAdjacent ? (half + 3) / 4 : half), two = cdiv(items, 2 * 32) * 32;
    const int threads = two < 64 ? 64 : two < 256 ? two : 256;
    int stages = kRopeMaxStages;
    while (stages > 1 && stages * row_bytes + turns > kRopeSmem) --stages;
    const int smem = stages * row_bytes + turns;
    ZL_CHECK_SUPPORTED(smem <= kRopeSmem);
    const int by_smem = kSmSmem / (smem + kCtaSmem + 256), by_threads = 1024 / threads, most = device_sm_count() * (by_smem < by_threads ? by_smem : by_threads);
    const AxesRope p = {qkv, q_out, pos, axis, token_seq, placement, inv_freq, ldq, ld_pos, axes, half, heads, kv_heads, dim, mscale, T, stages, row_bytes};
    if (dtype == ZL_F16) return form == kRopePairs ? axes_rope<__half, kRopePairs>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream)
                                : form == kRopeAdjacent ? axes_rope<__half, kRopeAdjacent>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream)
                                                        : axes_rope<__half, kRopeAny>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream);
    return form == kRopePairs      ? axes_rope<__nv_bfloat16, kRopePairs>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream)
           : form == kRopeAdjacent ? axes_rope<__nv_bfloat16, kRopeAdjacent>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream)
                                   : axes_rope<__nv_bfloat16, kRopeAny>(p, c, T < most ? T : most, threads, smem, pdl != 0, stream);
}
