// Rotation of fused query / key / value rows by positions on several axes, and their append to a paged cache: the counterpart of zl_qkv_rope_append
// for pictures and video, whose tokens have a place in time, height and width, each turning frequencies of its own.
//
//   angle[t][i] = pos[axis[i]][t] * inv_freq[i];   (a, b) -> (a cos - b sin, b cos + a sin) * mscale for the pair i of every query and key head
//
// A CTA serves tokens in turn and asks for the pieces of the next one's row before it works on this one's: 16 bytes, a thread two of them (in halves with
// their partners).  One thread for each frequency works out the angle's cosine and sine into shared memory.  Angle and reduction are in 64 bits (at
// position 4e6 a 32-bit angle is off by 0.25 rad): the angle in turns, less the nearest whole number, is exact to 1e-9 of a turn, and what is left of it
// goes through CUDA's 32-bit functions (within 2e-7).  Products and sums are in 32 bits, rounded once.  Bound by bytes: a row is read once and written once.
#include "paged.cuh"

namespace zl {

constexpr int kRopeThreads = 512, kRopeAhead = 2;   // most threads; pieces that a thread asks for ahead

struct AxesRope {
    const void* qkv;
    void* q;
    const int32_t *pos, *axis, *token_seq, *placement;
    const double* inv_freq;
    long long ldq, ld_pos;
    int axes, half, heads, kv_heads, dim, adjacent, pairs;   // pairs: a piece of the first and its partner of the second half are turned together
    float mscale;
    int rows;
};

// grid: CTAs that share the tokens
template <typename T>
__global__ void __launch_bounds__(kRopeThreads, 2) k_axes_rope_append(const AxesRope p, const PagedCache c) {
    extern __shared__ float2 turns[];   // (cos, sin) of every frequency, of two tokens in turn
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, threads = blockDim.x, d8 = p.dim >> 3, h8 = p.half >> 3;
    // pieces of a turned head: with pairs a piece of the first half brings its partner along
    const int each = p.pairs ? d8 - h8 : d8, turned = (p.heads + p.kv_heads) * each, total = turned + p.kv_heads * d8;
    auto place = [&](int it, int& head, int& at, bool& two) {
        two = false;
        if (it < turned) {
            head = it / each;
            at = it - head * each;
            two = p.pairs && at < h8;
            if (p.pairs && !two) at += h8;   // behind the turned columns
        } else {
            it -= turned;
            head = p.heads + p.kv_heads + it / d8;
            at = it % d8;
        }
    };
    auto row_of = [&](int t) { return static_cast<const T*>(p.qkv) + (size_t)t * p.ldq; };
    int head[kRopeAhead], at[kRopeAhead];
    bool two[kRopeAhead];
#pragma unroll
    for (int u = 0; u < kRopeAhead; ++u) head[u] = -1, place(min(tid + u * threads, total - 1), head[u], at[u], two[u]);
    uint4 a[kRopeAhead], b[kRopeAhead];
    auto fetch = [&](int t) {
        const T* row = row_of(t);
#pragma unroll
        for (int u = 0; u < kRopeAhead; ++u)
            if (tid + u * threads < total) {
                const uint4* src = reinterpret_cast<const uint4*>(row + head[u] * p.dim);
                a[u] = src[at[u]];
                if (two[u]) b[u] = src[at[u] + h8];
            }
    };
    // this thread's first frequency; further ones are looked up again
    const int ax = tid < p.half ? p.axis[tid] : -1;
    const double freq = tid < p.half ? p.inv_freq[tid] * 0.15915494309189533577 : 0.0;
    auto pos_of = [&](int axis, int t) { return (unsigned)axis < (unsigned)p.axes ? p.pos[(size_t)axis * p.ld_pos + t] : 0; };
    auto angle = [&](int pos, double f) {
        const double x = (double)pos * f;
        float sn, cs;
        sincospif(2.0f * (float)(x - rint(x)), &sn, &cs);
        return make_float2(cs * p.mscale, sn * p.mscale);
    };
    int t = blockIdx.x, pos = pos_of(ax, t), seq = p.token_seq[t], pl = p.placement[t];
    fetch(t);
    for (int turn_of = 0; t < p.rows; turn_of ^= 1) {
        float2* turn = turns + turn_of * p.half;
        const long long cache = pl >= 0 && (unsigned)seq < (unsigned)c.seqs ? c.row_at(seq, pl) : -1;
        if (tid < p.half) turn[tid] = angle(pos, freq);
        for (int i = tid + threads; i < p.half; i += threads) turn[i] = angle(pos_of(p.axis[i], t), p.inv_freq[i] * 0.15915494309189533577);
        auto finish = [&](int head, int at, bool two, uint4 x, uint4 y) {
            T* dst;
            if (head < p.heads) {
                dst = static_cast<T*>(p.q) + ((size_t)t * p.heads + head) * p.dim;
            } else {
                const bool is_k = head < p.heads + p.kv_heads;
                dst = static_cast<T*>(is_k ? c.k : c.v) + cache + (long long)(head - p.heads - (is_k ? 0 : p.kv_heads)) * c.head_stride;
                if (cache < 0) return;
            }
            if (head < p.heads + p.kv_heads) {
                float f[8];
                unpack8<T>(x, f);
                if (two) {
                    float g[8];
                    unpack8<T>(y, g);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 w = turn[at * 8 + i];
                        const float v = f[i] * w.x - g[i] * w.y;
                        g[i] = g[i] * w.x + f[i] * w.y;
                        f[i] = v;
                    }
                    reinterpret_cast<uint4*>(dst)[at + h8] = pack8<T>(g);
                    x = pack8<T>(f);
                } else if (p.adjacent) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        if (at * 4 + (i >> 1) < p.half) {
                            const float2 w = turn[at * 4 + (i >> 1)];
                            const float v = f[i] * w.x - f[i + 1] * w.y;
                            f[i + 1] = f[i + 1] * w.x + f[i] * w.y;
                            f[i] = v;
                        }
                    }
                    x = pack8<T>(f);
                } else if (!p.pairs) {   // halves that do not begin on 16 bytes: the partner of every element by itself
                    const T* src = row_of(t) + head * p.dim;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int col = at * 8 + i;
                        if (col < p.half) {
                            const float2 w = turn[col];
                            f[i] = f[i] * w.x - to_f32<T>(src[col + p.half]) * w.y;
                        } else if (col < 2 * p.half) {
                            const float2 w = turn[col - p.half];
                            f[i] = f[i] * w.x + to_f32<T>(src[col - p.half]) * w.y;
                        }
                    }
                    x = pack8<T>(f);
                }
            }
            reinterpret_cast<uint4*>(dst)[at] = x;
        };
        const uint4 x0 = a[0], y0 = b[0], x1 = a[1], y1 = b[1];
        const int next = t + (int)gridDim.x;
        if (next < p.rows) fetch(next), pos = pos_of(ax, next), seq = p.token_seq[next], pl = p.placement[next];
        __syncthreads();   // the other buffer's readers are a barrier behind
        if (tid < total) finish(head[0], at[0], two[0], x0, y0);
        if (tid + threads < total) finish(head[1], at[1], two[1], x1, y1);
        for (int it = tid + kRopeAhead * threads; it < total; it += threads) {
            int h, at_;
            bool both;
            place(it, h, at_, both);
            const uint4* src = reinterpret_cast<const uint4*>(row_of(t) + h * p.dim);
            finish(h, at_, both, src[at_], both ? src[at_ + h8] : make_uint4(0, 0, 0, 0));
        }
        t = next;
    }
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
    ZL_CHECK_SUPPORTED((long long)(heads + 2 * kv_heads) * dim < 1 << 24);
    const PagedCache c = {k_cache, v_cache, num_pages, page_stride, row_stride, head_stride, page_table, ld_table, max_pages, page_size, seqs, paged_divisor(page_size)};
    const bool adjacent = layout == ZL_ROT_ADJACENT;
    const AxesRope p = {qkv, q_out, pos, axis, token_seq, placement, inv_freq, ldq, ld_pos, axes, half, heads, kv_heads, dim, adjacent, !adjacent && half % 8 == 0, mscale, T};
    // two pieces a thread where that is up to 512 threads, and as many CTAs as the SMs hold at 64 registers a thread
    const int d8 = dim / 8, pieces = (heads + kv_heads) * (p.pairs ? d8 - half / 8 : d8) + kv_heads * d8, two = cdiv(pieces, 2 * 32) * 32;
    const int threads = two < kRopeThreads ? two : kRopeThreads, most = device_sm_count() * (1024 / threads), ctas = T < most ? T : most;
    const size_t smem = 2 * (size_t)half * sizeof(float2);
    if (dtype == ZL_F16) ZL_CHECK_CUDA(launch(k_axes_rope_append<__half>, dim3(ctas), dim3(threads), smem, stream, pdl != 0, p, c));
    else if (dtype == ZL_BF16) ZL_CHECK_CUDA(launch(k_axes_rope_append<__nv_bfloat16>, dim3(ctas), dim3(threads), smem, stream, pdl != 0, p, c));
    else ZL_CHECK_SUPPORTED(dtype == ZL_F16 || dtype == ZL_BF16);
    return ZL_OK;
}
