// Rotation of fused query / key / value rows by positions on several axes, and their append to a paged cache: the counterpart of zl_qkv_rope_append
// for pictures and video, whose tokens have a place in time, height and width, each turning frequencies of its own.
//
//   angle[t][i] = pos[axis[i]][t] * inv_freq[i];   (a, b) -> (a cos - b sin, b cos + a sin) * mscale for the pair i of every query and key head
//
// A CTA serves a token: its threads first ask for their pieces of the row, then one thread for each frequency works out the angle's cosine and sine
// into shared memory.  Angle and reduction are in 64 bits (at position 4e6 a 32-bit angle is off by 0.25 rad): the angle in turns, less the nearest
// whole number, is exact to 1e-9 of a turn, and what is left of it goes through the 32-bit functions of CUDA (within 2e-7).  Bound by bytes: a row is read
// once and written once.  Products and sums are in 32 bits, rounded once.
#include "paged.cuh"

namespace zl {

constexpr int kRopeThreads = 256, kRopeAhead = 2;   // pieces of 16 bytes (pairs of them, where turned) that a thread asks for ahead of the angles

struct AxesRope {
    const void* qkv;
    void* q;
    const int32_t *pos, *axis, *token_seq, *placement;
    const double* inv_freq;
    long long ldq, ld_pos;
    int axes, half, heads, kv_heads, dim, adjacent, pairs;   // pairs: a piece of the first and its partner of the second half are turned together
    float mscale;
};

// grid (T)
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) k_axes_rope_append(const AxesRope p, const PagedCache c) {
    extern __shared__ float2 turn[];   // (cos, sin) of every frequency
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, tid = threadIdx.x;
    const T* row = static_cast<const T*>(p.qkv) + (size_t)t * p.ldq;
    const int d8 = p.dim >> 3, h8 = p.half >> 3;
    // pieces of a turned head: with pairs a piece of the first half brings its partner along
    const int each = p.pairs ? d8 - h8 : d8, turned = (p.heads + p.kv_heads) * each, total = turned + p.kv_heads * d8;
    auto place = [&](int it, int& head, int& at, bool& two) {
        if (it < turned) {
            head = it / each;
            at = it - head * each;
            two = p.pairs && at < h8;
            if (p.pairs && !two) at += h8;   // behind the turned columns
        } else {
            it -= turned;
            head = p.heads + p.kv_heads + it / d8;
            at = it % d8;
            two = false;
        }
    };
    uint4 a[kRopeAhead], b[kRopeAhead];
#pragma unroll
    for (int u = 0; u < kRopeAhead; ++u) {
        const int it = tid + u * kRopeThreads;
        if (it < total) {
            int head, at;
            bool two;
            place(it, head, at, two);
            const uint4* src = reinterpret_cast<const uint4*>(row + (size_t)head * p.dim);
            a[u] = src[at];
            if (two) b[u] = src[at + h8];
        }
    }
    for (int i = tid; i < p.half; i += kRopeThreads) {
        const int ax = p.axis[i];
        const double turns = (unsigned)ax < (unsigned)p.axes ? (double)p.pos[(size_t)ax * p.ld_pos + t] * p.inv_freq[i] * 0.15915494309189533577 : 0.0;
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        turn[i] = make_float2(cs * p.mscale, sn * p.mscale);
    }
    const int seq = p.token_seq[t], pl = p.placement[t];
    const long long at_cache = pl >= 0 && (unsigned)seq < (unsigned)c.seqs ? c.row_at(seq, pl) : -1;
    __syncthreads();
    for (int it = tid, u = 0; it < total; it += kRopeThreads, ++u) {
        int head, at;
        bool two;
        place(it, head, at, two);
        uint4 x, y;
        if (u < kRopeAhead) {
            x = u ? a[1] : a[0], y = u ? b[1] : b[0];
        } else {
            const uint4* src = reinterpret_cast<const uint4*>(row + (size_t)head * p.dim);
            x = src[at];
            if (two) y = src[at + h8];
        }
        T* dst;
        if (head < p.heads) {
            dst = static_cast<T*>(p.q) + ((size_t)t * p.heads + head) * p.dim;
        } else {
            const bool is_k = head < p.heads + p.kv_heads;
            dst = static_cast<T*>(is_k ? c.k : c.v) + at_cache + (long long)(head - p.heads - (is_k ? 0 : p.kv_heads)) * c.head_stride;
            if (at_cache < 0) continue;
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
                const T* src = row + (size_t)head * p.dim;
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
    const AxesRope p = {qkv, q_out, pos, axis, token_seq, placement, inv_freq, ldq, ld_pos, axes, half, heads, kv_heads, dim, adjacent, !adjacent && half % 8 == 0, mscale};
    const size_t smem = (size_t)half * sizeof(float2);
    if (dtype == ZL_F16) ZL_CHECK_CUDA(launch(k_axes_rope_append<__half>, dim3(T), dim3(kRopeThreads), smem, stream, pdl != 0, p, c));
    else if (dtype == ZL_BF16) ZL_CHECK_CUDA(launch(k_axes_rope_append<__nv_bfloat16>, dim3(T), dim3(kRopeThreads), smem, stream, pdl != 0, p, c));
    else ZL_CHECK_SUPPORTED(dtype == ZL_F16 || dtype == ZL_BF16);
    return ZL_OK;
}
