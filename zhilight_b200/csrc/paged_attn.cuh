// What the kernels of attention over pages share: their arguments, the blocks of rows that the sequences are cut into, and a row from its definition.
#pragma once
#include "paged.cuh"

namespace zl {

struct PagedAttn {
    const void* q;
    void* out;
    const int32_t *lens, *starts;
    int rows, heads, group, window;   // group: heads of a kv head
    float scale;                      // times log2(e)
    int few;                          // sequences of up to so many (token, head) rows of a kv head are the other kernel's
    int splits;                       // key ranges of a block
    float2* ml;                       // {maximum, sum} of the parts, then their outputs
    float* part;
};

// One block of up to `size` (token, head) rows of a kv head of one sequence.
struct PagedBlock {
    int seq, first;      // its sequence, whose new tokens begin at row `first` of q
    int row0, rows;      // (token, head) rows of the block, token-major
    int place0;          // place of the sequence's first new token
    int have;            // keys of the sequence
    int lo, hi;          // keys that any row of the block sees; hi < 0: none
};

// The new tokens of sequence b, as far as q has them.
__device__ __forceinline__ int paged_new(const PagedAttn& p, int b, int& first) {
    first = max(p.starts[b], 0);
    return max(min(p.starts[b + 1], p.rows) - first, 0);
}

__device__ __forceinline__ void paged_bounds(const PagedAttn& p, const PagedCache& c, PagedBlock& k) {
    const int len = p.lens[k.seq];
    k.place0 = len - p.starts[k.seq + 1] + k.first;
    k.have = min(max(len, 0), c.room());
    const int t0 = k.row0 / p.group, t1 = (k.row0 + k.rows - 1) / p.group;
    k.hi = min(k.place0 + t1, k.have - 1);
    k.lo = p.window ? max(0, k.place0 + t0 - p.window + 1) : 0;
    if (k.lo > k.hi) k.hi = -1, k.lo = 0;
}

// The blocks of the sequences with more than p.few rows, sequence by sequence, the last blocks of a sequence, which see the most keys, first.  Called by
// whole warps; false: there is no block `item`.
__device__ __forceinline__ bool paged_block(const PagedAttn& p, const PagedCache& c, int item, int size, PagedBlock& k) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < c.seqs; b0 += 32) {
        int first = 0, n = 0;
        if (b0 + lane < c.seqs) n = paged_new(p, b0 + lane, first) * p.group;
        const int mine = n > p.few ? (n + size - 1) / size : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, item < upto);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int at = __shfl_sync(0xffffffffu, upto - 1, src) - item;   // 0: the sequence's first block
            k.seq = b0 + src;
            k.first = __shfl_sync(0xffffffffu, first, src);
            k.row0 = at * size;
            k.rows = min(size, __shfl_sync(0xffffffffu, n, src) - k.row0);
            paged_bounds(p, c, k);
            return true;
        }
        item -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Row t of q, one head, from the definition, by one warp: keys lo .. hi, one at a time.
template <typename T, int D>
__device__ __noinline__ void paged_row_exact(const PagedAttn& p, const PagedCache& c, int seq, int t, int h, int lo, int hi) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long head = (long long)(h / p.group) * c.head_stride + lane;
    const size_t row = ((size_t)t * p.heads + h) * D + lane;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = to_f32<T>(static_cast<const T*>(p.q)[row + e * 32]);
    for (int j = lo; j <= hi; ++j) {
        const long long r = c.row_at(seq, j);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (r >= 0) s = fmaf(q[e], to_f32<T>(static_cast<const T*>(c.k)[r + head + e * 32]), s);
        s = warp_sum(s) * p.scale;
        const float up = s != s ? s : fmaxf(m, s), f = up == -INFINITY ? 1.f : exp2f(m - up), w = up == -INFINITY ? 0.f : exp2f(s - up);
        m = up;
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + (r >= 0 ? w * to_f32<T>(static_cast<const T*>(c.v)[r + head + e * 32]) : 0.f);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) static_cast<T*>(p.out)[row + e * 32] = from_f32<T>(l > 0.f || l != l ? o[e] / l : 0.f);
}

}  // namespace zl
