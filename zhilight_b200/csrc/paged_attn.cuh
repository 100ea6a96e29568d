// What the kernels of attention over pages share: their arguments, the blocks of rows that the sequences are cut into, and a row from its definition.
#pragma once
#include "paged.cuh"

namespace zl {

struct PagedAttn {
    const void* q;
    void* out;
    const int32_t *lens, *starts;
    int rows, heads, group, window;   // group: heads of a kv head
    PagedDivisor by_group;
    float scale;                      // times log2(e)
    int few, kv_heads;                // sequences of up to so many (token, head) rows of a kv head go to the kernel for few rows
    float2* ml;                       // parts of blocks that were cut, two places for every CTA: {maximum, sum} of their rows, and the rows
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

// What the block's rows see
__device__ __forceinline__ void paged_sees(const PagedAttn& p, PagedBlock& k) {
    const int t0 = p.by_group(k.row0), t1 = p.by_group(k.row0 + k.rows - 1);
    k.hi = min(k.place0 + t1, k.have - 1);
    k.lo = p.window ? max(0, k.place0 + t0 - p.window + 1) : 0;
    if (k.lo > k.hi) k.hi = -1, k.lo = 0;
}
__device__ __forceinline__ void paged_bounds(const PagedAttn& p, const PagedCache& c, PagedBlock& k) {
    const int len = p.lens[k.seq];
    k.place0 = len - p.starts[k.seq + 1] + k.first;
    k.have = min(max(len, 0), c.room());
    paged_sees(p, k);
}

struct PagedPlace {
    int hk, off, units;   // kv head; unit within the block, and how many that has
    int start;            // the block's place in the line
};

// A warp's view of the line that the blocks of a kernel's work stand in: sequence by sequence, in it kv head by kv head, in that block by block, each
// block KIND::units() long.  A CTA of the grid takes an equal stretch of the line.  128 sequences are in view at a time, four to a lane; the blocks of a
// sequence that has many are looked at by the whole warp.  Everything fits 32 bits, which the entry point sees to.
template <typename KIND>
struct PagedLine {
    static constexpr int kAlone = 4;   // blocks of a sequence that a lane looks at by itself
    int kv_heads, above, upto_rows;   // sequences of more than `above` and up to `upto_rows` (token, head) rows of a kv head are in it
    int b0, before, upto, cum[4];     // first sequence in view and its place; units of a kv head up to and with this lane's, and of this lane's four

    // units of the blocks of a sequence from `from` on, every `step`-th
    __device__ __forceinline__ int sum(const PagedAttn& p, PagedBlock& k, int n, int from, int step) {
        int units = 0;
        for (k.row0 = from * KIND::kRows; k.row0 < n; k.row0 += step * KIND::kRows) {
            k.rows = min(KIND::kRows, n - k.row0);
            paged_sees(p, k);
            units += KIND::units(k);
        }
        return units;
    }
    __device__ __forceinline__ void view(const PagedAttn& p, const PagedCache& c) {
        const int lane = threadIdx.x & 31, b = b0 + lane * 4;
        int at[5], len[4];
#pragma unroll
        for (int u = 0; u < 5; ++u) at[u] = b + u <= c.seqs ? p.starts[b + u] : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) len[u] = b + u < c.seqs ? p.lens[b + u] : 0;
        int all = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            PagedBlock k;
            k.first = max(at[u], 0);
            int n = b + u < c.seqs ? max(min(at[u + 1], p.rows) - k.first, 0) * p.group : 0;
            if (n <= above || n > upto_rows) n = 0;
            k.place0 = len[u] - at[u + 1] + k.first;
            k.have = min(max(len[u], 0), c.room());
            const bool many = n > kAlone * KIND::kRows;
            int units = many ? 0 : sum(p, k, n, 0, 1);
            for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
                const int src = __ffs(left) - 1;
                PagedBlock o;
                o.place0 = __shfl_sync(0xffffffffu, k.place0, src), o.have = __shfl_sync(0xffffffffu, k.have, src);
                const int x = __reduce_add_sync(0xffffffffu, sum(p, o, __shfl_sync(0xffffffffu, n, src), lane, 32));
                if (lane == src) units = x;
            }
            all += units;
            cum[u] = all;
        }
        upto = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
    }
    // length of the line; the view is at its beginning then
    __device__ __forceinline__ int begin(const PagedAttn& p, const PagedCache& c) {
        int total = 0;
        before = 0;
        for (b0 = (c.seqs - 1) & ~127;; b0 -= 128) {
            view(p, c);
            total += __shfl_sync(0xffffffffu, upto, 31) * kv_heads;
            if (b0 == 0) return total;
        }
    }
    // the block at place w, which is in view or behind it
    __device__ __forceinline__ void at(const PagedAttn& p, const PagedCache& c, int w, PagedBlock& k, PagedPlace& place) {
        const int lane = threadIdx.x & 31;
        unsigned hit;
        while (!(hit = __ballot_sync(0xffffffffu, before + upto * kv_heads > w))) {
            before += __shfl_sync(0xffffffffu, upto, 31) * kv_heads;
            b0 += 128;
            view(p, c);
        }
        const int src = __ffs(hit) - 1;
        int rem = w - before - __shfl_sync(0xffffffffu, upto - cum[3], src) * kv_heads, each = 0, u = 0;
#pragma unroll
        for (int v = 0, below = 0; v < 4; ++v) {
            const int x = __shfl_sync(0xffffffffu, cum[v], src) - below;   // units of this one
            if (each == 0) {
                if (rem < x * kv_heads) each = x, u = v;
                else rem -= x * kv_heads;
            }
            below += x;
        }
        place.hk = rem / each;
        rem -= place.hk * each;
        k.seq = b0 + src * 4 + u;
        const int n = paged_new(p, k.seq, k.first) * p.group;
        k.row0 = 0, k.rows = min(KIND::kRows, n);
        paged_bounds(p, c, k);
        place.units = KIND::units(k);
        // 32 blocks at a time
        for (int i0 = 0; n > KIND::kRows; i0 += 32) {
            PagedBlock o = k;
            o.row0 = (i0 + lane) * KIND::kRows, o.rows = min(KIND::kRows, n - o.row0);
            int mine = 0;
            if (o.row0 < n) paged_sees(p, o), mine = KIND::units(o);
            int up = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, up, d);
                if (lane >= d) up += x;
            }
            const unsigned here = __ballot_sync(0xffffffffu, up > rem);
            if (here) {
                const int l = __ffs(here) - 1;
                rem -= __shfl_sync(0xffffffffu, up - mine, l);
                k.row0 = (i0 + l) * KIND::kRows, k.rows = min(KIND::kRows, n - k.row0);
                paged_sees(p, k);
                place.units = KIND::units(k);
                break;
            }
            rem -= __shfl_sync(0xffffffffu, up, 31);
        }
        place.off = rem;
        place.start = w - rem;
    }
};

// Row t of q, one head, from the definition, by one warp: keys lo .. hi, one at a time.
template <typename T, int D>
__device__ __noinline__ void paged_row_exact(const PagedAttn& p, const PagedCache& c, int seq, int t, int h, int lo, int hi) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long head = (long long)p.by_group(h) * c.head_stride + lane;
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

// Row r of a block, D columns from `o`(e) of this lane, E neighbouring ones each: rounded and stored, or done again where it is no number
template <typename T, int D>
__device__ __forceinline__ void paged_row_out(const PagedAttn& p, const PagedCache& c, const PagedBlock& k, int hk, int r, float l, const float (&o)[D / 32]) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, row = k.row0 + r, t = p.by_group(row), head = hk * p.group + row - t * p.group, place = k.place0 + t;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T v[E];
    bool broken = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float x = l == 0.f ? 0.f : o[e] * inv;
        broken |= x != x;
        v[e] = from_f32<T>(x);
    }
    T* dst = static_cast<T*>(p.out) + ((size_t)(k.first + t) * p.heads + head) * D + lane * E;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
    else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(v);
    if (__any_sync(0xffffffffu, broken)) {
        __syncwarp();
        paged_row_exact<T, D>(p, c, k.seq, k.first + t, head, p.window ? max(0, place - p.window + 1) : 0, min(place, k.have - 1));
    }
}

// Blocks that were cut.  grid (the CTAs of the first kernel, groups of kJoinRows rows): CTA i joins the block that begins in stretch i of the line and goes on
// behind it -- there is one at the most.  Its first part lies in that CTA's place 1, the others in the place 0 of theirs.  HALVES: blocks of up to half
// of KIND::kRows rows have two parts in a place, one behind the other.
constexpr int kJoinRows = 16, kJoinThreads = 128;
template <typename T, int D, typename KIND, bool HALVES>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const PagedAttn p, const PagedCache c, int above, int upto_rows) {
    constexpr int R = KIND::kRows, E = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i0 = blockIdx.x;
    PagedLine<KIND> line;
    line.kv_heads = p.kv_heads, line.above = above, line.upto_rows = upto_rows;
    const int total = line.begin(p, c), per = cdiv(total, (int)gridDim.x), end = per * (i0 + 1);   // the first kernel has seen its predecessors end
    PagedBlock k;
    PagedPlace at;
    bool cut = end < total;
    if (cut) {
        line.at(p, c, end - 1, k, at);
        cut = at.start >= per * i0 && at.start + at.units > end;   // else it begins in an earlier stretch, or ends here
    }
    pdl_trigger();
    pdl_wait();
    if (!cut) return;
    const bool halves = HALVES && k.rows <= R / 2;
    const int parts = ((at.start + at.units - 1) / per - i0 + 1) << (halves ? 1 : 0);
    auto place = [&](int s, int r) {
        const int i = halves ? s >> 1 : s;
        return ((size_t)(i0 + i) * 2 + (i == 0)) * R + r + (halves && (s & 1) ? R / 2 : 0);
    };
    for (int r = blockIdx.y * kJoinRows + warp; r < min(k.rows, (int)(blockIdx.y + 1) * kJoinRows); r += kJoinThreads / 32) {
        float m = -INFINITY, l = 0.f, v[E] = {};
        for (int s = lane; s < parts; s += 32) m = fmaxf(m, p.ml[place(s, r)].x);
        m = warp_max(m);
        for (int s0 = 0; s0 < parts; s0 += 32) {
            const float2 x = s0 + lane < parts ? p.ml[place(s0 + lane, r)] : make_float2(-INFINITY, 0.f);
            const float f = s0 + lane < parts ? exp2f(x.x - m) : 0.f;
            l += warp_sum(x.y * f);
            const int n = min(32, parts - s0);
#pragma unroll 4
            for (int s = 0; s < n; ++s) {
                const float w = __shfl_sync(0xffffffffu, f, s);
                const float* from = p.part + place(s0 + s, r) * D + lane * E;
                if constexpr (E == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(from);
                    v[0] = fmaf(y.x, w, v[0]), v[1] = fmaf(y.y, w, v[1]), v[2] = fmaf(y.z, w, v[2]), v[3] = fmaf(y.w, w, v[3]);
                } else {
                    const float2 y = *reinterpret_cast<const float2*>(from);
                    v[0] = fmaf(y.x, w, v[0]), v[1] = fmaf(y.y, w, v[1]);
                }
            }
        }
        paged_row_out<T, D>(p, c, k, at.hk, r, l, v);
    }
}

}  // namespace zl
