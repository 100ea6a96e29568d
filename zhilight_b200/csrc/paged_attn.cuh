// What the kernels of attention over pages share: their arguments, the blocks of rows that the sequences are cut into, the join of few rows.
#pragma once
#include "paged.cuh"

#include <cfloat>

namespace zl {

// once for every device: `done` remembers
template <typename... KArgs>
static cudaError_t allow_smem(void (*kernel)(KArgs...), int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return e;
}

struct PagedAttn {
    const void* q;
    void* out;
    const int32_t *lens, *starts;
    int rows, heads, group, window;   // group: heads of a kv head
    PagedDivisor by_group;
    float scale;                      // times log2(e)
    int kv_heads;
    int block_rows, tile_rows;        // of a block; of one of its two tiles, 0 where blocks are one tile
    float2* ml;                       // parts of blocks that were cut, two places for every CTA: {maximum, sum} of their rows, and the rows
    float* part;
    struct PagedCut* cuts;            // for every CTA
    int split;                        // of kernels that share a call's sequences (KIND::takes): (token, head) rows of a kv head up to which one of them takes a sequence; 0 where one has all
};

// Exponentials carry 2^up, and a row's reference follows its maximum once that is more than `tau` above it.  fp16 probabilities are at most 2^15, and with 2^10 the
// small ones keep their bits.  bf16 ones have the exponents of 32-bit numbers: 2^(tau - 40) times the largest value, for as many keys as 31 bits count, stays
// below the largest 32-bit number; what is lost behind the lowest exponent is less than 2^-86, of the largest probability or of a product with a value.
template <bool HALF>
struct PagedExp {
    static constexpr float kTau = HALF ? 5.f : 8.f, kUp = HALF ? 10.f : -40.f;
};
constexpr float kPagedNone = -FLT_MAX;   // reference maximum of a row that has not seen a key yet: below every score, and finite (a masked score less it is -inf)

// One block of up to `size` (token, head) rows of a kv head of one sequence.
struct PagedBlock {
    int seq, first, n;   // its sequence, whose new tokens begin at row `first` of q and make up n (token, head) rows
    int row0, rows;      // (token, head) rows of the block, token-major
    int place0;          // place of the sequence's first new token
    int have;            // keys of the sequence
    int lo, hi;          // keys that any row of the block sees; hi < 0: none
};

// The first key that a row at `place` sees.  Rows before the sequence's beginning have negative places and see none; windows go up to the largest int.
__device__ __forceinline__ int paged_from(const PagedAttn& p, int place) { return p.window ? max(max(place + 1, 0) - p.window, 0) : 0; }

// What the block's rows see
__device__ __forceinline__ void paged_sees(const PagedAttn& p, PagedBlock& k) {
    const int t0 = p.by_group(k.row0), t1 = p.by_group(k.row0 + k.rows - 1);
    k.hi = min(k.place0 + t1, k.have - 1);
    k.lo = paged_from(p, k.place0 + t0);
    if (k.lo > k.hi) k.hi = -1, k.lo = 0;
}
struct PagedPlace {
    int hk, off, units;   // kv head; place within the block, and its length in the line: KIND::kSetup, what a block costs beside its turns, and then those
    int start;            // the block's place in the line
};

// A block that begins in a CTA's stretch of the line and goes on in the next ones: there is one at the most
struct PagedCut {
    PagedBlock k;
    int hk, parts;   // its kv head; stretches that have a part, 0: there is no such block
};

// A warp's view of the line that the blocks of a kernel's work stand in: sequence by sequence of those that KIND::takes(), in it kv head by kv head, in that block by block, each
// KIND::kSetup + KIND::turns() long.  A CTA of the grid takes an equal stretch of the line.  128 sequences are in view at a time, four to a lane; the blocks of a
// sequence that has many are looked at by the whole warp.  Everything fits 32 bits, which the entry point sees to, for sequences that have no more rows together
// than q: where they have, their rows overlap, and the line is empty.  No loop here goes by the lengths alone: one that changes under the kernel cannot keep it running.
template <typename KIND>
struct PagedLine {
    static constexpr int kAlone = 4;   // blocks of a sequence that a lane looks at by itself
    int total, per;                    // length of the line and of a stretch
    int b0, before, upto, cum[4];      // first sequence in view and its place; units of a kv head up to and with this lane's, and of this lane's four
    unsigned low, high;                // new tokens of this lane's four, 16 bits each and the rest

    static __device__ __forceinline__ int block(const PagedAttn& p, PagedBlock& k, int row0) {
        k.row0 = row0, k.rows = min(p.block_rows, k.n - row0);
        paged_sees(p, k);
        return KIND::kSetup + KIND::turns(p, k);
    }
    __device__ __forceinline__ void view(const PagedAttn& p, const PagedCache& c) {
        const int lane = threadIdx.x & 31, b = b0 + lane * 4;
        int at[5], len[4];
#pragma unroll
        for (int u = 0; u < 5; ++u) at[u] = b + u <= c.seqs ? p.starts[b + u] : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) len[u] = b + u < c.seqs ? p.lens[b + u] : 0;
        int all = 0;
        low = high = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            PagedBlock k;
            k.first = max(at[u], 0);
            k.n = b + u < c.seqs ? max(min(at[u + 1], p.rows), k.first) - k.first : 0;
            low += k.n & 0xffff, high += k.n >> 16;
            k.n *= p.group;
            if (!KIND::takes(p, k.n)) k.n = 0;
            k.place0 = len[u] - at[u + 1] + k.first;
            k.have = min(max(len[u], 0), c.room());
            const bool many = k.n > kAlone * p.block_rows;
            int units = 0;
            if (!many)
                for (int r = 0; r < k.n; r += p.block_rows) units += block(p, k, r);
            for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
                const int src = __ffs(left) - 1;
                PagedBlock o;
                o.place0 = __shfl_sync(0xffffffffu, k.place0, src), o.have = __shfl_sync(0xffffffffu, k.have, src), o.n = __shfl_sync(0xffffffffu, k.n, src);
                int x = 0;
                for (int r = lane * p.block_rows; r < o.n; r += 32 * p.block_rows) x += block(p, o, r);
                x = __reduce_add_sync(0xffffffffu, x);
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
    // length of the line, which `ctas` share; the view is at its beginning then
    __device__ __forceinline__ void begin(const PagedAttn& p, const PagedCache& c, int ctas) {
        total = before = 0;
        long long rows = 0;
        for (b0 = (c.seqs - 1) & ~127;; b0 -= 128) {
            view(p, c);
            rows += ((long long)__reduce_add_sync(0xffffffffu, high) << 16) + __reduce_add_sync(0xffffffffu, low);
            total += __shfl_sync(0xffffffffu, upto, 31) * p.kv_heads;
            if (b0 == 0) break;
        }
        if (rows > p.rows) total = 0;
        per = (total + ctas - 1) / ctas;
    }
    // the block at place w, which is in view or behind it; false: there is none
    __device__ __forceinline__ bool at(const PagedAttn& p, const PagedCache& c, int w, PagedBlock& k, PagedPlace& place) {
        const int lane = threadIdx.x & 31;
        unsigned hit;
        while (!(hit = __ballot_sync(0xffffffffu, before + upto * p.kv_heads > w))) {
            before += __shfl_sync(0xffffffffu, upto, 31) * p.kv_heads;
            b0 += 128;
            if (b0 >= c.seqs) return false;
            view(p, c);
        }
        const int src = __ffs(hit) - 1;
        int rem = w - before - __shfl_sync(0xffffffffu, upto - cum[3], src) * p.kv_heads, each = 0, u = 0;
#pragma unroll
        for (int v = 0, below = 0; v < 4; ++v) {
            const int x = __shfl_sync(0xffffffffu, cum[v], src) - below;   // units of this one
            if (each == 0) {
                if (rem < x * p.kv_heads) each = x, u = v;
                else rem -= x * p.kv_heads;
            }
            below += x;
        }
        place.hk = rem / each;
        rem -= place.hk * each;
        k.seq = b0 + src * 4 + u;
        k.first = max(p.starts[k.seq], 0);
        k.n = (max(min(p.starts[k.seq + 1], p.rows), k.first) - k.first) * p.group;
        const int len = p.lens[k.seq];
        k.place0 = len - p.starts[k.seq + 1] + k.first;
        k.have = min(max(len, 0), c.room());
        // 32 blocks at a time
        int row0 = 0;
        for (int r0 = 0; k.n > p.block_rows && r0 < k.n; r0 += 32 * p.block_rows) {
            PagedBlock o = k;
            const int r = r0 + lane * p.block_rows, mine = r < k.n ? block(p, o, r) : 0;
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
                row0 = r0 + l * p.block_rows;
                break;
            }
            rem -= __shfl_sync(0xffffffffu, up, 31);
        }
        place.units = block(p, k, row0);
        place.off = min(rem, place.units - 1);
        place.start = w - place.off;
        return true;
    }
};

// A CTA's way along its stretch of the line
template <typename KIND>
struct PagedWalk {
    PagedBlock k;
    PagedPlace place;
    int w, end, per;   // place in the line, end of the stretch, length of a stretch

    // at w, or (w < 0) at the beginning of the CTA's stretch
    __device__ __forceinline__ void find(const PagedAttn& p, const PagedCache& c, int at) {
        PagedLine<KIND> line;
        line.begin(p, c, (int)gridDim.x);
        per = line.per;
        const int first = min(line.total, per * (int)blockIdx.x);
        w = at < 0 ? first : at;
        end = min(line.total, first + per);
        if (w < end && !line.at(p, c, w, k, place)) w = end;
    }
    // turns first .. first + count - 1 of the block are this CTA's; none where the stretch ends before the block's first turn
    __device__ __forceinline__ void share(int& first, int& count) const {
        first = max(place.off - KIND::kSetup, 0);
        count = max(place.off + min(end - w, place.units - place.off) - KIND::kSetup, 0) - first;
    }
    __device__ __forceinline__ bool whole(int count) const { return count == place.units - KIND::kSetup; }
    // on to the next block
    __device__ __forceinline__ void go(const PagedAttn& p, const PagedCache& c) {
        w += min(end - w, place.units - place.off);
        if (w >= end) return;
        int row0 = k.row0 + p.block_rows;
        if (row0 >= k.n) {
            if (place.hk + 1 == p.kv_heads) return find(p, c, w);
            row0 = 0, ++place.hk;
        }
        place.units = PagedLine<KIND>::block(p, k, row0);
        place.off = 0;
        place.start = w;
    }
    // notes a block that this CTA has the first, but not all turns of: there is one at the most
    __device__ __forceinline__ void cut(const PagedAttn& p, int first, int count) const {
        if (first == 0 && !whole(count)) {
            PagedCut x = {k, place.hk, (place.start + place.units - 1) / per - (int)blockIdx.x + 1};
            p.cuts[blockIdx.x] = x;
        }
    }
};

// Row r of a block, D columns, E neighbouring ones of this lane: rounded and stored
template <typename T, int D>
__device__ __forceinline__ void paged_row_out(const PagedAttn& p, const PagedBlock& k, int hk, int r, float l, const float (&o)[D / 32]) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, row = k.row0 + r, t = p.by_group(row), head = hk * p.group + row - t * p.group;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = from_f32<T>(l == 0.f ? 0.f : o[e] * inv);
    T* dst = static_cast<T*>(p.out) + ((size_t)(k.first + t) * p.heads + head) * D + lane * E;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
    else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(v);
}

// Blocks that were cut, of the kernel for few rows.  grid (its CTAs): the first part of a block lies in its CTA's place 1, the others in the place 0 of theirs,
// R rows each.  A chain of three loads bounds it, so the warps share out the rows and, where there are fewer, the parts of a row too, and ask for many at
// once; more CTAs, a row each, cost more than they give (37 blocks that nothing cuts: 13.4 -> 22.5 us a call).
constexpr int kJoinWarps = 16, kJoinAhead = 4;   // not fewer warps than rows
template <typename T, int D, int R>
__global__ void __launch_bounds__(kJoinWarps * 32) k_paged_join(const PagedAttn p) {
    constexpr int E = D / 32;
    static_assert(R <= kJoinWarps, "a warp for every row");
    __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_v[kJoinWarps][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const PagedCut x = p.cuts[blockIdx.x];
    if (x.parts == 0) return;
    const int each = kJoinWarps / x.k.rows, group = warp % each, r = warp / each;   // warps of a row, and this one's
    const bool mine = r < x.k.rows;
    auto place = [&](int s) { return ((size_t)(blockIdx.x + s) * 2 + (s == 0)) * R + r; };
    float m = -INFINITY, l = 0.f, v[E] = {};
    for (int s0 = group; s0 < x.parts && mine; s0 += each * kJoinAhead) {
        float2 ml[kJoinAhead];
        float z[kJoinAhead][E];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
            const int s = s0 + u * each;
            ml[u] = make_float2(-INFINITY, 0.f);
            if (s < x.parts) {
                ml[u] = p.ml[place(s)];
                const float* from = p.part + place(s) * D + lane * E;
#pragma unroll
                for (int e = 0; e < E; e += 2) *reinterpret_cast<float2*>(&z[u][e]) = *reinterpret_cast<const float2*>(from + e);
            }
        }
        float up = m;
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) up = fmaxf(up, ml[u].x);
        const float f = exp2f(m - up);
        l *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= f;
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
            if (s0 + u * each >= x.parts) break;
            const float g = exp2f(ml[u].x - up);
            l = fmaf(ml[u].y, g, l);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = fmaf(z[u][e], g, v[e]);
        }
        m = up;
    }
    if (each > 1) {
        if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
        for (int e = 0; e < E; ++e) s_v[warp][lane * E + e] = v[e];
        __syncthreads();
        if (group == 0 && mine) {
            float up = m;
            for (int w = 1; w < each; ++w) up = fmaxf(up, s_m[warp + w]);
            const float f = exp2f(m - up);
            l *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] *= f;
            for (int w = 1; w < each; ++w) {
                const float g = s_m[warp + w] == -INFINITY ? 0.f : exp2f(s_m[warp + w] - up);   // a warp without a part
                l = fmaf(s_l[warp + w], g, l);
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fmaf(s_v[warp + w][lane * E + e], g, v[e]);
            }
        }
    }
    if (group == 0 && mine) paged_row_out<T, D>(p, x.k, x.hk, r, l, v);
}

// The kernel for tiles and its join, over a cache of 16 bits (paged_attn.cu): checked arguments
int paged_tiles(const PagedAttn& p, const PagedCache& c, int ctas, int dim, int dtype, bool pdl, zl_stream_t stream);

}  // namespace zl
