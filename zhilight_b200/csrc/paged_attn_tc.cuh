// Attention of many new tokens over pages on the 5th-generation tensor cores.  A tile is up to 128 (token, head) rows of one kv head of one sequence, whole
// tokens with all heads of the group; blocks of one or two tiles walk the keys of their rows in turns, two tiles of 128 x 128 scores a turn: the block's two
// row tiles over the same keys, or its one tile over two tiles of keys, whose results are joined at the end.  The turns of all blocks stand in one
// line that the CTAs, one per SM, share out evenly (paged_attn.cuh).
//
//   warps 0-3, 4-7  softmax of a tile each: thread = row = lane of tensor memory; running maximum and sum in 32 bits; probabilities go back over the scores
//   warp 8          one thread issues S = Q K^T of both tiles, 64 keys at a time into two buffers each
//   warp 9          one thread issues O += P V of both tiles (P from tensor memory, V as it lies: rows of keys, the B operand along n)
//   warps 10, 11    Q by TMA, once for a block; K and V, a warp each, from the pages into a ring of tiles of 64 keys by TMA, a box for the rows of a tile
//                   that one page has (where these are fewer than four, or a page has fewer than 8, both copy 16 bytes at a time)
//
// A page's rows behind the last visible key may hold anything.  Copies of 16 bytes leave them out; behind TMA the softmax's threads make those values zeros
// before they hand the tile's probabilities on.  Rows behind a page number outside the pool are zeros either way.  Tensor memory: scores of the two tiles
// (128 columns each, probabilities over their first half), then their outputs.  Probabilities are rounded to the rows' type once (half a step each, of random sign: beside the output's own rounding), the
// sums that divide them are not.  A row's reference maximum follows the true one only once that has grown by 2^5 (fp16) or 2^8:
// any reference gives the same quotient (PagedExp).
//
// A masked probability is exactly zero, but zero times an infinity or NaN that a row must not see (a later token's value, one before its window) is NaN in its
// sum.  Of the keys that not all rows of a block see (its last ones, and the first ones of a window) the softmax's threads therefore look the values over before they
// hand the tile's probabilities on, and put zeros where they are no numbers (pt_clean); at the block's end they add those to the rows that do see them (pt_add_broken).
//
// 4096 tokens behind 4096, 32 heads on 8, bf16: 395 us in a graph, 455 in a row of calls, 0.91 to 1.04 PFLOP/s; the look at the values takes 5 us of it.  A turn takes 3000 cycles, of
// which the MMAs need 2050 at least and the exponentials of both groups 2050; under this load the SM runs at 1.2 GHz.  On the way, the same in us: copies of 16 bytes by two warps 693 (they bound it),
// TMA 544, scores of 64 keys ahead of the softmax in two buffers 503 (128 keys at a time leave no room for a second one, and S -> softmax -> P V is
// then one chain of 4400 cycles), a thread each for S and P V 434, Q and the first scores under the results of the block before 420, parts column by column 395.
// Scores of 64 keys read Q twice as often; they are 450 cycles each instead of 300.  Blocks of up to 128 rows stream K and V like the kernel for few rows, five turns
// of 64 keys in flight: drafts of 16 users, 64 heads on 8, 57 us for 186 MB under ncu, 65 a call with the join (when it took 68: 103 where a block's setup did not count
// as two turns).
//
// Where the look at the values stands was measured, drafts / mixed portions with a window / this prompt in us without it 68 / 68 / 388: here 70 / 69 / 393; with a barrier
// and the product of such tiles by the softmax's threads 69 / 78 / 394; by warp 9 before its products 73 / 80 / 404; by the loaders, once a tile has landed, 77 / 81 / 406.
#pragma once
#include "attn_ptx.cuh"
#include "int4_cache.cuh"
#include "paged_attn.cuh"

#include <type_traits>

namespace zl {

constexpr int kPtRows = 256, kPtKeys = 128, kPtHalf = 64, kPtWarpS = 8, kPtWarpO = 9, kPtWarpLoad = 10, kPtLoaders = 64;
// Of a cache of 4 bits: warps 10 and 11 bring codes of keys and of values, a ring of tiles each, as they are; warps 12 to 15 make them numbers of T on the way into the ring
// of tiles, 16 rows of every tile each (all four in every tile: a warp that passed over some could take one phase of their barriers for another).
// 2048 tokens of 32 heads on 8 behind 6000: 302 us, bound by these four warps, one on each scheduler beside two of the softmax (when it took 309, 1900 of the 2700 cycles
// for 64 keys went by in them).  More threads would leave the softmax too few registers.
constexpr int kPtWarpLoad4 = 12;
template <bool INT4>
constexpr int kPtThreads = INT4 ? 512 : 384;

// The exponent of a probability is a score times the scale less the reference, in one fused step that does not round the product, where the reference is
// one that was rounded: all exponents of a row are off by what that left, half a step of 32-bit numbers of its size.  That cancels in the quotient, but from here on
// (2^22, half a step of 1/4) it could leave the range of the probabilities, so the product is rounded as the reference was before the difference is taken.
constexpr float kPtFar = 4194304.f;

// The probabilities of 64 keys, of which a row sees from .. to, written over their scores at tb, where the reference is that far off: -> their sum
template <typename T>
__device__ __noinline__ float pt_far(uint32_t tb, float scale, float m_ref, float up, int from, int to) {
    float sum = 0.f;
#pragma unroll 1
    for (int part = 0; part < kPtHalf; part += 32) {
        uint32_t x[16];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float v[16];
            tc_ld16(tb + (uint32_t)(part + half * 16), v);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                T two[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = part + half * 16 + i + e;
                    const float y = key >= from && key <= to ? pa_exp2(__fadd_rn(__fsub_rn(__fmul_rn(v[i + e], scale), m_ref), up)) : 0.f;
                    sum += y;
                    two[e] = from_f32<T>(y);
                }
                x[half * 8 + i / 2] = *reinterpret_cast<const uint32_t*>(two);
            }
        }
        tc_st16(tb + (uint32_t)(part / 2), x);
    }
    return sum;
}

// turns of a block, at least one: a block that sees nothing is written too
struct PtKind {
    static constexpr int kSetup = 2;
    static __device__ __forceinline__ int turns(const PagedAttn& p, const PagedBlock& k) {
        const int tiles = k.hi >= 0 ? k.hi / kPtKeys - k.lo / kPtKeys + 1 : 1;
        return k.rows > p.tile_rows ? tiles : (tiles + 1) >> 1;
    }
    static __device__ __forceinline__ bool takes(const PagedAttn& p, int rows) { return rows > p.split; }
};

template <int D, bool INT4 = false>
struct PtCfg {
    static constexpr int kAtoms = D / 64;
    static constexpr int kQ = kAtoms * kPaRows * 128;       // a tile of Q: [64 of d][128 rows][128 B]
    static constexpr int kTile = kAtoms * kPtHalf * 128;    // K or V: [64 of d][64 keys][128 B]
    static constexpr int kRing = D == 64 ? 16 : INT4 ? 8 : 10;
    static constexpr int kRaw = D == 64 ? 6 : 3;            // tiles of codes, of keys and as many of values
    static constexpr int kCodes = kPtHalf * kInt4Pitch<D>;  // a tile's codes and pairs
    static constexpr int kRingOff = 2 * kQ, kRawOff = kRingOff + kRing * kTile;
    static constexpr int kBytes = kRawOff + (INT4 ? 2 * kRaw * kCodes : 0) + 1024;   // + slack for the manual 1024-byte alignment
    static_assert(tmem_alone(kBytes) && kBytes + 1024 <= 227 * 1024, "all of tensor memory, an SM to itself");
    static_assert(2 * kQ >= kPaRows * D * 4, "the second result of a row, where Q was");
    static constexpr int kO = 256;                          // TMEM columns: scores 0, 128; outputs from here
};

__device__ __forceinline__ void pt_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void pt_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
// tc2_wait for a barrier whose phase has mostly ended by now: all lanes look once
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, volatile int* s_abort, unsigned* err, unsigned code) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || tc2_wait(bar, parity, s_abort, err, code);
}

template <int D>
__device__ __forceinline__ void int4_box(uint32_t dst, const CUtensorMap* map, int form, int hk, int row, int page, uint64_t* bar) {
    const bool wide = D == 64 && form == kInt4Wide;
    pt_load_4d(dst, map, D == 128 ? 0 : wide ? hk * 10 - (hk & 1) * 2 : row * 10, D == 128 || wide ? row : 0, wide ? 0 : hk, page, bar);
}

template <typename T>
constexpr uint32_t kPtInf = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80;   // magnitudes from here on are no numbers
// the larger magnitudes of pairs of elements
__device__ __forceinline__ uint32_t pt_magnitude(const uint4& w) {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs), __vmaxu2(w.z & kAbs, w.w & kAbs));
}
// 8 values: those that are no numbers become zeros.  Whether there are any
template <typename T>
__device__ __forceinline__ bool pt_clean(uint4* at) {
    const uint32_t top = pt_magnitude(*at);
    if ((top & 0xffffu) < kPtInf<T> && top >> 16 < kPtInf<T>) return false;
    uint16_t* w = reinterpret_cast<uint16_t*>(at);
    for (int i = 0; i < 8; ++i)
        if ((w[i] & 0x7fffu) >= kPtInf<T>) w[i] = 0;
    return true;
}
// Adds the values that pt_clean takes out, of keys lo .. hi that a row sees, to the outputs of a warp's rows (tensor memory, D columns from `ob`): of the keys
// first .. last without those in from .. to, in tiles of 128 the first of every `step`.  A lane looks at a key at a time.
template <typename T, int D>
__device__ __noinline__ void pt_add_broken(const PagedCache& c, int seq, long long head, uint32_t ob, int lo, int hi, int first, int last, int from, int to, int step) {
    const int lane = threadIdx.x & 31;
    for (int key0 = first; key0 <= last; key0 += 32) {
        if (key0 >= from && key0 + 31 <= to) {
            key0 = to - 31;
            continue;
        }
        const int mine = key0 + lane;
        const long long at = mine <= last && (mine < from || mine > to) && (mine - first) / kPtKeys % step == 0 ? c.row_at(seq, mine) : -1;
        uint32_t top = 0;
        if (at >= 0)
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += 8) top = __vmaxu2(top, pt_magnitude(*reinterpret_cast<const uint4*>(static_cast<const T*>(c.v) + at + head + d0)));
        for (unsigned left = __ballot_sync(0xffffffffu, (top & 0xffffu) >= kPtInf<T> || top >> 16 >= kPtInf<T>); left; left &= left - 1) {
            const int key = key0 + __ffs(left) - 1;
            const long long row = __shfl_sync(0xffffffffu, at, key - key0);
#pragma unroll 1
            for (int d0 = 0; d0 < D; d0 += 16) {
                float o[16];
                tc_ld16(ob + (uint32_t)d0, o);
                const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(c.v) + row + head + d0);
                const uint4 two[2] = {v[0], v[1]};
                const T* x = reinterpret_cast<const T*>(two);
                uint32_t r[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float y = to_f32<T>(x[i]);
                    r[i] = __float_as_uint(key >= lo && key <= hi && !(fabsf(y) < INFINITY) ? o[i] + y : o[i]);
                }
                tc_st16(ob + (uint32_t)d0, r);
                tc_wait_st();
            }
        }
    }
}

// The same for a cache of 4 bits, whose values are none where their group's pair is none: a lane looks at the pairs of a key at a time.
template <typename T, int D>
__device__ __noinline__ void pt_add_broken4(const PagedCache& c, int seq, long long head, uint32_t ob, int lo, int hi, int first, int last, int from, int to, int step) {
    const int lane = threadIdx.x & 31;
    for (int key0 = first; key0 <= last; key0 += 32) {
        if (key0 >= from && key0 + 31 <= to) {
            key0 = to - 31;
            continue;
        }
        const int mine = key0 + lane;
        const long long at = mine <= last && (mine < from || mine > to) && (mine - first) / kPtKeys % step == 0 ? c.row_at(seq, mine) : -1;
        const uint8_t* pairs = static_cast<const uint8_t*>(c.v) + head + D / 2;
        bool whole = true;
        if (at >= 0)
#pragma unroll
            for (int g = 0; g < D / kInt4Group; ++g) whole = whole && int4_finite<T>(*reinterpret_cast<const uint32_t*>(pairs + at + g * 4));
        for (unsigned left = __ballot_sync(0xffffffffu, !whole); left; left &= left - 1) {
            const int key = key0 + __ffs(left) - 1;
            const long long row = __shfl_sync(0xffffffffu, at, key - key0);
#pragma unroll 1
            for (int d0 = 0; d0 < D; d0 += 16) {
                if (int4_finite<T>(*reinterpret_cast<const uint32_t*>(pairs + row + d0 / kInt4Group * 4))) continue;
                float o[16];
                tc_ld16(ob + (uint32_t)d0, o);
                uint32_t r[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(key >= lo && key <= hi ? __int_as_float(0x7fffffff) : o[i]);
                tc_st16(ob + (uint32_t)d0, r);
                tc_wait_st();
            }
        }
    }
}

// grid: CTAs that share the line.  box: rows of a TMA box of K and V, 0: no TMA.  INT4: one of kInt4Copies ..., for boxes of 16 rows
template <typename T, int D, bool INT4 = false>
__global__ void __launch_bounds__(kPtThreads<INT4>, 1)
k_paged_attn_tiles(const PagedAttn p, const PagedCache c, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, int box, unsigned* err) {
    using C = PtCfg<D, INT4>;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kScale = INT4 ? Int4Codes<T, false>::kScale : 1.f;   // of keys and values: probabilities carry it too, the scores' scale and the sums take it away
    constexpr int CH = D / 8;
    extern __shared__ uint8_t pt_smem[];
    uint8_t* smem = pt_smem + ((1024u - (smem_u32(pt_smem) & 1023u)) & 1023u);
    __shared__ uint64_t full[C::kRing], empty[C::kRing], s_full[2][2], p_full[2][2], o_done[2][2], q_full, q_free, o_free, joined;
    __shared__ uint64_t raw_full[2][INT4 ? C::kRaw : 1], raw_empty[2][INT4 ? C::kRaw : 1];
    __shared__ float2 s_ml[kPaRows];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up, s_blocks[2];
    // s_broken[i % 2] is i + 1 where block i had values that are no numbers and that not all rows see; no warp of the softmax is two blocks ahead of another
    volatile int *s_abort = &s_gave_up, *s_broken = s_blocks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < C::kRing; ++i) mbar_init(&full[i], INT4 ? kPtHalf / 16 : box ? 1 : kPtLoaders), mbar_init(&empty[i], 1);
        for (int i = 0; i < 4; ++i) mbar_init(&s_full[i >> 1][i & 1], 1), mbar_init(&p_full[i >> 1][i & 1], 4), mbar_init(&o_done[i >> 1][i & 1], 1);
        if constexpr (INT4)
            for (int i = 0; i < 2 * C::kRaw; ++i) mbar_init(&raw_full[i & 1][i >> 1], box ? 1 : 32), mbar_init(&raw_empty[i & 1][i >> 1], 4);
        mbar_init(&q_full, 1), mbar_init(&q_free, 1), mbar_init(&o_free, 8), mbar_init(&joined, 4);
        s_gave_up = s_blocks[0] = s_blocks[1] = 0;
        mbar_fence_init();
    }
    if (warp == kPtWarpS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    pdl_trigger();
    const uint32_t tmem = s_tmem;
    if (tid == 0) p.cuts[blockIdx.x].parts = 0;
    // Of the blocks before: how many, their turns, their tiles of the ring.  Every barrier's phases are waited for by each of its waiters without a gap, or a
    // later one cannot end before the waiter has gone on: a phase is told from its neighbours by its parity alone.
    int blocks = 0, turn = 0, ring = 0;   // ring / 2: of keys, and of values
    bool ok = true;           // no wait has given up
    PagedWalk<PtKind> walk;
    const PagedBlock& k = walk.k;
    const PagedPlace& at = walk.place;
    walk.find(p, c, -1);
    bool was_joined = false;  // the block before had one tile of rows, and its two results met where Q lies
    int joins_before = 0;     // blocks so far that did
    for (; walk.w < walk.end; walk.go(p, c)) {
        int first, count;
        walk.share(first, count);
        if (count == 0) continue;
        const bool two_rows = k.rows > p.tile_rows, joins = !two_rows && walk.whole(count);   // two row tiles; else two key tiles
        const int t0 = (k.hi >= 0 ? k.lo / kPtKeys : 0) + (two_rows ? first : 2 * first), items = two_rows ? 2 : 4;   // of the ring for 64 keys
        // keys that all rows of the block see
        const int all_hi = min(k.place0 + p.by_group(k.row0), k.have - 1);
        const int all_lo = paged_from(p, k.place0 + p.by_group(k.row0 + k.rows - 1));
        if (warp < kPtWarpS) {
            const int m = warp >> 2, rt = tid & (kPaRows - 1), r = two_rows ? m * p.tile_rows + rt : rt;   // tile; row of it and of the block
            const bool mine = rt < p.tile_rows && r < k.rows;
            const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = taddr + (uint32_t)(m * 128), to = taddr + (uint32_t)(C::kO + m * D);
            constexpr float kTau = PagedExp<kHalf>::kTau, kUp = PagedExp<kHalf>::kUp + (kScale > 1.f ? 20.f : 0.f);
            const float cs = p.scale * kScale;
            const int row = k.row0 + (mine ? r : 0), t = p.by_group(row), place = k.place0 + t;
            const int hi = mine ? min(place, k.have - 1) : -1, lo = mine ? paged_from(p, place) : 0;
            const int key0 = (t0 + (two_rows ? 0 : m)) * kPtKeys, step = two_rows ? kPtKeys : 2 * kPtKeys;
            float l = 0.f, m_ref = kPagedNone;
            bool far = false;                                          // a reference of this warp is beyond kPtFar
            for (int j = 0; j < 2 * count; ++j) {                      // 64 keys
                const int b = j & 1, base = key0 + (j >> 1) * step + b * kPtHalf, h = hi - base, from_ = lo - base;   // this row sees from_ .. h of them
                const uint32_t tb = ts + (uint32_t)(b * kPtHalf);
                if (!pt_wait(&s_full[m][b], (uint32_t)(turn + (j >> 1)) & 1u, s_abort, err, 0x5600 + m)) break;
                tc_fence_after();
                uint32_t raw[kPtHalf];
#pragma unroll
                for (int i = 0; i < kPtHalf; i += 32) pa_ld32(tb + i, raw + i);
                pa_wait_ld();
                if (!__all_sync(0xffffffffu, h >= kPtHalf - 1 && from_ <= 0)) {
                    const unsigned span = h >= from_ ? (unsigned)(h - from_) : 0u, from = h >= from_ ? (unsigned)from_ : 0x40000000u;
#pragma unroll
                    for (int i = 0; i < kPtHalf; ++i)
                        if ((unsigned)i - from > span) raw[i] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(raw[i]);
#pragma unroll
                for (int i = 4; i < kPtHalf - 4; i += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx[u] = pa_max3(mx[u], __uint_as_float(raw[i + 2 * u]), __uint_as_float(raw[i + 2 * u + 1]));
                mx[0] = pa_max3(mx[0], __uint_as_float(raw[kPtHalf - 4]), __uint_as_float(raw[kPtHalf - 3]));
                mx[1] = pa_max3(mx[1], __uint_as_float(raw[kPtHalf - 2]), __uint_as_float(raw[kPtHalf - 1]));
                const float m_tile = pa_max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * cs;
                const bool up = m_tile - m_ref > kTau;
                if (__any_sync(0xffffffffu, up | far)) {
                    const float f = up ? pa_exp2(m_ref - m_tile) : 1.f;
                    if (up) m_ref = m_tile;
                    l *= f;
                    if (j > 0 && __any_sync(0xffffffffu, up)) {
                        if (!tc2_wait(&o_done[m][b ^ 1], (uint32_t)(turn + ((j - 1) >> 1)) & 1u, s_abort, err, 0x5680 + m)) break;   // P V of the keys before
                        tc_fence_after();
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
                    far = __any_sync(0xffffffffu, fabsf(m_ref) >= kPtFar && m_ref != kPagedNone);
                }
                const uint64_t c2 = pa_two(cs, cs), m2 = pa_two(kUp - m_ref, kUp - m_ref);
                uint64_t sum[2] = {0, 0};
                if (far) l += pt_far<T>(tb, cs, m_ref, kUp, from_, h);
                else
#pragma unroll
                for (int part = 0; part < kPtHalf; part += 32) {
                    uint32_t x[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float a, e;
                        pa_split(pa_fma2(pa_two(__uint_as_float(raw[part + 2 * i]), __uint_as_float(raw[part + 2 * i + 1])), c2, m2), a, e);
                        a = pa_exp2(a);
                        e = pa_exp2(e);
                        sum[i & 1] = pa_add2(sum[i & 1], pa_two(a, e));
                        if constexpr (kHalf) {
                            const __half2 y = __floats2half2_rn(a, e);
                            x[i] = *reinterpret_cast<const uint32_t*>(&y);
                        } else {
                            const __nv_bfloat162 y = __floats2bfloat162_rn(a, e);
                            x[i] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                    }
                    tc_st16(tb + (uint32_t)(part / 2), x);
                }
                float s0, s1;
                pa_split(pa_add2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
                // Values of keys that not all rows see are looked over, and where the last visible key ends within a TMA box, those behind it become zeros (further boxes
                // are zeros already).  Of two row tiles the first sees to it, whose product comes first.  The tile is there or on its way: the ring's tiles before it
                // have been used.
                if (m == 0 || !two_rows) {
                    const int behind = min(k.hi + 1 - base, kPtHalf);   // rows that hold keys
                    const bool look = behind > 0 && (base + behind - 1 > all_hi || base < all_lo), cut = !INT4 && box && behind > 0 && behind % box != 0;
                    if (look || cut) {
                        const int it = ring + j * items + (two_rows ? 1 : 2 + m), slot = it % C::kRing;
                        if (!tc2_wait(&full[slot], (uint32_t)(it / C::kRing) & 1u, s_abort, err, 0x5800 + slot)) break;
                        const int r1 = cut ? (behind + box - 1) / box * box : behind;
                        bool broken = false;
#pragma unroll 1
                        for (int x = tid & (kPaRows - 1); x < r1 * CH; x += kPaRows) {   // whole rows: the swizzle stays within them
                            const int row = x / CH, ch = x % CH;
                            uint4* w = reinterpret_cast<uint4*>(smem + C::kRingOff + slot * C::kTile + (ch >> 3) * (kPtHalf * 128) + row * 128 + ((ch & 7) << 4));
                            if (row >= behind) *w = make_uint4(0, 0, 0, 0);
                            else if (base + row < all_lo || base + row > all_hi) broken |= pt_clean<T>(w);
                        }
                        if (broken) s_broken[blocks & 1] = blocks + 1;
                        pa_fence_async();
                    }
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[m][b]);
            }
            for (int b = 0; b < 2; ++b) tc2_wait(&o_done[m][b], (uint32_t)(turn + count - 1) & 1u, s_abort, err, 0x5700 + m);
            tc_fence_after();
            l /= kScale;
            // noted before the tile's probabilities were handed on, whose product has ended
            if (__any_sync(0xffffffffu, s_broken[blocks & 1] == blocks + 1))
                (INT4 ? pt_add_broken4<T, D> : pt_add_broken<T, D>)(c, k.seq, (long long)at.hk * c.head_stride, to, lo, hi, key0, min(t0 * kPtKeys + count * step - 1, k.hi), all_lo, all_hi, step / kPtKeys);
            if (!walk.whole(count)) {
                // A part: {maximum, sum}, then the output as it stands, column by column: the lanes of a warp are neighbours there.
                const size_t part = (size_t)blockIdx.x * 2 + (first > 0 ? 0 : 1);
                if (mine) p.ml[part * kPtRows + tid] = make_float2(m_ref, l);
                float* dst = p.part + part * kPtRows * D + tid;
                if (__any_sync(0xffffffffu, mine))
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += 32) {
                        uint32_t v[32];
                        pa_ld32(to + (uint32_t)d0, v);
                        pa_wait_ld();
                        if (mine)
#pragma unroll
                            for (int i = 0; i < 32; ++i) dst[(d0 + i) * kPtRows] = __uint_as_float(v[i]);
                    }
                if (tid == 0) walk.cut(p, first, count);
            } else {
                // Where the block's one tile has two results, the second goes to shared memory, where Q was, chunks of 16 bytes xor the row.
                float f_own = 1.f, f_other = 0.f;
                float4* other = reinterpret_cast<float4*>(smem) + rt * (D / 4);
                const int xr = rt & (D / 4 - 1);
                if (joins) {
                    if (m == 1) {
                        s_ml[rt] = make_float2(m_ref, l);
                        if (__any_sync(0xffffffffu, mine))
#pragma unroll 1
                        for (int d0 = 0; d0 < D; d0 += 32) {
                            uint32_t v[32];
                            pa_ld32(to + (uint32_t)d0, v);
                            pa_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(other + (((d0 + i) >> 2) ^ xr)) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        }
                    }
                    pa_fence_async();   // what Q's next copy writes over
                    asm volatile("bar.sync 3, 256;" ::: "memory");
                    if (m == 0) {
                        const float2 x = s_ml[rt];
                        const float top = fmaxf(m_ref, x.x);
                        f_own = pa_exp2(m_ref - top), f_other = pa_exp2(x.x - top);
                        l = fmaf(x.y, f_other, l * f_own);
                    }
                }
                if ((two_rows || m == 0) && __any_sync(0xffffffffu, mine)) {
                    const int head = at.hk * p.group + row - t * p.group;
                    T* dst = static_cast<T*>(p.out) + ((size_t)(k.first + t) * p.heads + head) * D;
                    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += 32) {
                        uint32_t v[32];
                        pa_ld32(to + (uint32_t)d0, v);
                        pa_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            float f[8];
#pragma unroll
                            for (int u = 0; u < 8; ++u) f[u] = __uint_as_float(v[i + u]);
                            if (joins)
#pragma unroll
                                for (int u = 0; u < 8; u += 4) {
                                    const float4 y = other[((d0 + i + u) >> 2) ^ xr];
                                    f[u] = fmaf(y.x, f_other, f[u] * f_own), f[u + 1] = fmaf(y.y, f_other, f[u + 1] * f_own);
                                    f[u + 2] = fmaf(y.z, f_other, f[u + 2] * f_own), f[u + 3] = fmaf(y.w, f_other, f[u + 3] * f_own);
                                }
#pragma unroll
                            for (int u = 0; u < 8; ++u) f[u] = l == 0.f ? 0.f : f[u] * inv;
                            if (mine) *reinterpret_cast<uint4*>(dst + d0 + i) = pack8<T>(f);
                        }
                    }
                }
            }
            tc_fence_before();   // the next block's products write where this one's results were read
            if (joins) pa_fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free);
            if (lane == 0 && joins && m == 0) mbar_arrive(&joined);
        } else if (warp == kPtWarpS) {
            if (tc_elect_one()) {
                constexpr uint32_t id = pa_idesc(!kHalf, kPtHalf, false);
                const uint64_t qd = tc_desc_sw128(smem_u32(smem));
                ok = ok && tc2_wait1(&q_full, (uint32_t)blocks & 1u, s_abort, err, 0x5000);
                // The scores of 64 keys come under the softmax of the 64 before; they lie over the probabilities of those before these, which P V has to have read.
                for (int j = 0; j < 2 * count && ok; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const int it = ring + j * items + (two_rows ? 0 : m), slot = it % C::kRing;
                        if (m == 0 || !two_rows) {
                            ok = ok && tc2_wait1(&full[slot], (uint32_t)(it / C::kRing) & 1u, s_abort, err, 0x5100 + slot);
                            if (!INT4 && !box) pa_fence_async();
                        }
                        if (turn + (j >> 1) > 0) ok = ok && tc2_wait1(&o_done[m][j & 1], (uint32_t)(turn + (j >> 1) - 1) & 1u, s_abort, err, 0x5400 + m);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t kd = tc_desc_sw128(smem_u32(smem + C::kRingOff + slot * C::kTile));
                        const uint64_t qm = qd + (uint64_t)((two_rows ? m : 0) * (C::kQ / 16));
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
                            pa_mma_ss(tmem + (uint32_t)(m * 128 + (j & 1) * kPtHalf), qm + (uint64_t)((i >> 2) * (kPaRows * 128 / 16) + (i & 3) * 2),
                                      kd + (uint64_t)((i >> 2) * (kPtHalf * 128 / 16) + (i & 3) * 2), id, i > 0 ? 1u : 0u);
                        tc_commit(&s_full[m][j & 1]);
                        if (m == 1 || !two_rows) tc_commit(&empty[slot]);
                    }
                tc_commit(&q_free);
            }
            __syncwarp();
        } else if (warp == kPtWarpO) {
            if (tc_elect_one()) {
                constexpr uint32_t id = pa_idesc(!kHalf, D, true);
                if (blocks > 0) ok = ok && tc2_wait1(&o_free, (uint32_t)(blocks - 1) & 1u, s_abort, err, 0x5080);   // the block before has been written
                for (int j = 0; j < 2 * count && ok; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const int it = ring + j * items + (two_rows ? 1 : 2 + m), slot = it % C::kRing;
                        if (m == 0 || !two_rows) {
                            ok = ok && tc2_wait1(&full[slot], (uint32_t)(it / C::kRing) & 1u, s_abort, err, 0x5200 + slot);
                            if (!INT4 && !box) pa_fence_async();
                        }
                        ok = ok && tc2_wait1(&p_full[m][j & 1], (uint32_t)(turn + (j >> 1)) & 1u, s_abort, err, 0x5300 + m);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t vd = pa_desc_mn(smem_u32(smem + C::kRingOff + slot * C::kTile), kPtHalf * 128);
#pragma unroll
                        for (int i = 0; i < kPtHalf / 16; ++i)
                            pa_mma_ts(tmem + (uint32_t)(C::kO + m * D), tmem + (uint32_t)(m * 128 + (j & 1) * kPtHalf + i * 8), vd + (uint64_t)(i * (16 * 128 / 16)), id,
                                      (j > 0 || i > 0) ? 1u : 0u);
                        tc_commit(&o_done[m][j & 1]);
                        if (m == 1 || !two_rows) tc_commit(&empty[slot]);
                    }
            }
            __syncwarp();
        } else if (warp >= kPtWarpLoad) {
            // first key of the ring's tile i of this block
            auto row_of = [&](int i) {
                const int j = two_rows ? i >> 1 : i >> 2;
                return (t0 + (two_rows ? j >> 1 : 2 * (j >> 1) + (i & 1))) * kPtKeys + (j & 1) * kPtHalf;
            };
            // Q, behind the first keys and values: the scores of the block before have been made, and its two results do not lie there any more
            auto load_q = [&]() {
                if (warp != kPtWarpLoad) return;
                if (blocks > 0) ok = ok && tc2_wait(&q_free, (uint32_t)(blocks - 1) & 1u, s_abort, err, 0x5900);
                if (was_joined) ok = ok && tc2_wait(&joined, (uint32_t)(joins_before - 1) & 1u, s_abort, err, 0x5980);
                if (lane == 0 && ok) {
                    const int tokens = p.by_group(p.tile_rows), t = k.first + p.by_group(k.row0);
                    mbar_expect_tx(&q_full, (two_rows ? 2 : 1) * C::kAtoms * p.tile_rows * 128);
                    for (int m = 0; m < (two_rows ? 2 : 1); ++m)
                        for (int a = 0; a < C::kAtoms; ++a)
                            pt_load_3d(smem_u32(smem) + (uint32_t)(m * C::kQ + a * (kPaRows * 128)), &q_map, a * 64, at.hk * p.group, t + m * tokens, &q_full);
                }
                __syncwarp();
            };
            if constexpr (INT4) {
                constexpr int kChunk = D / 8, kEach = 5 * kPtHalf / 32;
                const int tiles = count * items, pitch = int4_pitch<D>(box), skip = int4_skip<D>(box, at.hk);   // of keys, and as many of values
                if (warp < kPtWarpLoad4) {
                    // A lane looks up rows lane and lane + 32 of the tile, a tile ahead, and copies ten of its 320 chunks
                    const int is_v = warp - kPtWarpLoad;
                    const uint8_t* from = static_cast<const uint8_t*>(is_v ? c.v : c.k) + (long long)at.hk * c.head_stride;
                    auto first_row = [&](int n) { return row_of(two_rows ? 2 * n + is_v : (n >> 1) * 4 + 2 * is_v + (n & 1)); };
                    int ids[2];
                    auto ask = [&](int n) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int row = first_row(n) + (box ? (lane & 3) * 16 : u * 32 + lane), pg = c.by_page(row);
                            ids[u] = n < tiles && row <= k.hi && pg < c.max_pages ? c.table[(size_t)k.seq * c.ld_table + pg] : -1;
                        }
                    };
                    ask(0);
                    for (int n = 0; n < tiles && ok; ++n) {
                        if (n == 1) load_q();
                        const int it = ring / 2 + n, slot = it % C::kRaw;
                        if (box) {   // four boxes of 16 rows, a lane each
                            const int id = ids[0] >= 0 && ids[0] < c.num_pages ? ids[0] : -1, row = first_row(n) + (lane & 3) * 16;   // -1: reads as zeros
                            ask(n + 1);
                            if (it >= C::kRaw) ok = ok && pt_wait(&raw_empty[is_v][slot], (uint32_t)(it / C::kRaw - 1) & 1u, s_abort, err, 0x5a00 + is_v);
                            if (!ok) break;
                            if (lane == 0) mbar_expect_tx(&raw_full[is_v][slot], kPtHalf * pitch);
                            __syncwarp();
                            if (lane < 4)
                                int4_box<D>(smem_u32(smem) + (uint32_t)(C::kRawOff + (is_v * C::kRaw + slot) * C::kCodes + lane * 16 * pitch), is_v ? &v_map : &k_map, box, at.hk,
                                            row - c.by_page(row) * c.page_size, id, &raw_full[is_v][slot]);
                            continue;
                        }
                        long long offs[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int row = first_row(n) + u * 32 + lane;
                            offs[u] = ids[u] >= 0 && ids[u] < c.num_pages ? (long long)ids[u] * c.page_stride + (long long)(row - c.by_page(row) * c.page_size) * c.row_stride : -1;
                        }
                        ask(n + 1);
                        if (it >= C::kRaw) ok = ok && pt_wait(&raw_empty[is_v][slot], (uint32_t)(it / C::kRaw - 1) & 1u, s_abort, err, 0x5a00 + is_v);
                        if (!ok) break;
                        const uint32_t to = smem_u32(smem) + (uint32_t)(C::kRawOff + (is_v * C::kRaw + slot) * C::kCodes);
#pragma unroll 1
                        for (int u = 0; u < kEach; ++u) {
                            const int x = lane + 32 * u, r = x / 5, ch = x - r * 5;
                            const long long low = __shfl_sync(0xffffffffu, offs[0], r & 31), high = __shfl_sync(0xffffffffu, offs[1], r & 31), off = r < 32 ? low : high;
                            const uint8_t* src = from + (off < 0 ? 0 : off + ch * kChunk);
                            if constexpr (D == 128) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + x * kChunk), "l"(src), "r"(off < 0 ? 0 : 16) : "memory");
                            else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to + x * kChunk), "l"(src), "r"(off < 0 ? 0 : 8) : "memory");
                        }
                        pa_landed(&raw_full[is_v][slot]);
                    }
                } else {
                    // Two tiles at a time: lane = row, half of the warp a group of 32 columns each.  Reads of eight rows touch all banks once, and so do writes of 16 bytes of
                    // eight rows.  One fence for both: it waits for the writes.
                    const int rg = warp - kPtWarpLoad4, row = rg * 16 + (lane & 15);
                    // Loops that are not unrolled: the warps' instructions come from one small cache, and what is large here stops the softmax's (at a time unrolled 442 us, as it stands 309).
                    for (int x = 0; x < tiles && ok; ++x) {
                        const int is_v = two_rows ? 0 : x & 1, n = ring / 2 + (two_rows ? x : (x >> 1) * 2), i = ring + 2 * x;   // of the first of the two
#pragma unroll 1
                        for (int t = 0; t < 2; ++t) {
                            const int v = two_rows ? t : is_v, it = two_rows ? n : n + t, raw = it % C::kRaw, slot = (i + t) % C::kRing;
                            ok = ok && pt_wait(&raw_full[v][raw], (uint32_t)(it / C::kRaw) & 1u, s_abort, err, 0x5b00 + v);
                            if (i + t >= C::kRing) ok = ok && pt_wait(&empty[slot], (uint32_t)((i + t) / C::kRing - 1) & 1u, s_abort, err, 0x5500 + slot);
                            if (!ok) break;
                            const uint8_t* from = smem + C::kRawOff + (v * C::kRaw + raw) * C::kCodes + row * pitch + skip;
                            uint8_t* to = smem + C::kRingOff + slot * C::kTile + row * 128;
                            const int first = row_of(2 * x + t);
#pragma unroll
                            for (int u = 0; u < D / 64; ++u) {
                                const int g = 2 * u + (lane >> 4);
                                uint32_t w[4];
                                if constexpr (D == 128) {
                                    const uint4 y = *reinterpret_cast<const uint4*>(from + g * 16);
                                    w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
                                } else {
                                    const uint2 y = *reinterpret_cast<const uint2*>(from + g * 16), z = *reinterpret_cast<const uint2*>(from + g * 16 + 8);
                                    w[0] = y.x, w[1] = y.y, w[2] = z.x, w[3] = z.y;
                                }
                                const uint32_t pair = *reinterpret_cast<const uint32_t*>(from + D / 2 + g * 4);
                                const uint32_t stored = first + row > k.hi ? 0u : pair;   // what a page holds behind the last key may be anything
                                auto write = [&](auto codes, uint32_t track) {
                                    const uint32_t two = decltype(codes)::pair(stored, track);
                                    codes.set(__byte_perm(two, 0, 0x1010), __byte_perm(two, 0, 0x3232));
#pragma unroll
                                    for (int y = 0; y < 4; ++y)
                                        *reinterpret_cast<uint4*>(to + u * (kPtHalf * 128) + ((((lane >> 4) * 4 + y) ^ (row & 7)) << 4)) = codes.eight(w[y]);
                                    return decltype(codes)::served(track);
                                };
                                const bool served = write(Int4Codes<T, false>{}, 0u);
                                if constexpr (kScale > 1.f)
                                    if (__any_sync(0xffffffffu, !served)) write(Int4Codes<T, true>{}, 0u);
                            }
                        }
                        if (!ok) break;
                        pa_fence_async();
                        __syncwarp();
                        if (lane == 0) {
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                mbar_arrive(&raw_empty[two_rows ? t : is_v][(two_rows ? n : n + t) % C::kRaw]), mbar_arrive(&full[(i + t) % C::kRing]);
                        }
                    }
                }
            } else if (box) {
                // One warp for keys, one for values; a lane for each box of a tile, its rows and 64 columns.  The lanes hold the numbers of 32 pages in
                // a row, which is a turn's keys at least.
                const bool is_v = warp != kPtWarpLoad;
                const int boxes = kPtHalf / box, b_row = lane % boxes * box, last_page = min(c.by_page(max(k.hi, 0)), c.max_pages - 1);
                int page0 = -32, ids = -1;
                for (int j = 0; j < 2 * count && ok; ++j) {
                    if (j == 1) load_q();
                    for (int m = 0; m < (two_rows ? 1 : 2); ++m) {
                        const int i = j * items + (two_rows ? (is_v ? 1 : 0) : (is_v ? 2 : 0) + m), it = ring + i, slot = it % C::kRing;
                        const int row0 = row_of(i), row = row0 + b_row, pg = c.by_page(row);
                        // those of a whole turn, whose tiles are not in the order of their keys
                        if (m == 0 && !(j & 1) && c.by_page(row0 + (two_rows ? kPtKeys : 2 * kPtKeys) - 1) >= page0 + 32) {
                            page0 = c.by_page(row0);
                            ids = page0 + lane <= last_page ? c.table[(size_t)k.seq * c.ld_table + page0 + lane] : -1;
                        }
                        int id = __shfl_sync(0xffffffffu, ids, pg - page0);
                        if (row > k.hi || id < 0 || id >= c.num_pages) id = -1;   // outside of the tensor: reads as zeros
                        if (it >= C::kRing) ok = ok && tc2_wait(&empty[slot], (uint32_t)(it / C::kRing - 1) & 1u, s_abort, err, 0x5500 + slot);
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(&full[slot], C::kTile);
                        __syncwarp();
                        for (int b = lane; b < boxes * C::kAtoms; b += 32)
                            pt_load_4d(smem_u32(smem + C::kRingOff + slot * C::kTile) + (uint32_t)(b / boxes * (kPtHalf * 128) + b_row * 128), is_v ? &v_map : &k_map,
                                       b / boxes * 64, row - pg * c.page_size, at.hk, id, &full[slot]);
                    }
                }
            } else {
                // Two rows (four of 64 columns) a copy of a warp.  A lane looks up every 32nd row of the 64 keys, once for K and V, and asks for the next ones'
                // page numbers before it copies these.
                const int ch = lane % CH, tiles = two_rows ? 1 : 2;
                constexpr int kRowsAtOnce = 32 / CH;
                int ids[2][kPtHalf / 32];
                auto ask = [&](int j) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int u = 0; u < kPtHalf / 32; ++u) {
                            const int row = row_of(j * items + m) + u * 32 + lane, pg = c.by_page(row);
                            ids[m][u] = m < tiles && j < 2 * count && row <= k.hi && pg < c.max_pages ? c.table[(size_t)k.seq * c.ld_table + pg] : -1;
                        }
                };
                ask(0);
                for (int j = 0; j < 2 * count && ok; ++j) {
                    if (j == 1) load_q();
                    long long offs[2][kPtHalf / 32];
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int u = 0; u < kPtHalf / 32; ++u) {
                            const int row = row_of(j * items + m) + u * 32 + lane, id = ids[m][u];
                            offs[m][u] = id >= 0 && id < c.num_pages ? (long long)id * c.page_stride + (long long)(row - c.by_page(row) * c.page_size) * c.row_stride : -1;
                        }
                    ask(j + 1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i >= items) break;
                        const int it = ring + j * items + i, slot = it % C::kRing;
                        const bool is_v = two_rows ? i & 1 : i & 2;
                        if (it >= C::kRing) ok = ok && tc2_wait(&empty[slot], (uint32_t)(it / C::kRing - 1) & 1u, s_abort, err, 0x5500 + slot);
                        if (!ok) break;
                        const T* from = static_cast<const T*>(is_v ? c.v : c.k) + (long long)at.hk * c.head_stride + ch * 8;
                        const uint32_t to = smem_u32(smem) + (uint32_t)(C::kRingOff + slot * C::kTile + (ch >> 3) * (kPtHalf * 128));
#pragma unroll
                        for (int u = 0; u < kPtHalf / 32; ++u) {
                            const long long mine = two_rows || !(i & 1) ? offs[0][u] : offs[1][u];
#pragma unroll 4
                            for (int x = (warp - kPtWarpLoad) * kRowsAtOnce; x < 32; x += 2 * kRowsAtOnce) {
                                const int r = x + lane / CH;
                                const long long off = __shfl_sync(0xffffffffu, mine, r);
                                pa_cp16(to + (uint32_t)((u * 32 + r) * 128 + (((ch & 7) ^ (r & 7)) << 4)), from + (off < 0 ? 0 : off), off >= 0);
                            }
                        }
                        pa_landed(&full[slot]);
                    }
                }
            }
        }
        was_joined = joins, joins_before += joins;
        turn += count, ring += 2 * count * items, ++blocks;
    }
    if (!box && warp >= kPtWarpLoad) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    tc2_drain(s_abort);
    tc_fence_before();
    __syncthreads();
    if (warp == kPtWarpS) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
    }
}

// Q: 64 columns of the heads of a group, whole tokens of a tile
template <int D>
inline bool pt_q_map(CUtensorMap* map, const PagedAttn& p, CUtensorMapDataType dt) {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.heads, (uint64_t)p.rows}, strides[2] = {D * 2, (uint64_t)p.heads * D * 2};
    const uint32_t rows[3] = {64, (uint32_t)p.group, (uint32_t)(p.tile_rows / p.group)};
    return tc_make_map_nd(map, p.q, dt, 3, dims, strides, rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Blocks that were cut: grid (the CTAs of k_paged_attn_tiles, groups of 32 rows), lane = row, a warp for D / 8 columns.  The first part of a block lies in its
// CTA's place 1, the others in the place 0 of theirs.  Of a block with two tiles of rows the second begins at row 128 of its place; one with a single tile has
// two results in a place, the second there.
template <typename T, int D>
__global__ void __launch_bounds__(256, 1) k_paged_join_tiles(const PagedAttn p) {
    constexpr int W = D / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d0 = warp * W;
    pdl_trigger();
    pdl_wait();
    const PagedCut x = p.cuts[blockIdx.x];
    const int r0 = blockIdx.y * 32, r = r0 + lane;
    if (x.parts == 0 || r0 >= x.k.rows) return;
    const bool twice = x.k.rows <= p.tile_rows, mine = r < x.k.rows;
    const int row = r >= p.tile_rows ? r - p.tile_rows + kPaRows : r;   // not more than 255
    float m = -INFINITY, l = 0.f, v[W] = {};
    // As the softmax goes, from part to part, the loads of two at once: for which the compiler takes the registers (79) only where the bounds name a single CTA (one token
    // of 64 heads on one over 30000 keys, a block in 148 parts: 76 us a call, 201 with 48 registers).
    const int parts = twice ? 2 * x.parts : x.parts;
    auto take = [&](auto count, int s0) {
        constexpr int N = decltype(count)::value;
        float2 y[N];
        float z[N][W];
#pragma unroll
        for (int h = 0; h < N; ++h) {
            const int s = s0 + h, i = twice ? s >> 1 : s;
            const size_t part = (size_t)(blockIdx.x + i) * 2 + (i == 0);
            const int at = min(row + (twice && (s & 1) ? kPaRows : 0), kPtRows - 1);
            y[h] = p.ml[part * kPtRows + at];
#pragma unroll
            for (int u = 0; u < W; ++u) z[h][u] = p.part[(part * D + d0 + u) * kPtRows + at];
        }
#pragma unroll
        for (int h = 0; h < N; ++h) {
            const float up = fmaxf(m, y[h].x), f = pa_exp2(m - up), g = pa_exp2(y[h].x - up);
            m = up;
            l = fmaf(y[h].y, g, l * f);
#pragma unroll
            for (int u = 0; u < W; ++u) v[u] = fmaf(z[h][u], g, v[u] * f);
        }
    };
    int s0 = 0;
    for (; s0 + 2 <= parts; s0 += 2) take(std::integral_constant<int, 2>{}, s0);
    if (s0 < parts) take(std::integral_constant<int, 1>{}, s0);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) v[u] = l == 0.f ? 0.f : v[u] * inv;
    const int at = x.k.row0 + (mine ? r : 0), t = p.by_group(at), head = x.hk * p.group + at - t * p.group;
    if (mine) {
        T* dst = static_cast<T*>(p.out) + ((size_t)(x.k.first + t) * p.heads + head) * D + d0;
#pragma unroll
        for (int u = 0; u < W; u += 8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[u + i];
            *reinterpret_cast<uint4*>(dst + u) = pack8<T>(f);
        }
    }
}

}  // namespace zl
