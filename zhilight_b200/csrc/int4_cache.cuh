// Rows of a key / value cache that is held in 4 bits.  A head's row: dim / 2 bytes of codes, then for every 32 columns a pair (step, lowest value) in the type
// T of the rows that it was written from, 5 dim / 8 bytes in all.  A code c stands for T(lowest + step * c), rounded once.
//
// Of a group with lowest and highest value lo and hi, the step is (hi - lo) / 15 rounded down to T, so that no code stands for more than hi, and x becomes
// the nearest whole number of steps above lo, at most 15 (ties to even).  What is read is off by half a step; at the upper end by what the step's rounding leaves too, up to 15 units
// of T at the step (15 eps(T) of it; of fp16 steps below 2^-14, which are multiples of 2^-24, more: ranges below 15 * 2^-24 have a step of zero); and by its own rounding to T, half a
// unit of the value, which may be the largest part: bf16 values of 3 +- 0.15 are off by up to 0.94 steps.  lo
// is one of the values, so T holds it as it is.  Differences are taken of halves: a range may be beyond the largest 32-bit number.  A step below the normal
// 32-bit numbers counts as none.  A group with an infinity or NaN reads as NaN.
//
// 32 bits hold 8 columns, columns 0 2 4 6 in the lower half and 1 3 5 7 in the upper one: one `and` and one `or` with the bits of 2^10 (fp16, whose step is 1 there)
// or 2^7 (bf16) make two neighbouring columns' codes numbers of T, off by that power, which a subtraction takes away exactly.
#pragma once
#include "common.cuh"

#include <type_traits>

namespace zl {

constexpr int kInt4Group = 32;
constexpr int int4_row_bytes(int dim) { return dim / 8 * 5; }

// How 16 rows of a head of a 4-bit cache come to shared memory, and lie there.  Heads of 128: as a box of whole rows of 80 bytes.  Heads of 64, whose 40 bytes are no multiple of 16: as
// one piece where they lie behind one another (kRun), else 48 bytes of each row, from the 16-byte border at or before it, where a row has its heads behind one another (kWide).
// None of these, or pages that do not hold whole 16s: by copies of D / 8 bytes.
enum { kInt4Copies, kInt4Run, kInt4Wide };
template <int D>
constexpr int kInt4Pitch = D == 128 ? 80 : 48;   // most
template <int D>
__device__ __forceinline__ int int4_pitch(int form) { return D == 128 ? 80 : form == kInt4Wide ? 48 : 40; }
template <int D>
__device__ __forceinline__ int int4_skip(int form, int hk) { return D == 64 && form == kInt4Wide ? (hk & 1) * 8 : 0; }
template <typename T>
struct Int4Pair {
    using type = __half2;
};
template <>
struct Int4Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
};

// (step, step) and (lowest, lowest) of a group
template <typename T>
__device__ __forceinline__ void int4_meta(uint32_t meta, uint32_t& step, uint32_t& low) {
    step = __byte_perm(meta, 0, 0x1010);
    low = __byte_perm(meta, 0, 0x3232);
}
// Two values from the codes at bits 4 J .. of both halves of x, whose steps and lowest values stand in the halves of step and low
template <typename T, int J>
__device__ __forceinline__ uint32_t int4_two(uint32_t x, uint32_t step, uint32_t low) {
    using P = typename Int4Pair<T>::type;
    P c;
    if constexpr (std::is_same<T, __half>::value) {
        if constexpr (J & 1) {   // 16 c + 2^10, without a shift
            const uint32_t w = lop3_and_or<0x00f000f0u, 0x64006400u>(J & 2 ? x >> 8 : x);
            c = __hfma2(*reinterpret_cast<const P*>(&w), __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd400)));   // 1 / 16, -64
        } else {
            const uint32_t w = lop3_and_or<0x000f000fu, 0x64006400u>(J & 2 ? x >> 8 : x);
            c = __hsub2(*reinterpret_cast<const P*>(&w), __half2half2(__ushort_as_half(0x6400)));
        }
    } else {
        const uint32_t w = lop3_and_or<0x000f000fu, 0x43004300u>(x >> (4 * J));
        c = __hsub2(*reinterpret_cast<const P*>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0x4300)));
    }
    const P y = __hfma2(c, *reinterpret_cast<const P*>(&step), *reinterpret_cast<const P*>(&low));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// 8 neighbouring columns
template <typename T>
__device__ __forceinline__ uint4 int4_eight(uint32_t x, uint32_t step, uint32_t low) {
    return make_uint4(int4_two<T, 0>(x, step, low), int4_two<T, 1>(x, step, low), int4_two<T, 2>(x, step, low), int4_two<T, 3>(x, step, low));
}
// whether a group's pair is one of numbers
template <typename T>
__device__ __forceinline__ bool int4_finite(uint32_t meta) {
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80;
    return (meta & 0x7fffu) < kInf && (meta >> 16 & 0x7fffu) < kInf;
}

// Codes as numbers.  fp16: exactly what they stand for.  bf16: that times 2^-20, from a multiplication and a sum that are rounded together, like those of int4_two.  A code
// at bits 0 - 3 or 4 - 7 is, taken as a bf16 number, c * 2^-133 or 16 c * 2^-133 (also where it reaches the exponent's lowest bit), so the step is multiplied by 2^113 and
// the lowest value by 2^-20 beforehand.  That overflows for steps from 2^15 on; whoever calls keeps the largest pair in sight (track) and goes over such keys with SLOW.
template <typename T, bool SLOW>
struct Int4Codes {
    static constexpr bool kScaled = std::is_same<T, __nv_bfloat16>::value;
    static constexpr float kScale = kScaled ? 1048576.f : 1.f;       // what the numbers are to be multiplied by
    // pairs (step, lowest) of two groups in, steps and lowest values as operands out: a step for codes at bits 0 - 3 and one for those at bits 4 - 7
    uint32_t step, step16, low;
    __device__ __forceinline__ void set(uint32_t s, uint32_t l) {
        step = s, low = l;
        if constexpr (kScaled && !SLOW) step16 = times(s, 0x3d803d80u);   // 1 / 16
    }
    static __device__ __forceinline__ uint32_t times(uint32_t x, uint32_t y) {
        using P = typename Int4Pair<T>::type;
        const P z = __hmul2(*reinterpret_cast<const P*>(&x), *reinterpret_cast<const P*>(&y));
        return *reinterpret_cast<const uint32_t*>(&z);
    }
    // a pair (step, lowest) as it is stored
    static __device__ __forceinline__ uint32_t pair(uint32_t meta, uint32_t& track) {
        if constexpr (kScaled && !SLOW) {
            meta = times(meta, 0x35807800u);                              // 2^113 below, 2^-20 above
            const __nv_bfloat162 x = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&meta)), *reinterpret_cast<const __nv_bfloat162*>(&track));
            track = *reinterpret_cast<const uint32_t*>(&x);
        }
        return meta;
    }
    static __device__ __forceinline__ bool served(uint32_t track) { return (track & 0x7fffu) < 0x7f80u && (track >> 16 & 0x7fffu) < 0x7f80u; }
    template <int J>
    __device__ __forceinline__ uint32_t two(uint32_t x) const {
        if constexpr (!kScaled) {
            return int4_two<T, J>(x, step, low);
        } else if constexpr (SLOW) {
            return times(int4_two<T, J>(x, step, low), 0x35803580u);
        } else {
            const uint32_t c = (J & 2 ? x >> 8 : x) & (J & 1 ? 0x00f000f0u : 0x000f000fu);
            const __nv_bfloat162 y = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&c), *reinterpret_cast<const __nv_bfloat162*>(J & 1 ? &step16 : &step),
                                             *reinterpret_cast<const __nv_bfloat162*>(&low));
            return *reinterpret_cast<const uint32_t*>(&y);
        }
    }
    __device__ __forceinline__ uint4 eight(uint32_t x) const { return make_uint4(two<0>(x), two<1>(x), two<2>(x), two<3>(x)); }   // neighbouring columns
};

template <typename T>
__device__ __forceinline__ T int4_round_down(float x);
template <>
__device__ __forceinline__ __half int4_round_down<__half>(float x) { return __float2half_rz(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 int4_round_down<__nv_bfloat16>(float x) { return __float2bfloat16_rz(x); }

// the number above one that is at least zero
__device__ __forceinline__ __half int4_next(__half x) { return __ushort_as_half((unsigned short)(__half_as_ushort(x) + 1)); }
__device__ __forceinline__ __nv_bfloat16 int4_next(__nv_bfloat16 x) { return __ushort_as_bfloat16((unsigned short)(__bfloat16_as_ushort(x) + 1)); }

// 8 columns of a group whose other columns are in the neighbouring lanes of this group of four; all lanes of the warp call it.  -> the codes; the group's pair
template <typename T>
__device__ __forceinline__ uint32_t int4_encode(const uint4& x, uint32_t& meta) {
    using P = typename Int4Pair<T>::type;
    constexpr unsigned kAll = 0xffffffffu;
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80, kAbs = 0x7fff7fffu;
    const uint32_t size = __vmaxu2(__vmaxu2(x.x & kAbs, x.y & kAbs), __vmaxu2(x.z & kAbs, x.w & kAbs));
    const unsigned numbers = __ballot_sync(kAll, (size & 0xffffu) < kInf && size >> 16 < kInf) >> (threadIdx.x & 28) & 15u;
    // the highest value and the lowest one's opposite, in T
    const P* two = reinterpret_cast<const P*>(&x);
    const P high = __hmax2(__hmax2(two[0], two[1]), __hmax2(two[2], two[3])), less = __hmin2(__hmin2(two[0], two[1]), __hmin2(two[2], two[3]));
    const uint32_t h = *reinterpret_cast<const uint32_t*>(&high), l = *reinterpret_cast<const uint32_t*>(&less) ^ 0x80008000u, a = __byte_perm(h, l, 0x5410), b = __byte_perm(h, l, 0x7632);
    P ends = __hmax2(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const uint32_t other = __shfl_xor_sync(kAll, *reinterpret_cast<const uint32_t*>(&ends), o);
        ends = __hmax2(ends, *reinterpret_cast<const P*>(&other));
    }
    const T* of = reinterpret_cast<const T*>(&ends);
    const float half = -0.5f * to_f32<T>(of[1]);   // of the lowest
    // The step: the largest number of T that 7.5 times is at most half the range, all exactly: 32 bits hold 7.5 times a number of T, and rounding the range towards zero moves it
    // past none of them.  A product with 1 / 7.5, both rounded down, gives that number or the one below it.
    const float part = __fmaf_rz(to_f32<T>(of[0]), 0.5f, -half);
    T pair[2] = {int4_round_down<T>(__fmul_rz(part, 0x1.111110p-3f)), from_f32<T>(half * 2.f)};
    const T next = int4_next(pair[0]);
    if (__fmul_rn(to_f32<T>(next), 7.5f) <= part) pair[0] = next;
    meta = numbers == 15u ? *reinterpret_cast<const uint32_t*>(pair) : 0x7fff7fffu;
    const float step = to_f32<T>(pair[0]);
    if (numbers != 15u || !(step >= 1.17549435e-38f)) return 0;
    float f[8];
    unpack8<T>(x, f);
    uint32_t codes = 0;
    // half of x - lo, of which 32 bits may not hold all: what is lost leaves the last bit set, so that a difference beside the border between two codes, (c + 1/2) step, which
    // has 16 bits, does not become it
    auto above = [&](float x) {
        const uint32_t down = __float_as_uint(__fmaf_rz(x, 0.5f, -half)), up = __float_as_uint(__fmaf_ru(x, 0.5f, -half));   // the same number or neighbours
        return __uint_as_float(down | ((down ^ up) & 1u));
    };
    if (step >= 1e-30f) {
        // Quotients by the reciprocal and one correction of what is left over (Markstein 1990), a quarter of a division's instructions: rounded once.  One on the border between two
        // codes comes out exactly, and one beside it does not come out as the border: it is more than half a unit of 32 bits away from it.  Codes are whole numbers at the
        // end of 1.5 * 2^23 + c, each multiplied into its place; what that number adds there is taken away beforehand.
        const float inv = __fdiv_rn(1.f, step);
        constexpr uint32_t kWhole = 0x4b400000u;
        codes = 0u - kWhole * 0x11111111u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = above(f[i]);
            float q = __fmul_rn(d, inv);
            q = __fmaf_rn(__fmaf_rn(-q, step, d), inv, q);
            codes += __float_as_uint(__fmaf_rn(fminf(q, 7.5f), 2.f, 12582912.f)) << ((i & 1) * 16 + (i & 6) * 2);
        }
    } else {   // far down those products would lose bits
#pragma unroll 1
        for (int i = 0; i < 8; ++i) codes |= (uint32_t)__float2int_rn(fminf(2.f * __fdiv_rn(above(f[i]), step), 15.f)) << ((i & 1) * 16 + (i & 6) * 2);
    }
    return codes;
}

}  // namespace zl
