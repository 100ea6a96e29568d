// A paged key / value cache as the kernels see it: pages of page_size rows of all kv heads, and for every sequence a row of page numbers.  Rows and
// heads of a page lie anywhere (strides in elements), so both orders of a page are served.  A page number outside the pool is never followed: such
// rows read as zeros and take no writes.  Entries of the table behind a sequence's last row are not looked at.
#pragma once
#include "common.cuh"

namespace zl {

// i / d for 0 <= i < 2^31 by a multiplication (Granlund and Montgomery 1994): with 2^s >= d and mul = ceil(2^(31 + s) / d), which fits 32 bits
// because d > 2^(s - 1), the error mul * d - 2^(31 + s) is below d <= 2^s, and i times it below 2^(31 + s).
struct PagedDivisor {
    uint32_t mul;
    int shift;
    __host__ __device__ __forceinline__ int operator()(int i) const { return (int)((uint64_t)(uint32_t)i * mul >> shift); }
};
inline PagedDivisor paged_divisor(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}

struct PagedCache {
    void *k, *v;
    long long num_pages, page_stride, row_stride, head_stride;   // elements
    const int32_t* table;
    int ld_table, max_pages, page_size, seqs;
    PagedDivisor by_page;
    int limit;   // rows of a sequence, where its last page has more than there are; 0: whole pages
    // element offset of row i >= 0 of sequence b, -1: nowhere
    __device__ __forceinline__ long long row_at(int b, int i) const {
        const int pg = by_page(i);
        if (pg >= max_pages) return -1;
        const int id = table[(size_t)b * ld_table + pg];
        if (id < 0 || id >= num_pages) return -1;
        return (long long)id * page_stride + (long long)(i - pg * page_size) * row_stride;
    }
    // rows that the table has room for, as far as tiles of them are counted in 32 bits
    __device__ __forceinline__ int room() const { return limit ? limit : (int)min((long long)max_pages * page_size, 0x7fff0000ll); }
};

}  // namespace zl

// of an entry point's arguments
#define ZL_CHECK_PAGED(k, v, num_pages, page_size, page_stride, row_stride, head_stride, table, ld_table, max_pages, seqs)                        \
    ZL_CHECK_ARG((k) && (v) && (table) && (num_pages) > 0 && (page_size) > 0 && (max_pages) > 0 && (ld_table) >= (max_pages) && (seqs) > 0);       \
    ZL_CHECK_ARG((page_stride) >= 0 && (row_stride) >= 0 && (head_stride) >= 0);                                                                   \
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0);                                             \
    ZL_CHECK_SUPPORTED((page_stride) % 8 == 0 && (row_stride) % 8 == 0 && (head_stride) % 8 == 0)
// of a cache of 4 bits, strides in bytes: a chunk of a row is dim / 8 bytes, which the kernels copy at once
#define ZL_CHECK_PAGED_INT4(k, v, num_pages, page_size, page_stride, row_stride, head_stride, dim)                                                \
    ZL_CHECK_ARG((k) && (v) && (num_pages) > 0 && (page_size) > 0 && (page_stride) >= 0 && (row_stride) >= 0 && (head_stride) >= 0);               \
    ZL_CHECK_SUPPORTED((dim) == 64 || (dim) == 128);                                                                                               \
    ZL_CHECK_SUPPORTED(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & ((dim) / 8 - 1)) == 0);                                \
    ZL_CHECK_SUPPORTED((page_stride) % ((dim) / 8) == 0 && (row_stride) % ((dim) / 8) == 0 && (head_stride) % ((dim) / 8) == 0)
