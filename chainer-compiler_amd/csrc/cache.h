// A cache of keys and values in pages, as cache.hip and attention.hip take it.
#pragma once

#include "chx_internal.h"

namespace chx {

// Division of numbers below 2^31 by one that the host knows: n / d = (floor(n mul / 2^32) + n) >> shift with 2^(shift - 1) < d <= 2^shift and mul = floor(2^32 (2^shift - d) / d) + 1.  (A few
// instructions, also scalar ones; a division by a number of 32 bits is some 20 to 40 of the vector units'.)
struct Divisor {
    uint32_t mul;
    int32_t shift;
};
inline Divisor divisor_of(int32_t d) {
    Divisor r = {1, 0};
    while ((int64_t(1) << r.shift) < d) ++r.shift;
    if (d > 0) r.mul = (uint32_t)((((uint64_t(1) << r.shift) - (uint64_t)d) << 32) / (uint64_t)d + 1);
    return r;
}
__device__ __forceinline__ int32_t over(int32_t n, Divisor d) {
    return (int32_t)((__umulhi((uint32_t)n, d.mul) + (uint32_t)n) >> d.shift);
}

struct CacheArgs {
    char *k, *v;
    int64_t k_page, k_row, k_head, v_page, v_row, v_head;  // bytes
    const int32_t* tables;
    int64_t table_row;  // elements
    const int32_t* lengths;
    int32_t B, groups, D, pages, page_rows;
    Divisor by_page;  // rows of a page
    int32_t places;  // of a sequence: of its table
};

// Checks keys and values [pages, rows of a page, heads, elements], tables [B, pages of a sequence] and lengths [B], and describes them.
int check_cache(const chx_hip_tensor* keys, const chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, const char* what, CacheArgs* c);

// Whole elements at addresses that are multiples of them; the last axis without gaps.
int check_rows(const chx_hip_tensor* t, int ndim, int32_t dtype, const char* what, const char* name);

// Bytes from one index of an axis to the next; 0 where there is no next.
inline int64_t stride_of(const chx_hip_tensor& t, int axis) {
    return t.shape[axis] > 1 ? t.strides[axis] : 0;
}

// int32, contiguous, of these extents (-1: any).
int check_numbers(const chx_hip_tensor* t, int ndim, int64_t n0, int64_t n1, const char* what, const char* name);

// float32 [B, heads, places or more] with elements next to each other along the last axis.
int check_mass(const chx_hip_tensor* mass, const CacheArgs& c, const char* what);

// Refuses a result or an updated array that meets another array (a null one, or one without elements, meets none): one whose first to last byte meet its own, unless both have the same shape and
// strides and lie between each other's rows.
struct Named {
    const chx_hip_tensor* t;
    const char* name;
};
int check_apart(const Named& written, const Named* others, int count, const char* what);

// Where place p of sequence b lies; page < 0: nowhere.
struct Place {
    int32_t page, row;
};
template <typename Args>
__device__ __forceinline__ Place place_of(const Args& a, int32_t b, int32_t p) {
    const int32_t i = over(p, a.by_page), page = a.tables[b * a.table_row + i];
    return {page < a.pages ? page : -1, p - i * a.page_rows};
}

}  // namespace chx
