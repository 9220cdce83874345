// Attention over a cache of pages or over arrays of states: what attention.hip checks and chooses, and the kernels take (attention_kernel.h).
#pragma once

#include "cache.h"

namespace chx {

enum AttentionKind { kCross, kChain, kTree };  // which places a row sees: the sequence's; those and the drafted rows up to its own; those, its ancestors and itself

constexpr int32_t kMostNodes = 256;   // of a tree
constexpr int32_t kMostParts = 64;    // that a sequence's places are split into: a wavefront joins them, one to a lane
constexpr int32_t kMostSize = 256;    // elements of a head

struct AttentionArgs {
    const char *q, *k, *v;
    char* y;
    // bytes
    int64_t q_batch, q_token, q_head, y_batch, y_token, y_head;
    int64_t k_page, k_row, k_head, v_page, v_row, v_head;
    const int32_t* tables;  // null: page b of k and v is sequence b
    int64_t table_row;      // elements
    const int32_t* lengths;  // null: all have `places`
    const int32_t* counts;   // null: all have T
    const int32_t* parents;  // of a tree
    int32_t kind;
    int32_t B, T, groups, fan, D;
    int32_t pages, page_rows;
    Divisor by_fan, by_groups, by_page, by_row_tiles, by_parts;
    int32_t places;  // of a sequence, at most: of its table, or states
    float scale2;    // scale * log2(e): exponentials are powers of 2
    bool q_whole, k_whole, y_whole;  // whole 16-byte pieces at addresses that are multiples of 16 (y: 8)
    // Rows r = t * fan + g of a group's heads are next to each other; a work-group takes a tile of them and one part of the places.
    int32_t row_tiles, tile_rows, parts;
    float* part_sums;  // [B][groups][row_tiles][parts][tile_rows][size of the kernel]: a part's own mean
    float* part_stats;  // [..][parts][tile_rows][2]: m, l: the weights' sum is l 2^m
    float* sums;  // [B][groups][T fan]: m + log2(l), where `mass` is asked for
    float* mass;
    int64_t mass_batch, mass_head;  // elements
};

template <bool kHalf>
struct AttentionKernels {
    // Elements of a head that a kernel works on, at least D; rows that a work-group takes.
    static int attend(const AttentionArgs& a, int size, hipStream_t s);
    static int join(const AttentionArgs& a, int size, hipStream_t s);
    static int mass(const AttentionArgs& a, int size, hipStream_t s);
};

// Elements of a head that the kernels are built for.
inline int attention_size(int32_t D) {
    return D <= 64 ? 64 : D <= 128 ? 128 : 256;
}

}  // namespace chx
