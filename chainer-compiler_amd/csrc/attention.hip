// Attention over a cache of pages and over an encoder's states: checks, the choice of tiles and parts, the entry points.  The kernels are in attention_kernel.h.
#include <cmath>
#include <cstring>
#include <initializer_list>

#include "attention.h"

namespace chx {
namespace {

// How rows and places are shared out.
//
// Tiles of 128 rows read k and v once for all of them; those of 32 rows fill more compute units, and leave fewer rows empty.  us of the better number of parts, 32 rows / 128, of states that all sequences have:
//                                              float16: 64 elements   128          256          float32: 64       128          256
//   3 x 197 rows of 12 heads, 577 places               13.0 / 19.7    18.9 / 26.3                25.5 / 34.2       42.4 / 54.1
//   2 x 512 of 16, 512                                 13.3 / 14.3    20.2 / 23.8                30.4 / 40.1       63.6 / 62.5
//   2 x 512 of 16, 1500                                25.1 / 34.6    38.6 / 40.1  93.0 / 71.5   68.5 / 74.5       154 / 135    502 / 251
//   4 x 512 of 16, 1500                                41.3 / 36.1    68.8 / 57.9  188 / 115     126 / 123         311 / 238    999 / 453
//   8 x 512 of 16, 1500                                68.2 / 45.1    139 / 82     373 / 224     251 / 209         616 / 471
//   4 x 24 x 4 of 8, 8000                              27.4 / 28.0    57.5 / 45.9  112 / 98.5    84.5 / 84.9       171 / 176    504 / 328
//   16 x 16 x 4 of 8, 4000 (half of 128 rows empty)    46.2 / 42.4    73.6 / 65.6  129 / 166     93.4 / 142        201 / 325    629 / 605
// So: 128 from as many tiles on as there are compute units (half as many where a tile is much work), a tile of many places counted as several; in float32, whose products take the time, not
// where half of the rows are empty.
//
// Parts: as many as fill the compute units once, two work-groups to each (one where rows are longer than 256 bytes and the tiles take more than half of LDS), of at least 256 places each (float32: 128);
// where they would have 4096 or more, several times as many, up to four, so that the units are even where sequences are not (where they are, 4 x 32768 places of 8 heads cost 118 us in 16, 125 in 32).  us of one token by parts, 8 heads of k and v, sequences from a
// sixteenth of this length to the whole (2 of 30000: all of it):
//                                              1     2     4     8     12    16    24    32    64
//   float16, 128 elements,  8 of 2000          38    27    20    17    23
//                           1 of 32768               (8: 80)                     40    38    40
//            256 elements,  8 of 4000          89    58    43    47    52    60
//                           2 of 30000         569   303   170   108   97    94    107   102   117
//   float32, 64 elements,   8 of 4000          103   61    37    31    38    36    42    43
//            128 elements,  8 of 4000          171   98    60    63    67    71    81    88
//                           2 of 20000         786   405   214   116   89    72    85    73    89
//            192 elements, 5 of 60215, 4 heads       5770  2913  1476  998   946   832   747   659
// One part, and no launch that joins them, where parts would be short: float16 below 1024 places, and below 2048 where whole sequences nearly fill the units.  us of 1 part / 2 / 4, 64 elements, the 252 to
// states that all sequences have, the others of sequences from a sixteenth of this length to the whole:
//                                              577 places      1500            4000
//   float16, 96 work-groups                    13 / 16 / 16    19 / 17 / 16
//            192                               12 / 14 / 14    19 / 18 / 18    41 / 33 / 29
//            252                               12 / 19 / 19    18 / 22 / 26    33 / 30 / 32
//   float32, 96                                23 / 19 / 19    44 / 31 / 26
//            192                               25 / 23 / 29    45 / 37 / 39    108 / 76 / 69
//            252                               25 / 31 / 39    43 / 46 / 51    93 / 87 / 92
void share_out(AttentionArgs* a, bool half) {
    const int64_t rows = (int64_t)a->T * a->fan, sets = (int64_t)a->B * a->groups, tiles = (rows + 127) / 128;
    const int size = attention_size(a->D);
    bool few = rows <= 32;
    if (!few && (half || size < 256)) {
        const int64_t wide = sets * tiles * (a->places < 1024 ? 1 : a->places / 1024);
        few = wide < (size == 64 || (half && size == 128) ? 256 : 128) || (!half && 2 * rows <= 128 * tiles);
    }
    a->tile_rows = few ? 32 : 128;
    a->row_tiles = (int32_t)((rows + a->tile_rows - 1) / a->tile_rows);
    const int64_t groups = sets * a->row_tiles, least = half ? 256 : 128, most = (a->places + least - 1) / least;
    int64_t parts = (size * (half ? 2 : 4) <= 256 ? 512 : 256) / (groups < 1 ? 1 : groups);
    if (parts > 0) parts *= a->places / parts / 2048 < 1 ? 1 : a->places / parts / 2048 > 4 ? 4 : a->places / parts / 2048;
    parts = parts > most ? most : parts;
    if (a->places < (groups > 224 ? 2048 : half ? 1024 : 0)) parts = 1;
    a->parts = (int32_t)(parts < 1 ? 1 : parts > kMostParts ? kMostParts : parts);
}

// Bytes of statistics, sums of weights and parts' results, one behind the other, each aligned to 16.
struct Space {
    int64_t stats, sums, all;
};
Space space_of(const AttentionArgs& a, bool with_mass) {
    const int64_t rows = (int64_t)a.B * a.groups * a.row_tiles * a.parts * a.tile_rows;
    Space s;
    s.stats = a.parts > 1 ? 8 * rows : 0;
    s.sums = with_mass ? (4 * (int64_t)a.B * a.groups * a.T * a.fan + 15) / 16 * 16 : 0;
    s.all = s.stats + s.sums + (a.parts > 1 ? 4 * rows * attention_size(a.D) : 0);
    return s;
}

// q and y [B, T, heads, elements], over k and v with `groups` heads.
int check_queries(const chx_hip_tensor* q, int32_t dtype, int64_t B, const char* what, AttentionArgs* a) {
    CHX_PROPAGATE(check_rows(q, 4, dtype, what, "q"));
    CHX_REQUIRE(q->shape[0] == B, "%s: q has %lld sequences, the others %lld", what, (long long)q->shape[0], (long long)B);
    CHX_REQUIRE(q->shape[3] == a->D, "%s: q has %lld elements of a head, keys %d", what, (long long)q->shape[3], a->D);
    CHX_REQUIRE(q->shape[2] >= 1 && q->shape[2] % a->groups == 0 && q->shape[2] < (int64_t(1) << 16), "%s: %lld heads of q do not share %d heads of keys", what, (long long)q->shape[2], a->groups);
    CHX_REQUIRE(q->shape[1] < (int64_t(1) << 24) && q->shape[1] * (q->shape[2] / a->groups) < (int64_t(1) << 30), "%s: 2^24 tokens, or 2^30 rows to a head of keys", what);
    a->B = (int32_t)B;
    a->T = (int32_t)q->shape[1];
    a->fan = (int32_t)(q->shape[2] / a->groups);
    share_out(a, q->dtype == CHX_HIP_FLOAT16);
    a->by_fan = divisor_of(a->fan);
    a->by_groups = divisor_of(a->groups);
    a->by_page = divisor_of(a->page_rows);
    a->by_row_tiles = divisor_of(a->row_tiles);
    a->by_parts = divisor_of(a->parts);
    CHX_REQUIRE((int64_t)a->B * a->groups * a->parts * a->row_tiles < (int64_t(1) << 23), "%s: more tiles than one launch has", what);
    return CHX_HIP_OK;
}

bool all_multiples(int64_t of, std::initializer_list<int64_t> bytes) {
    for (int64_t b : bytes)
        if (b % of != 0) return false;
    return true;
}
int64_t at_of(const void* p) {
    return (int64_t)reinterpret_cast<intptr_t>(p);
}

// The rest of a call, its arrays checked one by one: results apart from what is read, scale, workspace, launches.
int run(AttentionArgs& a, const chx_hip_tensor* q, const chx_hip_tensor* keys, const chx_hip_tensor* values, const Named* read, int reads, const chx_hip_tensor* mass, float scale,
        chx_hip_tensor* y, void* workspace, size_t workspace_bytes, hipStream_t s, const char* what) {
    CHX_PROPAGATE(check_rows(y, 4, q->dtype, what, "y"));
    CHX_REQUIRE(same_shape(*q, *y), "%s: y must have q's shape", what);
    CHX_REQUIRE(numel(*y) == 0 || elements_apart(*y), "%s: elements of y overlap", what);
    CHX_PROPAGATE(check_apart({y, "y"}, read, reads, what));
    a.scale2 = scale * 1.44269504f;
    CHX_REQUIRE(scale > 0.f && a.scale2 > 0.f && std::isfinite(a.scale2), "%s: the scale must be a positive number", what);
    const Space space = space_of(a, mass != nullptr);
    CHX_REQUIRE((int64_t)workspace_bytes >= space.all && (space.all == 0 || (workspace != nullptr && aligned(workspace, 16))), "%s: a workspace of %lld bytes, aligned to 16, is needed", what,
                (long long)space.all);
    if (numel(*q) == 0) return CHX_HIP_OK;
    char* at = static_cast<char*>(workspace);
    a.part_stats = reinterpret_cast<float*>(at);
    a.sums = mass ? reinterpret_cast<float*>(at + space.stats) : nullptr;
    a.part_sums = reinterpret_cast<float*>(at + space.stats + space.sums);
    a.q = static_cast<const char*>(q->data);
    a.y = static_cast<char*>(y->data);
    a.q_batch = stride_of(*q, 0), a.q_token = stride_of(*q, 1), a.q_head = stride_of(*q, 2);
    a.y_batch = stride_of(*y, 0), a.y_token = stride_of(*y, 1), a.y_head = stride_of(*y, 2);
    a.k = static_cast<const char*>(keys->data);
    a.v = static_cast<const char*>(values->data);
    a.k_page = stride_of(*keys, 0), a.k_row = stride_of(*keys, 1), a.k_head = stride_of(*keys, 2);
    a.v_page = stride_of(*values, 0), a.v_row = stride_of(*values, 1), a.v_head = stride_of(*values, 2);
    const int64_t row = (int64_t)a.D * dtype_size(q->dtype);
    a.q_whole = all_multiples(16, {at_of(a.q), a.q_batch, a.q_token, a.q_head, row});
    a.k_whole = all_multiples(16, {at_of(a.k), at_of(a.v), a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head, row});
    a.y_whole = all_multiples(q->dtype == CHX_HIP_FLOAT16 ? 8 : 16, {at_of(a.y), a.y_batch, a.y_token, a.y_head, row});
    const int size = attention_size(a.D);
    const bool half = q->dtype == CHX_HIP_FLOAT16;
    CHX_PROPAGATE(half ? AttentionKernels<true>::attend(a, size, s) : AttentionKernels<false>::attend(a, size, s));
    if (a.parts > 1) CHX_PROPAGATE(half ? AttentionKernels<true>::join(a, size, s) : AttentionKernels<false>::join(a, size, s));
    if (mass && a.places > 0) CHX_PROPAGATE(half ? AttentionKernels<true>::mass(a, size, s) : AttentionKernels<false>::mass(a, size, s));
    return CHX_HIP_OK;
}

void describe(const CacheArgs& c, AttentionArgs* a) {
    a->tables = c.tables;
    a->table_row = c.table_row;
    a->lengths = c.lengths;
    a->groups = c.groups;
    a->D = c.D;
    a->pages = c.pages;
    a->page_rows = c.page_rows;
    a->places = c.places;
}

int check_states(const chx_hip_tensor* keys, const char* what, AttentionArgs* a) {
    CHX_PROPAGATE(check_rows(keys, 4, 0, what, "keys"));
    CHX_REQUIRE(keys->shape[2] >= 1 && keys->shape[2] < (int64_t(1) << 16) && keys->shape[3] >= 1 && keys->shape[3] <= kMostSize, "%s: keys need 1 to 2^16 - 1 heads of 1 to %d elements", what, kMostSize);
    CHX_REQUIRE(keys->shape[0] < (int64_t(1) << 24) && keys->shape[1] < (int64_t(1) << 30), "%s: 2^24 sequences, or 2^30 states", what);
    a->kind = kCross;
    a->groups = (int32_t)keys->shape[2];
    a->D = (int32_t)keys->shape[3];
    a->pages = (int32_t)keys->shape[0];
    a->page_rows = a->places = (int32_t)keys->shape[1];
    return CHX_HIP_OK;
}

}  // namespace
}  // namespace chx

using namespace chx;

extern "C" int chx_hip_tree_attention_workspace(const chx_hip_tensor* q, const chx_hip_tensor* keys, const chx_hip_tensor* tables, int32_t with_mass, size_t* bytes) {
    const char* what = "tree attention";
    CHX_REQUIRE(bytes != nullptr, "%s: null output", what);
    CHX_PROPAGATE(check_tensor(tables, "tables"));
    CHX_REQUIRE(tables->ndim == 2, "%s: tables must be an int32 matrix", what);
    chx_hip_tensor lengths;
    memset(&lengths, 0, sizeof(lengths));
    lengths.data = tables->data, lengths.dtype = CHX_HIP_INT32, lengths.ndim = 1, lengths.shape[0] = tables->shape[0], lengths.strides[0] = 4;
    if (numel(*tables) == 0) lengths.data = bytes;  // (only asked whether it is there)
    CacheArgs c;
    AttentionArgs a;
    memset(&a, 0, sizeof(a));
    CHX_PROPAGATE(check_cache(keys, keys, tables, &lengths, what, &c));
    describe(c, &a);
    CHX_PROPAGATE(check_queries(q, keys->dtype, c.B, what, &a));
    *bytes = (size_t)space_of(a, with_mass != 0).all;
    return CHX_HIP_OK;
}

extern "C" int chx_hip_tree_attention(
        const chx_hip_tensor* q, const chx_hip_tensor* keys, const chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, const chx_hip_tensor* parents,
        const chx_hip_tensor* counts, float scale, chx_hip_tensor* mass, chx_hip_tensor* y, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "tree attention";
    CacheArgs c;
    AttentionArgs a;
    memset(&a, 0, sizeof(a));
    CHX_PROPAGATE(check_cache(keys, values, tables, lengths, what, &c));
    describe(c, &a);
    CHX_PROPAGATE(check_queries(q, keys->dtype, c.B, what, &a));
    a.kind = parents ? kTree : kChain;
    if (parents) {
        CHX_REQUIRE(a.T <= kMostNodes, "%s: a tree of at most %d nodes, not %d", what, kMostNodes, a.T);
        CHX_PROPAGATE(check_numbers(parents, 2, a.B, a.T, what, "parents"));
        a.parents = static_cast<const int32_t*>(parents->data);
    }
    if (counts) {
        CHX_PROPAGATE(check_numbers(counts, 1, a.B, 0, what, "counts"));
        a.counts = static_cast<const int32_t*>(counts->data);
    }
    const Named read[] = {{q, "q"}, {keys, "keys"}, {values, "values"}, {tables, "tables"}, {lengths, "lengths"}, {parents, "parents"}, {counts, "counts"}, {mass, "mass"}};
    if (mass) {
        CHX_PROPAGATE(check_mass(mass, c, what));
        CHX_PROPAGATE(check_apart({mass, "mass"}, read, 7, what));
        CHX_REQUIRE((int64_t)a.B * a.groups * ((a.places + 31) / 32) < (int64_t(1) << 24), "%s: more places than one launch has", what);
        a.mass = static_cast<float*>(mass->data);
        a.mass_batch = mass->strides[0] / 4;
        a.mass_head = mass->strides[1] / 4;
    }
    return run(a, q, keys, values, read, 8, mass, scale, y, workspace, workspace_bytes, as_stream(stream), what);
}

extern "C" int chx_hip_cross_attention_workspace(const chx_hip_tensor* q, const chx_hip_tensor* keys, size_t* bytes) {
    const char* what = "cross attention";
    CHX_REQUIRE(bytes != nullptr, "%s: null output", what);
    AttentionArgs a;
    memset(&a, 0, sizeof(a));
    CHX_PROPAGATE(check_states(keys, what, &a));
    CHX_PROPAGATE(check_queries(q, keys->dtype, keys->shape[0], what, &a));
    *bytes = (size_t)space_of(a, false).all;
    return CHX_HIP_OK;
}

extern "C" int chx_hip_cross_attention(
        const chx_hip_tensor* q, const chx_hip_tensor* keys, const chx_hip_tensor* values, const chx_hip_tensor* lengths, float scale, chx_hip_tensor* y, void* workspace,
        size_t workspace_bytes, void* stream) {
    const char* what = "cross attention";
    AttentionArgs a;
    memset(&a, 0, sizeof(a));
    CHX_PROPAGATE(check_states(keys, what, &a));
    CHX_PROPAGATE(check_rows(values, 4, keys->dtype, what, "values"));
    CHX_REQUIRE(same_shape(*keys, *values), "%s: keys and values must have one shape", what);
    CHX_PROPAGATE(check_queries(q, keys->dtype, keys->shape[0], what, &a));
    if (lengths) {
        CHX_PROPAGATE(check_numbers(lengths, 1, a.B, 0, what, "lengths"));
        a.lengths = static_cast<const int32_t*>(lengths->data);
    }
    const Named read[] = {{q, "q"}, {keys, "keys"}, {values, "values"}, {lengths, "lengths"}};
    return run(a, q, keys, values, read, 4, nullptr, scale, y, workspace, workspace_bytes, as_stream(stream), what);
}
