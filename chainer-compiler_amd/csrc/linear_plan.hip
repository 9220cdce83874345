// Matrix products with bias, activation and residual in their epilogue, from weights that are laid out once: the host side and the
// layout (linear_plan.h); the kernels are in linear_kernel.h.
#include <algorithm>
#include <cstring>
#include <new>

#include "linear_plan.h"

struct chx_hip_linear_plan {
    chx::LinearType type = chx::kHalfHalf;
    char* w = nullptr;       // laid out; then scales and biases, each float32 [experts][n_padded]
    float* scale = nullptr;
    float* bias = nullptr;
    int64_t w_group = 0, w_expert = 0;
    int32_t N = 0, K = 0, units = 0, experts = 0, n_padded = 0;  // experts 0: a plan without
    int device = 0;
};

namespace chx {
namespace {

struct LayoutArgs {
    const char* w;
    int64_t ws_e, ws_n, ws_k;  // bytes
    char* out;
    int32_t N, K, units, groups, type;
    int64_t w_group;
    int64_t kilobytes;  // of all
    int64_t first;      // work-group of this launch
};

// One lane writes 16 bytes, a wavefront 1 KB: a fragment, or two of int8.  Runs once per layer; w is read through its strides.
__global__ __launch_bounds__(256) void linear_layout_kernel(LayoutArgs a) {
    const int64_t at = (a.first + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (at >= a.kilobytes) return;
    const int lane = threadIdx.x & 63, each = a.type == kHalfInt8 ? 2 : 4;
    const int part = (int)(at % each);
    const int64_t unit = at / each % a.units, group = at / each / a.units % a.groups, expert = at / each / a.units / a.groups;
    const char* first = a.w + expert * a.ws_e + group * kGroupRows * a.ws_n;
    uint32_t v[4] = {0, 0, 0, 0};
    const int64_t k0 = unit * (a.type == kFloatFloat ? 16 : 32) + (lane >> 4) * (a.type == kFloatFloat ? 4 : 8);
    auto element = [&](int fragment, int j) -> const char* {
        const int r = group_row(fragment, lane & 15);
        return group * kGroupRows + r < a.N && k0 + j < a.K ? first + r * a.ws_n + (k0 + j) * a.ws_k : nullptr;
    };
    if (a.type == kHalfHalf) {
        for (int j = 0; j < 8; ++j)
            if (const char* p = element(part, j)) v[j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p) << (16 * (j & 1));
    } else if (a.type == kHalfInt8) {
        for (int j = 0; j < 16; ++j)
            if (const char* p = element(2 * part + (j >> 3), j & 7)) v[j / 4] |= (uint32_t)*reinterpret_cast<const uint8_t*>(p) << (8 * (j & 3));
    } else {
        for (int j = 0; j < 4; ++j)
            if (const char* p = element(part, j)) v[j] = *reinterpret_cast<const uint32_t*>(p);
    }
    *reinterpret_cast<uint4*>(a.out + (expert * a.groups + group) * a.w_group + (unit * each + part) * 1024 + lane * 16) = make_uint4(v[0], v[1], v[2], v[3]);
}

struct VectorArgs {
    const char* v;
    int64_t s_e, s_n;  // bytes
    float* out;
    int32_t N, n_padded, half;
    int64_t total, first;
};

__global__ __launch_bounds__(256) void linear_vector_kernel(VectorArgs a) {
    const int64_t at = (a.first + blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.total) return;
    const int64_t e = at / a.n_padded, n = at % a.n_padded;
    const char* p = a.v + e * a.s_e + n * a.s_n;
    a.out[at] = n >= a.N ? 0.f : a.half ? (float)*reinterpret_cast<const _Float16*>(p) : *reinterpret_cast<const float*>(p);
}

// x in rows of whole blocks of 16-byte pieces, with zeros behind K, for the tiles: one lane a piece.
struct RowsArgs {
    const char* x;
    int64_t x_row, x_col;  // bytes
    char* out;
    int64_t pitch, pieces;  // bytes of a row; 16-byte pieces of all
    int64_t first;
    int32_t K;
};

template <typename T>
__global__ __launch_bounds__(256) void linear_pieces_kernel(RowsArgs a) {
    const int64_t at = (a.first + blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.pieces) return;
    constexpr int kCount = 16 / sizeof(T);
    const int64_t row = at / (a.pitch / 16), k0 = at % (a.pitch / 16) * kCount;
    const char* p = a.x + row * a.x_row + k0 * a.x_col;
    T v[kCount];
    if (a.x_col == sizeof(T) && k0 + kCount <= a.K) {
        __builtin_memcpy(v, __builtin_assume_aligned(p, sizeof(T)), 16);
    } else {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = k0 + j < a.K ? *reinterpret_cast<const T*>(p + j * a.x_col) : T(0);
    }
    __builtin_memcpy(__builtin_assume_aligned(a.out + at * 16, 16), v, 16);
}

// The axes before the last as one run of rows.
bool as_rows(const chx_hip_tensor& t, int64_t* rows, int64_t* row_stride) {
    int64_t count = 1, st = 0;
    bool first = true;
    for (int d = t.ndim - 2; d >= 0; --d) {
        if (t.shape[d] == 1) continue;
        if (first) {
            st = t.strides[d];
            first = false;
        } else if (t.strides[d] != st * count) {
            return false;
        }
        count *= t.shape[d];
    }
    *rows = count;
    *row_stride = st;
    return true;
}

// Distances and address that are whole elements: the kernels load by element where they cannot load more.
int check_elements(const chx_hip_tensor& t, const char* name) {
    const int64_t es = dtype_size(t.dtype);
    CHX_REQUIRE(aligned(t.data, (size_t)es), "linear plan: %s does not begin at an element's address", name);
    for (int d = 0; d < t.ndim; ++d) CHX_REQUIRE(t.strides[d] % es == 0, "linear plan: a stride of %s is not a number of whole elements", name);
    return CHX_HIP_OK;
}

bool aligned_rows(const void* p, int64_t row_stride, int64_t rows, int64_t bytes) {
    return aligned(p, (size_t)bytes) && (rows == 1 || row_stride % bytes == 0);
}

struct Call {
    LinearArgs a;
    int64_t x_rows;
    bool direct;
};

// Bytes of a row of x in whole pieces, as the tiles take it.
int64_t pitch_of(int32_t K, LinearType type) {
    return ((int64_t)K * (type == kFloatFloat ? 4 : 2) + 127) / 128 * 128;
}

// Whether a tile can address rows of x that are `pitch` bytes apart: 32 bits from its first one, or from x for experts.  (Where x of experts spans 4 GiB this costs two thirds of
// the rate: 528,000 rows to 8 experts of 4096 x 2048 19.3 ms, 480,000 in tiles 6.3.)
bool within_reach(int64_t pitch, int64_t x_rows, bool experts) {
    return pitch < (int64_t(1) << 23) && (!experts || pitch * x_rows + 128 < (int64_t(1) << 32));
}

int prepare_call(const chx_hip_linear_plan* plan, const chx_hip_tensor* x, int32_t activation, const chx_hip_tensor* r, chx_hip_tensor* y, Call* c) {
    CHX_REQUIRE(plan != nullptr, "linear plan: null plan");
    CHX_PROPAGATE(check_tensor(x, "linear plan x"));
    CHX_PROPAGATE(check_tensor(y, "linear plan y"));
    const int32_t type = plan->type == kFloatFloat ? CHX_HIP_FLOAT32 : CHX_HIP_FLOAT16;
    CHX_REQUIRE(x->dtype == type, "linear plan: x must be %s for these weights, not %s", dtype_name(type), dtype_name(x->dtype));
    CHX_REQUIRE(y->dtype == CHX_HIP_FLOAT32 || (y->dtype == CHX_HIP_FLOAT16 && type == CHX_HIP_FLOAT16), "linear plan: y must be float32%s, not %s",
                type == CHX_HIP_FLOAT16 ? " or float16" : "", dtype_name(y->dtype));
    CHX_REQUIRE(activation >= CHX_HIP_ACT_NONE && activation <= CHX_HIP_ACT_SILU, "linear plan: unknown activation %d", activation);
    CHX_REQUIRE(x->ndim >= 1 && x->shape[x->ndim - 1] == plan->K, "linear plan: the last axis of x must have %d elements", plan->K);
    CHX_REQUIRE(y->ndim >= 1 && y->shape[y->ndim - 1] == plan->N, "linear plan: the last axis of y must have %d elements", plan->N);
    CHX_PROPAGATE(check_elements(*x, "x"));
    CHX_PROPAGATE(check_elements(*y, "y"));
    int device = 0;
    CHX_HIP_CALL(hipGetDevice(&device));
    CHX_REQUIRE(device == plan->device, "linear plan: created on device %d, run on device %d", plan->device, device);
    LinearArgs& a = c->a;
    memset(&a, 0, sizeof(a));
    int64_t x_rows = 0, y_rows = 0;
    CHX_REQUIRE(as_rows(*x, &x_rows, &a.x_row), "linear plan: the leading axes of x are not one run of rows");
    CHX_REQUIRE(as_rows(*y, &y_rows, &a.y_row), "linear plan: the leading axes of y are not one run of rows");
    CHX_REQUIRE(y_rows < (int64_t(1) << 31) && x_rows < (int64_t(1) << 31), "linear plan: 2^31 rows or more");
    const int64_t xe = dtype_size(x->dtype), ye = dtype_size(y->dtype);
    a.x = static_cast<const char*>(x->data);
    a.y = static_cast<char*>(y->data);
    a.x_col = plan->K == 1 ? xe : x->strides[x->ndim - 1];
    a.y_col = plan->N == 1 ? ye : y->strides[y->ndim - 1];
    a.y_half = y->dtype == CHX_HIP_FLOAT16;
    a.vector_y = a.y_col == ye && aligned_rows(a.y, a.y_row, y_rows, 4 * ye);
    if (r != nullptr) {
        CHX_PROPAGATE(check_tensor(r, "linear plan r"));
        CHX_REQUIRE(r->dtype == y->dtype && same_shape(*r, *y), "linear plan: r must have the type and shape of y");
        CHX_PROPAGATE(check_elements(*r, "r"));
        int64_t r_rows = 0;
        CHX_REQUIRE(as_rows(*r, &r_rows, &a.r_row), "linear plan: the leading axes of r are not one run of rows");
        a.r = static_cast<const char*>(r->data);
        a.r_col = plan->N == 1 ? ye : r->strides[r->ndim - 1];
        a.vector_r = a.r_col == ye && aligned_rows(a.r, a.r_row, r_rows, 4 * ye);
    }
    if (numel(*y) > 0) {
        CHX_REQUIRE(elements_apart(*y), "linear plan: elements of y overlap");
        CHX_REQUIRE(numel(*x) == 0 || !arrays_overlap(*x, *y), "linear plan: x and y overlap");
        CHX_REQUIRE(r == nullptr || same_array(*r, *y) || !arrays_overlap(*r, *y), "linear plan: r and y overlap and are not the same array");
    }
    a.w = plan->w;
    a.scale = plan->scale;
    a.bias = plan->bias;
    a.w_group = plan->w_group;
    a.w_expert = plan->w_expert;
    a.M = (int32_t)y_rows;
    a.N = plan->N;
    a.K = plan->K;
    a.units = plan->units;
    a.n_padded = plan->n_padded;
    a.activation = activation;
    a.fan = 1;
    c->x_rows = x_rows;
    // whole blocks that can be copied in pieces of 16 bytes, addressed with 32 bits from a tile's first row
    c->direct = a.K % (2 * unit_k(plan->type)) == 0 && a.x_col == xe && aligned_rows(a.x, a.x_row, x_rows, 16) && a.x_row >= 0 && within_reach(a.x_row, x_rows, false);
    return CHX_HIP_OK;
}

// What runs a product: work-groups of 16 row_tiles rows and 16 fragments columns (linear_rows_kernel), or, with fragments 0, a tile.
struct Choice {
    int row_tiles, fragments;
    LinearTile tile;
};

// float32, M > 32: the kernel with the least time, where one of 256 compute units has the most work-groups to do.  us of a work-group each, by K = 4096 (512 rows of
// 4096 x 4096: 205 us in 32 x 32, 185 in 32 x 64, 168 in 64 x 32, 152 in 64 x 64, 131 in tiles of 64 x 128; 2048 rows 829, 755, 667, 598 and 472):
// the first that fits instead cost up to half as much again where a few work-groups were left over.  (What a work-group costs beside its products is not told apart, so with short K the choice is not the
// best: 2777 x 64 x 16225 takes 148 us, a library's product 110.)  us of each in this order, and of a library's product alone:
//   690 x 10880 x 1560 rows x K x N   320   344   304   366   334   213
//   91 x 3648 x 9760                   95    87   112   132   117    62
//   699 x 3328 x 13056                800   726   642   574   476   452
//   1782 x 5248 x 867                 180   207   193   183   169   139
//   300 x 1024 x 1024                16.7  15.5  15.3  25.7  37.9  23.4
Choice choose_float(int64_t M, int64_t N) {
    static const struct {
        Choice c;
        int rows, columns;
        float first, next;
    } kernels[] = {{{2, 2, kTile64}, 32, 32, 25.5f, 25.5f}, {{2, 4, kTile64}, 32, 64, 46.f, 46.f}, {{4, 2, kTile64}, 64, 32, 42.f, 42.f},
                   {{4, 4, kTile64}, 64, 64, 76.f, 76.f},   {{0, 0, kTile64}, 64, 128, 131.f, 115.f}};
    Choice best = kernels[0].c;
    float least = 0.f;
    for (const auto& k : kernels) {
        const int64_t each = ((M + k.rows - 1) / k.rows * ((N + k.columns - 1) / k.columns) + 255) / 256;
        const float us = k.first + (float)(each - 1) * k.next;
        if (least == 0.f || us < least) {
            least = us;
            best = k.c;
        }
    }
    return best;
}

// The kernel for M rows that are all multiplied with the same weights: the smallest of its sizes that does not need more work-groups than there are compute
// units.  All sizes were timed over 7 weights from 1024 x 1024 to 4096 x 16384, 12 numbers of rows and the three types, recorded, three layers in turn.
// us in float16 of the one chosen, and of the next smaller and larger ones:
//  K x N            rows   16 x 16   32 x 16   32 x 32   32 x 64   64 x 64   64 x 128   128 x 128   256 x 256
//  4096 x 4096        32     16.0     [10.7]     13.6      17.6      19.3                  28.4
//                     64     28.9      18.4     [13.3]     17.1      21.5                  29.1
//                    128     54.4      34.0      22.7     [16.9]     20.8                  29.3
//                    256                         43.5      29.8     [21.0]      29.0       33.4        77
//                    512                                   62.0      41.8      [30.3]      33.6        78
//                   1024                                             80.1       43.1      [40.1]       78
//                   2048                                            158.1       84.1      [68.2]       80
//  4096 x 16384     1024                                            414.7                 147.3      [111]
// Where the tiles of 128 are too few, products of int8 lose more by that (512 rows of 4096 x 4096: 42.2 in 128 x 128, 33.0 in 64 x 128 and 29.2 in 64 x 64).
// Tiles of 64 x 128 take the place of those of 128 x 128 where a compute unit has less than twice as many of them to do: 436 rows of 8448 x 9056
// 81.5 instead of 102.4 (int8 91.6 and 97.2), 2048 of 1024 x 1024 11.6 instead of 15.2.
// Up to 8 rows x is not copied into LDS (16 x 16, 16 x 32 and 16 x 64).
Choice choose(int64_t M, int64_t N, LinearType type) {
    const int64_t most = 256;
    auto groups = [&](int64_t rows, int64_t columns) { return (M + rows - 1) / rows * ((N + columns - 1) / columns); };
    const int first = type == kHalfInt8 ? 2 : 1;  // (two fragments of int8 are one piece)
    const int row_tiles = M <= 8 ? 1 : 2;
    for (int fragments = first; fragments <= 4; fragments *= 2)
        if (groups(16 * row_tiles, 16 * fragments) <= most) return {row_tiles, fragments, kTile64};
    if (M <= 32) return {row_tiles, 4, kTile64};
    if (type == kFloatFloat) return choose_float(M, N);
    const int64_t tiles = groups(128, 128);
    if (M <= 64 || groups(64, 64) <= most || (type == kHalfInt8 && tiles < 160)) return {4, 4, kTile64};
    if (tiles > 2 * most) return {0, 0, kTile256};
    return {0, 0, (groups(64, 128) + most - 1) / most < 2 * ((tiles + most - 1) / most) ? kTile64 : kTile128};
}

// The same for experts, by the rows that each has on the average.  us with 16 x 64 / 32 x 64 / 64 x 64 / tiles of 64 x 128 / of 128 / of 256, experts' loads
// as uneven as their normally distributed scores make them:
//   64 experts of 1536 x 2048:  rows each  2   float16   47 /   46 /   63 /   58 /   72 /   76   int8    32 /   32 /   54 /   30 /   51 /   68
//                                          8             58 /   52 /   67 /   65 /   77 /   81           41 /   36 /   65 /   37 /   55 /   70
//                                         16             80 /   66 /   79 /   73 /   82 /   87           56 /   46 /   66 /   40 /   60 /   72
//                                         32            123 /   94 /  103 /   90 /   88 /   93           87 /   63 /   78 /   51 /   64 /   79
//   64 experts of 1024 x 2048:            64            128 /   94 /   94 /   74 /   76 /   86          101 /   65 /   78 /   46 /   56 /   75
//   32 experts of 2048 x 4096:           128            497 /  320 /  241 /  167 /  152 /  159          318 /  190 /  184 /  121 /  124 /  157
//                                        512           1849 / 1093 /  780 /  433 /  345 /  295         1192 /  658 /  588 /  356 /  308 /  297
//   8 experts of 4096 x 4096:            512           1028 /  621 /  434 /  206 /  178 /  180          681 /  357 /  310 /  180 /  165 /  183
// (float32, the first four: 8 rows each 136 / 141 / 233 / 138, 32 rows 307 / 242 / 281 / 221, 64 rows 358 / 242 / 276 / 194, 128 rows 1364 / 853 / 784 / 631; 32 rows each
// of 1024 x 2048 202 / 155 / 198 / 162.)
Choice choose_for_experts(int64_t M, int64_t experts, int64_t N, LinearType type) {
    const int64_t each = (M + experts - 1) / experts;
    if (each > (type == kFloatFloat ? 32 : type == kHalfHalf ? 24 : 12))
        return {0, 0, type == kFloatFloat || each <= 96 ? kTile64 : each >= 256 && type == kHalfHalf ? kTile256 : kTile128};
    const int row_tiles = each <= (type == kFloatFloat ? 8 : 4) ? 1 : 2;
    const int64_t wide = (M / (16 * row_tiles) + std::min(M, experts)) * ((N + kGroupRows - 1) / kGroupRows);
    return {row_tiles, wide >= 256 ? 4 : wide >= 128 || type == kHalfInt8 ? 2 : 1, kTile64};
}

// The kernel for a call: experts 0 without experts; x of x_rows rows.
Choice choice_of(int64_t M, int64_t experts, int64_t x_rows, int64_t N, int32_t K, LinearType type) {
    const Choice c = experts ? choose_for_experts(M, experts, N, type) : choose(M, N, type);
    // (rows that a tile cannot address: the other kernel has 64 bits for them)
    if (c.fragments == 0 && !within_reach(pitch_of(K, type), x_rows, experts > 0)) return {4, 4, kTile64};
    return c;
}

// Whether x is brought into whole blocks first: for tiles always, for the other kernel where the launch that this takes (2 to 3 us) is made up for by copies instead of
// loads through registers (512 rows of 2047 x 4096: int8 31 us and 23 with the launch, float32 91 and 85; below some 256 rows that is what it costs).
bool into_pieces(const Choice& c, bool direct, int64_t x_rows, int32_t K, bool experts, LinearType type) {
    return !direct && (c.fragments == 0 || (c.row_tiles > 1 && x_rows > 256 && within_reach(pitch_of(K, type), x_rows, experts)));
}

template <LinearType kType>
int launch(Call& call, void* workspace, size_t workspace_bytes, hipStream_t s) {
    LinearArgs& a = call.a;
    const Choice c = choice_of(a.M, a.experts, call.x_rows, a.N, a.K, kType);
    const int32_t height = c.fragments > 0 ? 16 * c.row_tiles : c.tile == kTile256 ? 256 : c.tile == kTile128 ? 128 : 64;
    const int32_t width = c.fragments > 0 ? 16 * c.fragments : std::max(height, 128);
    // The most tiles of rows there can be: experts' tiles begin anew with each of them.
    const int64_t tiles_m = a.order ? a.M / height + std::min(a.M, a.experts) : ((int64_t)a.M + height - 1) / height;
    // (those of few rows take all fragments of whole groups)
    const int64_t tiles_n = c.fragments > 0 ? (int64_t)a.n_padded / width : (a.N + width - 1) / width;
    const int64_t work_groups = c.fragments == 0 && a.order ? expert_grid(tiles_m, tiles_n) : tiles_m * tiles_n;
    const int64_t threads = c.fragments > 0 || c.tile == kTile256 ? 512 : 256;
    CHX_REQUIRE(work_groups * threads < (int64_t(1) << 32), "linear plan: too many results: %lld work-groups of %lld threads, and a launch has fewer than 2^32 threads",
                (long long)work_groups, (long long)threads);
    a.tiles_m = (int32_t)tiles_m;
    a.tiles_n = (int32_t)tiles_n;
    if (into_pieces(c, call.direct, call.x_rows, a.K, a.order != nullptr, kType)) {
        RowsArgs r = {a.x, a.x_row, a.x_col, static_cast<char*>(workspace), pitch_of(a.K, kType), 0, 0, a.K};
        CHX_REQUIRE(workspace != nullptr && aligned(workspace, 16) && (int64_t)workspace_bytes >= r.pitch * call.x_rows,
                    "linear plan: a workspace of %lld bytes, aligned to 16, is needed for rows like these", (long long)(r.pitch * call.x_rows));
        r.pieces = r.pitch / 16 * call.x_rows;
        CHX_PROPAGATE(in_launches((r.pieces + 255) / 256, "linear_pieces_kernel", [&](int64_t first, unsigned count) {
            r.first = first;
            if (kType == kFloatFloat) linear_pieces_kernel<uint32_t><<<count, 256, 0, s>>>(r);
            else linear_pieces_kernel<uint16_t><<<count, 256, 0, s>>>(r);
        }));
        a.x = r.out;
        a.x_row = r.pitch;
        a.x_col = kType == kFloatFloat ? 4 : 2;
        call.direct = true;
    }
    return c.fragments > 0 ? LinearKernels<kType>::rows(a, c.row_tiles, c.fragments, call.direct, s) : LinearKernels<kType>::tile(a, c.tile, s);
}

int launch_of(const chx_hip_linear_plan* plan, Call& c, void* workspace, size_t workspace_bytes, hipStream_t s) {
    if (c.a.M == 0 || c.a.N == 0) return CHX_HIP_OK;
    switch (plan->type) {
        case kHalfHalf: return launch<kHalfHalf>(c, workspace, workspace_bytes, s);
        case kHalfInt8: return launch<kHalfInt8>(c, workspace, workspace_bytes, s);
        default: return launch<kFloatFloat>(c, workspace, workspace_bytes, s);
    }
}

}  // namespace
}  // namespace chx

using namespace chx;

extern "C" int chx_hip_linear_plan_create(
        const chx_hip_tensor* w, const chx_hip_tensor* w_scale, const chx_hip_tensor* b, void* stream, chx_hip_linear_plan** out) {
    CHX_REQUIRE(out != nullptr, "linear plan: null output");
    *out = nullptr;
    CHX_PROPAGATE(check_tensor(w, "linear plan w"));
    CHX_REQUIRE(w->dtype == CHX_HIP_FLOAT16 || w->dtype == CHX_HIP_FLOAT32 || w->dtype == CHX_HIP_INT8, "linear plan: w must be float16, float32 or int8, not %s",
                dtype_name(w->dtype));
    CHX_REQUIRE(w->ndim == 2 || w->ndim == 3, "linear plan: w must be [N, K] or [experts, N, K]");
    CHX_PROPAGATE(check_elements(*w, "w"));
    const int lead = w->ndim - 2;
    const int64_t E = lead ? w->shape[0] : 1, N = w->shape[lead], K = w->shape[lead + 1];
    CHX_REQUIRE(E >= 1 && N >= 1 && K >= 1, "linear plan: w has no elements");
    CHX_REQUIRE(E <= 65536 && N <= (1 << 24) && K <= (1 << 24), "linear plan: more than 65536 experts, or more than 2^24 rows or columns of w");
    CHX_REQUIRE((w->dtype == CHX_HIP_INT8) == (w_scale != nullptr), "linear plan: int8 weights have a w_scale, others have none");
    auto check_vector = [&](const chx_hip_tensor* t, const char* name) -> int {
        CHX_PROPAGATE(check_tensor(t, name));
        CHX_REQUIRE(t->dtype == CHX_HIP_FLOAT32 || (t->dtype == CHX_HIP_FLOAT16 && t == b), "linear plan: the type of %s", name);
        CHX_REQUIRE(t->ndim == lead + 1 && t->shape[lead] == N && (lead == 0 || t->shape[0] == E), "linear plan: %s must be [N], or [experts, N]", name);
        return check_elements(*t, name);
    };
    if (w_scale) CHX_PROPAGATE(check_vector(w_scale, "w_scale"));
    if (b) CHX_PROPAGATE(check_vector(b, "b"));
    chx_hip_linear_plan p;
    p.type = w->dtype == CHX_HIP_FLOAT16 ? kHalfHalf : w->dtype == CHX_HIP_INT8 ? kHalfInt8 : kFloatFloat;
    const int64_t groups = (N + kGroupRows - 1) / kGroupRows;
    p.units = (int32_t)((K + 2 * unit_k(p.type) - 1) / (2 * unit_k(p.type)) * 2);
    p.N = (int32_t)N;
    p.K = (int32_t)K;
    p.experts = lead ? (int32_t)E : 0;
    p.n_padded = (int32_t)(groups * kGroupRows);
    p.w_group = (int64_t)p.units * unit_bytes(p.type);
    p.w_expert = groups * p.w_group;
    // (a tile's groups are addressed with 32 bits)
    CHX_REQUIRE(p.w_group < (int64_t(1) << 29), "linear plan: a row of w is too long");
    CHX_REQUIRE((double)E * (double)p.w_expert < 0x1p46, "linear plan: too many weights");
    // (memory is allocated and the stream waited for: neither can be recorded)
    if (stream_is_capturing(as_stream(stream))) CHX_FAIL(CHX_HIP_EUNSUPPORTED, "linear plan: cannot be created while the stream is being captured into a graph");
    CHX_HIP_CALL(hipGetDevice(&p.device));
    const int64_t vector_bytes = E * p.n_padded * 4, bytes = E * p.w_expert + (w_scale ? vector_bytes : 0) + (b ? vector_bytes : 0);
    void* memory = nullptr;
    CHX_PROPAGATE(spare_memory(&memory, (size_t)bytes, "linear plan"));
    p.w = static_cast<char*>(memory);
    char* next = p.w + E * p.w_expert;
    LayoutArgs l = {static_cast<const char*>(w->data), lead ? w->strides[0] : 0, w->strides[lead], w->strides[lead + 1], p.w, p.N, p.K, p.units,
                    (int32_t)groups, (int32_t)p.type, p.w_group, E * groups * p.units * unit_bytes(p.type) / 1024, 0};
    int rc = in_launches((l.kilobytes + 3) / 4, "linear_layout_kernel", [&](int64_t first, unsigned count) {
        l.first = first;
        linear_layout_kernel<<<count, 256, 0, as_stream(stream)>>>(l);
    });
    auto vector = [&](const chx_hip_tensor* t) {
        float* out_v = reinterpret_cast<float*>(next);
        next += vector_bytes;
        if (rc != CHX_HIP_OK) return out_v;
        VectorArgs v = {static_cast<const char*>(t->data), lead ? t->strides[0] : 0, t->strides[lead], out_v, p.N, p.n_padded, t->dtype == CHX_HIP_FLOAT16, E * p.n_padded, 0};
        rc = in_launches((v.total + 255) / 256, "linear_vector_kernel", [&](int64_t first, unsigned count) {
            v.first = first;
            linear_vector_kernel<<<count, 256, 0, as_stream(stream)>>>(v);
        });
        return out_v;
    };
    if (w_scale) p.scale = vector(w_scale);
    if (b) p.bias = vector(b);
    // (later calls may come on any stream)
    if (rc == CHX_HIP_OK && hipStreamSynchronize(as_stream(stream)) != hipSuccess) {
        set_error("linear plan: the stream is in error, or being recorded");
        rc = CHX_HIP_ERUNTIME;
    }
    chx_hip_linear_plan* made = rc == CHX_HIP_OK ? new (std::nothrow) chx_hip_linear_plan(p) : nullptr;
    if (made == nullptr) {
        (void)hipFree(memory);
        if (rc == CHX_HIP_OK) CHX_FAIL(CHX_HIP_ERUNTIME, "linear plan: no memory on the host");
        return rc;
    }
    *out = made;
    return CHX_HIP_OK;
}

extern "C" void chx_hip_linear_plan_destroy(chx_hip_linear_plan* plan) {
    if (!plan) return;
    (void)hipFree(plan->w);
    delete plan;
}

extern "C" int chx_hip_linear_plan_workspace(const chx_hip_linear_plan* plan, const chx_hip_tensor* x, int64_t y_rows, size_t* bytes) {
    CHX_REQUIRE(bytes != nullptr, "linear plan: null output");
    *bytes = 0;
    CHX_REQUIRE(plan != nullptr, "linear plan: null plan");
    CHX_PROPAGATE(check_tensor(x, "linear plan x"));
    int64_t rows = 0, row_stride = 0;
    // (what a run refuses needs none)
    if (x->ndim < 1 || y_rows < 1 || x->shape[x->ndim - 1] != plan->K || !as_rows(*x, &rows, &row_stride) || rows < 1) return CHX_HIP_OK;
    const Choice c = choice_of(y_rows, plan->experts, rows, plan->N, plan->K, plan->type);
    const int64_t xe = plan->type == kFloatFloat ? 4 : 2;
    const bool direct = plan->K % (2 * unit_k(plan->type)) == 0 && x->strides[x->ndim - 1] == xe && aligned_rows(x->data, row_stride, rows, 16) && row_stride >= 0 && within_reach(row_stride, rows, plan->experts > 0);
    if (into_pieces(c, direct, rows, plan->K, plan->experts > 0, plan->type)) *bytes = (size_t)(pitch_of(plan->K, plan->type) * rows);
    return CHX_HIP_OK;
}

extern "C" int chx_hip_linear_plan_run(
        const chx_hip_linear_plan* plan, const chx_hip_tensor* x, int32_t activation, const chx_hip_tensor* r, chx_hip_tensor* y, void* workspace,
        size_t workspace_bytes, void* stream) {
    Call c;
    CHX_PROPAGATE(prepare_call(plan, x, activation, r, y, &c));
    CHX_REQUIRE(plan->experts == 0, "linear plan: the weights are experts': run_experts takes them");
    CHX_REQUIRE(x->ndim == y->ndim, "linear plan: x and y differ in their number of axes");
    for (int d = 0; d + 1 < x->ndim; ++d) CHX_REQUIRE(x->shape[d] == y->shape[d], "linear plan: x and y differ on axis %d", d);
    return launch_of(plan, c, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int chx_hip_linear_plan_run_experts(
        const chx_hip_linear_plan* plan, const chx_hip_tensor* x, const chx_hip_tensor* order, const chx_hip_tensor* offsets, int32_t activation,
        chx_hip_tensor* y, void* workspace, size_t workspace_bytes, void* stream) {
    Call c;
    CHX_PROPAGATE(prepare_call(plan, x, activation, nullptr, y, &c));
    CHX_REQUIRE(plan->experts > 0, "linear plan: the weights have no experts: run takes them");
    CHX_PROPAGATE(check_tensor(order, "linear plan order"));
    CHX_PROPAGATE(check_tensor(offsets, "linear plan offsets"));
    CHX_REQUIRE(x->ndim == 2 && y->ndim == 2, "linear plan: x and y must be matrices for experts");
    CHX_REQUIRE(order->dtype == CHX_HIP_INT32 && is_contiguous(*order) && numel(*order) == y->shape[0], "linear plan: order must be int32, contiguous, a number for each row of y");
    CHX_REQUIRE(offsets->dtype == CHX_HIP_INT32 && is_contiguous(*offsets) && numel(*offsets) == plan->experts + 1, "linear plan: offsets must be int32, contiguous, %d numbers",
                plan->experts + 1);
    CHX_REQUIRE(aligned(order->data, 4) && aligned(offsets->data, 4), "linear plan: order and offsets must begin at an element's address");
    if (y->shape[0] == 0) return CHX_HIP_OK;
    CHX_REQUIRE(x->shape[0] > 0 && y->shape[0] % x->shape[0] == 0, "linear plan: the rows of y must be a multiple of those of x");
    CHX_REQUIRE(!arrays_overlap(*order, *y) && !arrays_overlap(*offsets, *y), "linear plan: y overlaps order or offsets");
    c.a.order = static_cast<const int32_t*>(order->data);
    c.a.offsets = static_cast<const int32_t*>(offsets->data);
    c.a.experts = plan->experts;
    c.a.fan = (int32_t)(y->shape[0] / x->shape[0]);
    // (rows are gathered: all of x, and a block of 128 bytes behind its last row's beginning, within 32 bits)
    c.direct = c.direct && within_reach(c.a.x_row, x->shape[0], true);
    return launch_of(plan, c, workspace, workspace_bytes, as_stream(stream));
}
