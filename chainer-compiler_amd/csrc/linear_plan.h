// Products with an epilogue from a plan (linear_plan.hip): what the host hands to the kernels, and the order of the laid-out weights.
#pragma once

#include "chx_internal.h"

namespace chx {

enum LinearType { kHalfHalf = 0, kHalfInt8 = 1, kFloatFloat = 2 };  // x and w

// Weights [N, K] are laid out in groups of 64 rows, along k in units that belong to 64 bytes of a row of x, a unit as four fragments: the
// operand of one matrix instruction (16 rows; four instructions' for float32), a lane's bytes together.
//   float16  32 k a unit: 16 bytes of lane l hold k = 8 (l / 16) + j;  a fragment is 1 KB
//   float32  16 k a unit: k = 4 (l / 16) + j; instruction j of the unit takes the k that are j modulo 4
//   int8     32 k a unit, as for float16 with 8 bytes; those of fragments 2 p and 2 p + 1 are next to each other, 16 bytes of a lane
// Row r of fragment f is row 16 (r / 4) + 4 f + r % 4 of the group: a lane of the result then holds 16 neighbouring columns, 32 bytes of
// float16, and four lanes a whole line.  K is filled up with zeros to whole blocks of two units (128 bytes of x), N to whole groups.
constexpr int kGroupRows = 64;

__host__ __device__ constexpr int unit_bytes(LinearType t) {
    return t == kHalfInt8 ? 2048 : 4096;
}
__host__ __device__ constexpr int unit_k(LinearType t) {
    return t == kFloatFloat ? 16 : 32;
}

__host__ __device__ inline int group_row(int fragment, int r) {
    return 16 * (r >> 2) + 4 * fragment + (r & 3);
}

// The tiles of experts that one XCD takes together: kPieceRows of rows times kPieceColumns, or of so many columns less that as few as may be are missing
// from the last piece (work-groups without a tile, a quarter of all where three columns were counted as four: 2048 rows to 8 of 128 experts of 2048 x 768 164 us instead of
// 188, 4096 rows to 8 of 64 of 2048 x 1280 217 instead of 269).
constexpr int32_t kPieceRows = 2, kPieceColumns = 4;
__host__ __device__ inline int32_t piece_columns(int32_t tiles_n) {
    const int32_t across = (tiles_n + kPieceColumns - 1) / kPieceColumns;
    return (tiles_n + across - 1) / across;
}
// Work-groups for them: whole pieces, the same number for each XCD.
inline int64_t expert_grid(int64_t tiles_m, int64_t tiles_n) {
    const int64_t wide = piece_columns((int32_t)tiles_n), pieces = (tiles_m + kPieceRows - 1) / kPieceRows * ((tiles_n + wide - 1) / wide);
    return (pieces + 7) / 8 * 8 * kPieceRows * wide;
}

struct LinearArgs {
    const char* x;
    const char* w;
    const float* scale;  // of int8 rows, [N], or null
    const float* bias;   // [N] or null
    const char* r;       // residual or null
    char* y;
    int64_t x_row, x_col, r_row, r_col, y_row, y_col;  // bytes
    int64_t w_group, w_expert;                          // bytes from one group, one expert, to the next
    int32_t M, N, K, units;                             // units: of laid-out weights along k, an even number
    int32_t activation, y_half;                         // y_half: y and r are float16
    int32_t vector_y, vector_r;                         // 16 bytes of neighbouring columns at a time
    int32_t tiles_m, tiles_n;
    // rows that a routing has sent to experts: M of them
    const int32_t* order;
    const int32_t* offsets;
    int32_t experts, fan, n_padded;
};

// The kernels, by the types of x and w (linear_half.hip, linear_int8.hip, linear_float.hip).  `rows`: few rows, weights straight into
// registers; `tile`: both operands through LDS.  `direct`: x lies in rows of whole blocks that can be
// copied in 16-byte pieces (for tiles it does).
enum LinearTile { kTile256 = 0, kTile128 = 1, kTile64 = 2 };  // 256 x 256, 128 x 128, 64 x 128 (rows x columns); float32 has the last one alone
template <LinearType kType>
struct LinearKernels {
    static int rows(const LinearArgs& a, int row_tiles, int fragments, bool direct, hipStream_t s);
    static int tile(const LinearArgs& a, LinearTile t, hipStream_t s);
};

}  // namespace chx
