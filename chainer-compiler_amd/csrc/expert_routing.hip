// Routing rows to experts, and the sum of what the experts made of a row.
//
//   s = softmax(x) or 1 / (1 + exp(-x)) over the E logits of a row;  key = s + bias
//   groups of E / G neighbours: a group's score is the sum of its best one or two keys; the experts of the best groups stay
//   the k largest keys, the lower index first where two are equal;  weight = s / (sum of the chosen s, if normalized) * scale
//   order: the places t * k + j by expert, within one in ascending order;  offsets: where each expert's begin
//
// A wavefront takes a row, its lanes the experts lane + 64 i.  Without a bias and groups the choice is made on the logits themselves, of which the
// keys are a monotonic function; else the keys are 64-bit numbers, so that which expert is chosen does not hang on how exp
// rounds.  Bound by latency: k times the largest of 64 lanes, which takes some 80 cycles through the lanes' data paths (DPP) where six exchanges through
// LDS take 400.
#include <cfloat>
#include <cstring>
#include <type_traits>

#include "chx_internal.h"

namespace chx {
namespace {

constexpr int kMostExperts = 1024, kMostChosen = 64, kMostGroups = 64;
// Wavefronts of a work-group (with 16 experts to a lane and keys in 64 bits, sixteen would have to spill registers)
constexpr int waves_of(int per) {
    return per > 8 ? 8 : 16;
}
// Rows that one launch takes: us for one / two launches over 256 experts with k = 8 and a bias, 16 rows 9.4 / 10.8 (host 7 / 10.6), 32 rows 16.1 / 10.8.  Without a bias, 16 rows in one / 17 in two: 64
// experts 4.5 / 5.8, 256 6.7 / 7.5, but 1024, where eight wavefronts have two rows each, 16.9 / 14.3.
constexpr int kMostChunks = 256, kSingleRows = 16;

struct RoutingArgs {
    const char* logits;
    int64_t row, col;  // bytes
    const float* bias;
    int32_t T, E, k, groups, top_groups, group_best;
    int32_t half, sigmoid, normalize;
    float scale;
    int32_t* experts;
    float* weights;
    int32_t* order;
    int32_t* offsets;
    int32_t* counts;  // [chunk][E]
    int32_t chunk;    // rows of a chunk
};

// Larger for larger numbers; a NaN (there is none among the logits any more) would be the largest.
__device__ __forceinline__ uint32_t sortable(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);  // (-0 is 0)
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t sortable(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}

// Reductions over the wavefront: within rows of 16 lanes, then from row to row; lane 63 has them all.
template <int kControl, int kRows>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kControl, kRows, 0xf, false);  // (0 where no lane is)
}
template <int kControl, int kRows>
__device__ __forceinline__ float moved(float v) {
    return __builtin_bit_cast(float, moved<kControl, kRows>(__builtin_bit_cast(uint32_t, v)));
}
template <int kControl, int kRows>
__device__ __forceinline__ double moved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)moved<kControl, kRows>((uint32_t)(b >> 32)) << 32 | moved<kControl, kRows>((uint32_t)b));
}
constexpr int kShift1 = 0x111, kShift2 = 0x112, kShift4 = 0x114, kShift8 = 0x118, kToNextRow = 0x142, kToUpperHalf = 0x143;

// (of numbers from 0 on)
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, moved<kShift1, 0xf>(v));
    v = max(v, moved<kShift2, 0xf>(v));
    v = max(v, moved<kShift4, 0xf>(v));
    v = max(v, moved<kShift8, 0xf>(v));
    v = max(v, moved<kToNextRow, 0xa>(v));
    v = max(v, moved<kToUpperHalf, 0xc>(v));
    return __builtin_amdgcn_readlane(v, 63);
}
// What the lanes up to this one have together.
template <typename T>
__device__ __forceinline__ T sum_up_to(T v) {
    v += moved<kShift1, 0xf>(v);
    v += moved<kShift2, 0xf>(v);
    v += moved<kShift4, 0xf>(v);
    v += moved<kShift8, 0xf>(v);
    v += moved<kToNextRow, 0xa>(v);
    v += moved<kToUpperHalf, 0xc>(v);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    return __shfl(sum_up_to(v), 63);
}
__device__ __forceinline__ float of_sortable(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// The choice for one row; lane j holds the j-th expert and its weight afterwards (j < k).  keys: LDS for E numbers of this wavefront.
template <int kPer, bool kExact>
__device__ void route(const RoutingArgs& a, int32_t t, double* keys, int32_t* expert, float* weight) {
    const int lane = threadIdx.x & 63;
    const char* row = a.logits + (int64_t)t * a.row;
    float x[kPer];
    uint32_t most_key = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 64 * i;
        x[i] = -INFINITY;
        if (e < a.E) {
            const char* p = row + e * a.col;
            const float v = a.half ? (float)*reinterpret_cast<const _Float16*>(p) : *reinterpret_cast<const float*>(p);
            x[i] = v != v ? -INFINITY : fminf(v, FLT_MAX);
        }
        most_key = max(most_key, sortable(x[i]));
    }
    const float most = of_sortable(wave_max(most_key));
    // (a row of nothing but -inf: no expert has a score)
    const float base = most == -INFINITY ? 0.f : most;
    typedef typename std::conditional<kExact, uint64_t, uint32_t>::type Key;
    Key key[kPer];  // 0: not to be had (any more)
    double sum = 0.0;  // of the softmax
    if constexpr (kExact) {
        double score[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane + 64 * i;
            score[i] = 0.0;
            if (e < a.E && x[i] != -INFINITY) score[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)base);
            sum += score[i];
        }
        if (!a.sigmoid) {
            sum = wave_sum(sum);
#pragma unroll
            for (int i = 0; i < kPer; ++i) score[i] = sum > 0.0 ? score[i] / sum : 0.0;
        }
        uint64_t taken = ~0ull;
        double v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane + 64 * i;
            v[i] = e < a.E ? score[i] + (a.bias ? (double)a.bias[e] : 0.0) : 0.0;
            if (v[i] != v[i]) v[i] = -INFINITY;
        }
        if (a.groups > 1) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (lane + 64 * i < a.E) keys[lane + 64 * i] = v[i];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int size = a.E / a.groups;
            double first = -INFINITY, second = -INFINITY;
            if (lane < a.groups) {
#pragma unroll 8
                for (int i = 0; i < size; ++i) {
                    const double o = keys[lane * size + i];
                    second = fmax(second, fmin(first, o));
                    first = fmax(first, o);
                }
            }
            double of_group = a.group_best > 1 ? first + second : first;
            if (of_group != of_group) of_group = -INFINITY;
            const uint64_t mine = lane < a.groups ? sortable(of_group) : 0;
            int before = 0;
            for (int g = 0; g < a.groups; ++g) {
                const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), g) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, g);
                before += other > mine || (other == mine && g < lane);
            }
            taken = __builtin_amdgcn_ballot_w64(lane < a.groups && before < a.top_groups);
            __builtin_amdgcn_wave_barrier();
            const float of_size = 1.f / (float)size;  // (e / size, exactly: (e + 0.5) / size is 0.5 / size or more from a border, the product off by 2^-22 of itself)
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int e = lane + 64 * i;
                key[i] = e < a.E && ((taken >> (int)(((float)e + 0.5f) * of_size)) & 1) ? sortable(v[i]) : 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) key[i] = lane + 64 * i < a.E ? sortable(v[i]) : 0;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = lane + 64 * i < a.E ? sortable(x[i]) : 0;
    }
    int32_t chosen = 0;
    float of_chosen = -INFINITY;  // its logit
    for (int j = 0; j < a.k; ++j) {
        // this lane's best, the largest of all, and the lowest index among those that have it
        Key best = key[0];
        int32_t at = lane;
        float value = x[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) {
            const bool better = key[i] > best;
            best = better ? key[i] : best;
            at = better ? lane + 64 * i : at;
            value = better ? x[i] : value;
        }
        const uint32_t upper = kExact ? (uint32_t)((uint64_t)best >> 32) : (uint32_t)best;
        const uint32_t most_upper = wave_max(upper);
        uint64_t with = __builtin_amdgcn_ballot_w64(upper == most_upper);
        if (with & (with - 1)) {
            bool mine = upper == most_upper;
            if constexpr (kExact) {
                const uint32_t most_lower = wave_max(mine ? (uint32_t)best : 0);
                mine = mine && (uint32_t)best == most_lower;
            }
            const uint32_t lowest = wave_max(mine ? (uint32_t)~at : 0);
            with = __builtin_amdgcn_ballot_w64(mine && (uint32_t)~at == lowest);
        }
        const int from = __builtin_ctzll(with);
        const int32_t which = __builtin_amdgcn_readlane(at, from);
        const float of_which = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, value), from));
        chosen = lane == j ? which : chosen;
        of_chosen = lane == j ? of_which : of_chosen;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (lane + 64 * i == which) key[i] = 0;
    }
    if (kExact || a.sigmoid) {
        // (Scores that only 64 bits hold still share a row among them, so the rounding to 32 comes last: with scores rounded first, rows whose logits all lay
        // below -88 lost their experts.  A lane has one chosen expert, so this is one exponential and one division of 64 bits to a row.)
        double w = 0.0;
        if (lane < a.k && of_chosen != -INFINITY) {
            w = a.sigmoid ? 1.0 / (1.0 + exp(-(double)of_chosen)) : exp((double)of_chosen - (double)base);
            if (!a.sigmoid) w = w / sum;
        }
        if (a.normalize) {
            const double all = wave_sum(w);
            w = all > 0.0 ? w / all : 0.0;
        }
        *weight = (float)(w * (double)a.scale);
    } else {
        float w = lane < a.k ? expf(of_chosen - base) : 0.f;
        if (!a.normalize) {
            float all = 0.f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) all += expf(x[i] - base);
            all = wave_sum(all);
            w = all > 0.f ? w / all : 0.f;
        } else {
            // (the largest logit is among the chosen: their sum is 1 or more, or 0 in a row without any)
            const float all = wave_sum(w);
            w = all > 0.f ? w / all : 0.f;
        }
        *weight = w * a.scale;
    }
    *expert = chosen;
}

// The places [first, first + count) of the routing into the order, ascending; one wavefront.  at: LDS, where each expert's next place goes.
__device__ void put_in_order(const int32_t* experts, int32_t first, int32_t count, int32_t* at, int32_t* order, int32_t bits) {
    const int lane = threadIdx.x & 63;
    for (int32_t i0 = 0; i0 < count; i0 += 64) {
        const int32_t i = i0 + lane;
        const bool there = i < count;
        const int32_t e = there ? experts[i] : 0;
        uint64_t same = __builtin_amdgcn_ballot_w64(there);  // the lanes with this one's expert
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __builtin_amdgcn_ballot_w64((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        const uint64_t before = same & ((1ull << lane) - 1);
        if (there) order[at[e] + __popcll(before)] = first + i;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (there && before == 0) at[e] += __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Sums of the counts of the experts before each; E of them in LDS, one wavefront.
__device__ void sums_before(int32_t* counts, int32_t E, int32_t* total) {
    const int lane = threadIdx.x & 63;
    int32_t carry = 0;
    for (int32_t e0 = 0; e0 < E; e0 += 64) {
        const int32_t n = e0 + lane < E ? counts[e0 + lane] : 0;
        const int32_t upto = (int32_t)sum_up_to((uint32_t)n);
        if (e0 + lane < E) counts[e0 + lane] = carry + upto - n;
        carry += __builtin_amdgcn_readlane(upto, 63);
    }
    *total = carry;
}

__device__ __forceinline__ int32_t bits_of(int32_t E) {
    return E > 1 ? 32 - __builtin_clz(E - 1) : 0;
}

// Few rows: everything in one work-group.
template <int kPer, bool kExact>
__global__ __launch_bounds__(64 * waves_of(kPer)) void routing_single_kernel(RoutingArgs a) {
    __shared__ double keys[waves_of(kPer)][kExact ? 64 * kPer : 1];
    __shared__ int32_t counts[64 * kPer];
    __shared__ int32_t chosen[kSingleRows * kMostChosen];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < a.E; e += 64 * waves_of(kPer)) counts[e] = 0;
    __syncthreads();
    for (int32_t t = wave; t < a.T; t += waves_of(kPer)) {
        int32_t e;
        float w;
        route<kPer, kExact>(a, t, keys[wave], &e, &w);
        if (lane < a.k) {
            a.experts[(int64_t)t * a.k + lane] = e;
            a.weights[(int64_t)t * a.k + lane] = w;
            chosen[t * a.k + lane] = e;
            atomicAdd(&counts[e], 1);
        }
    }
    __syncthreads();
    if (wave != 0) return;
    int32_t total;
    sums_before(counts, a.E, &total);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int e = lane; e < a.E; e += 64) a.offsets[e] = counts[e];
    if (lane == 0) a.offsets[a.E] = total;
    put_in_order(chosen, 0, a.T * a.k, counts, a.order, bits_of(a.E));
}

// Many rows: a chunk of them to a work-group, which counts how many went to each expert ...
template <int kPer, bool kExact>
__global__ __launch_bounds__(64 * waves_of(kPer)) void routing_kernel(RoutingArgs a) {
    __shared__ double keys[waves_of(kPer)][kExact ? 64 * kPer : 1];
    __shared__ int32_t counts[64 * kPer];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < a.E; e += 64 * waves_of(kPer)) counts[e] = 0;
    __syncthreads();
    // (unsigned: with close to 2^31 rows, a chunk's end and the step behind it lie above)
    const uint32_t begin = blockIdx.x * (uint32_t)a.chunk, end = min(begin + (uint32_t)a.chunk, (uint32_t)a.T);
    for (uint32_t t = begin + wave; t < end; t += waves_of(kPer)) {
        int32_t e;
        float w;
        route<kPer, kExact>(a, (int32_t)t, keys[wave], &e, &w);
        if (lane < a.k) {
            a.experts[(int64_t)t * a.k + lane] = e;
            a.weights[(int64_t)t * a.k + lane] = w;
            atomicAdd(&counts[e], 1);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += 64 * waves_of(kPer)) a.counts[(int64_t)blockIdx.x * a.E + e] = counts[e];
}

// ... and one that adds up what the chunks before its own have, and puts its places in order.
__global__ __launch_bounds__(1024) void routing_order_kernel(RoutingArgs a) {
    __shared__ int32_t at[kMostExperts], before[kMostExperts];
    for (int e = threadIdx.x; e < a.E; e += 1024) at[e] = before[e] = 0;
    __syncthreads();
    const int chunks = gridDim.x;
    // (several threads to an expert, eight loads of each under way)
    const int share = 1024 / a.E, e = threadIdx.x % a.E, part = threadIdx.x / a.E;
    if (part < share) {
        int32_t all = 0, earlier = 0;
#pragma unroll 8
        for (int c = part; c < chunks; c += share) {
            const int32_t n = a.counts[(int64_t)c * a.E + e];
            all += n;
            earlier += c < (int)blockIdx.x ? n : 0;
        }
        atomicAdd(&at[e], all);
        atomicAdd(&before[e], earlier);
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    int32_t total;
    sums_before(at, a.E, &total);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int e = threadIdx.x; e < a.E; e += 64) {
        if (blockIdx.x == 0) a.offsets[e] = at[e];
        at[e] += before[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = total;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t begin = blockIdx.x * (uint32_t)a.chunk, end = min(begin + (uint32_t)a.chunk, (uint32_t)a.T);
    put_in_order(a.experts + (int64_t)begin * a.k, (int32_t)(begin * a.k), (int32_t)((end - begin) * a.k), at, a.order, bits_of(a.E));
}

template <int kPer>
void launch_routing(const RoutingArgs& a, bool exact, int32_t chunks, hipStream_t s) {
    if (chunks == 0) {
        if (exact) routing_single_kernel<kPer, true><<<1, 64 * waves_of(kPer), 0, s>>>(a);
        else routing_single_kernel<kPer, false><<<1, 64 * waves_of(kPer), 0, s>>>(a);
        return;
    }
    if (exact) routing_kernel<kPer, true><<<(unsigned)chunks, 64 * waves_of(kPer), 0, s>>>(a);
    else routing_kernel<kPer, false><<<(unsigned)chunks, 64 * waves_of(kPer), 0, s>>>(a);
}

// Rows to a chunk: as many chunks as there may be, of 4 rows at least.
int32_t rows_of_chunk(int64_t T) {
    const int64_t rows = (T + kMostChunks - 1) / kMostChunks;
    return (int32_t)((rows + 3) / 4 * 4);
}

int64_t workspace_of(int64_t T, int64_t E) {
    if (T <= kSingleRows) return 0;
    const int64_t rows = rows_of_chunk(T);
    return (T + rows - 1) / rows * E * 4;
}

// ---- the weighted sum -------------------------------------------------------------------------------

struct CombineArgs {
    const char* x;
    const float* weights;
    const char* r;
    char* y;
    int64_t x_row, x_col, r_row, r_col, y_row, y_col;  // bytes
    int64_t pieces, total;                              // of kWidth columns
    int64_t first;                                      // work-group of this launch
    int32_t N, k;
};

template <typename T, int kWidth>
__device__ __forceinline__ void load_piece(const char* p, int64_t col, float* v) {
    if constexpr (kWidth > 1) {
        T h[kWidth];
        __builtin_memcpy(h, __builtin_assume_aligned(p, kWidth * sizeof(T)), kWidth * sizeof(T));
#pragma unroll
        for (int i = 0; i < kWidth; ++i) v[i] = (float)h[i];
    } else {
        v[0] = (float)*reinterpret_cast<const T*>(p);
    }
}

// Bound by bytes, each of x read once: a lane has 16 bytes of every row of a sum under way at a time (four rows; kWidth 1: one element, for arrays of other strides and alignments).
// 8192 x 4 x 4096 in float16 73 us, 5.5 TB/s; an element a lane, 4097 columns, 130 us; in float32 145 and 150.
template <typename T, int kWidth>
__global__ __launch_bounds__(256) void expert_combine_kernel(CombineArgs a) {
    const int64_t at = (a.first + blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.total) return;
    const int64_t t = at / a.pieces, n = (at - t * a.pieces) * kWidth;
    const char* x = a.x + t * a.k * a.x_row + n * a.x_col;
    const float* w = a.weights + t * a.k;
    float sum[kWidth];
#pragma unroll
    for (int i = 0; i < kWidth; ++i) sum[i] = 0.f;
    int j = 0;
    for (; j + 4 <= a.k; j += 4) {
        float v[4][kWidth];
#pragma unroll
        for (int q = 0; q < 4; ++q) load_piece<T, kWidth>(x + (j + q) * a.x_row, a.x_col, v[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float f = w[j + q];
#pragma unroll
            for (int i = 0; i < kWidth; ++i) sum[i] = f != 0.f ? __builtin_fmaf(f, v[q][i], sum[i]) : sum[i];
        }
    }
    for (; j < a.k; ++j) {
        float v[kWidth];
        load_piece<T, kWidth>(x + j * a.x_row, a.x_col, v);
        const float f = w[j];
#pragma unroll
        for (int i = 0; i < kWidth; ++i) sum[i] = f != 0.f ? __builtin_fmaf(f, v[i], sum[i]) : sum[i];
    }
    if (a.r) {
        float v[kWidth];
        load_piece<T, kWidth>(a.r + t * a.r_row + n * a.r_col, a.r_col, v);
#pragma unroll
        for (int i = 0; i < kWidth; ++i) sum[i] += v[i];
    }
    char* y = a.y + t * a.y_row + n * a.y_col;
    T h[kWidth];
#pragma unroll
    for (int i = 0; i < kWidth; ++i) h[i] = (T)sum[i];
    if constexpr (kWidth > 1) __builtin_memcpy(__builtin_assume_aligned(y, kWidth * sizeof(T)), h, kWidth * sizeof(T));
    else *reinterpret_cast<T*>(y) = h[0];
}

int check_float(const chx_hip_tensor* t, const char* op, const char* name) {
    CHX_PROPAGATE(check_tensor(t, op));
    const int64_t es = dtype_size(t->dtype);
    CHX_REQUIRE(t->dtype == CHX_HIP_FLOAT16 || t->dtype == CHX_HIP_FLOAT32, "%s: %s must be float16 or float32, not %s", op, name, dtype_name(t->dtype));
    CHX_REQUIRE(t->ndim == 2, "%s: %s must be a matrix", op, name);
    CHX_REQUIRE(aligned(t->data, (size_t)es) && t->strides[0] % es == 0 && t->strides[1] % es == 0, "%s: %s is not made of whole elements", op, name);
    return CHX_HIP_OK;
}

int check_dense(const chx_hip_tensor* t, int32_t dtype, int64_t elements, const char* op, const char* name) {
    CHX_PROPAGATE(check_tensor(t, op));
    CHX_REQUIRE(t->dtype == dtype && numel(*t) == elements && (elements == 0 || is_contiguous(*t)) && aligned(t->data, (size_t)dtype_size(dtype)), "%s: %s must be %s, contiguous, %lld elements", op,
                name, dtype_name(dtype), (long long)elements);
    return CHX_HIP_OK;
}

}  // namespace
}  // namespace chx

using namespace chx;

extern "C" int chx_hip_expert_routing_workspace(int64_t rows, int64_t experts, size_t* bytes) {
    CHX_REQUIRE(bytes != nullptr, "expert routing: null output");
    CHX_REQUIRE(rows >= 0 && experts >= 1 && experts <= kMostExperts, "expert routing: at most %d experts", kMostExperts);
    *bytes = (size_t)workspace_of(rows, experts);
    return CHX_HIP_OK;
}

extern "C" int chx_hip_expert_routing(
        const chx_hip_tensor* logits, const chx_hip_tensor* bias, int32_t sigmoid, int32_t groups, int32_t top_groups, int32_t group_best,
        int32_t normalize, float scale, chx_hip_tensor* experts, chx_hip_tensor* weights, chx_hip_tensor* order, chx_hip_tensor* offsets,
        void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "expert routing";
    CHX_PROPAGATE(check_float(logits, op, "logits"));
    const int64_t T = logits->shape[0], E = logits->shape[1];
    CHX_REQUIRE(E >= 1 && E <= kMostExperts, "%s: 1 to %d experts, not %lld", op, kMostExperts, (long long)E);
    CHX_PROPAGATE(check_tensor(experts, op));
    CHX_REQUIRE(experts->ndim == 2, "%s: experts must be a matrix", op);
    const int64_t k = experts->shape[1];
    CHX_REQUIRE(k >= 1 && k <= kMostChosen && k <= E, "%s: 1 to %d experts are chosen, and no more than there are, not %lld", op, kMostChosen, (long long)k);
    CHX_REQUIRE(T * k < (int64_t(1) << 31), "%s: 2^31 places or more", op);
    CHX_REQUIRE(groups >= 1 && groups <= kMostGroups && E % groups == 0, "%s: 1 to %d groups of equal size, not %d", op, kMostGroups, groups);
    CHX_REQUIRE(top_groups >= 1 && top_groups <= groups && k <= top_groups * (E / groups), "%s: %d groups have no %lld experts", op, top_groups, (long long)k);
    CHX_REQUIRE(group_best == 1 || (group_best == 2 && E / groups >= 2), "%s: a group's score is of one or two of its experts", op);
    CHX_PROPAGATE(check_dense(experts, CHX_HIP_INT32, T * k, op, "experts"));
    CHX_PROPAGATE(check_dense(weights, CHX_HIP_FLOAT32, T * k, op, "weights"));
    CHX_PROPAGATE(check_dense(order, CHX_HIP_INT32, T * k, op, "order"));
    CHX_PROPAGATE(check_dense(offsets, CHX_HIP_INT32, E + 1, op, "offsets"));
    if (bias != nullptr) CHX_PROPAGATE(check_dense(bias, CHX_HIP_FLOAT32, E, op, "bias"));
    CHX_REQUIRE((int64_t)workspace_bytes >= workspace_of(T, E) && (workspace_of(T, E) == 0 || (workspace != nullptr && aligned(workspace, 4))),
                "%s: a workspace of %lld bytes is needed", op, (long long)workspace_of(T, E));
    RoutingArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = static_cast<const char*>(logits->data);
    a.row = logits->strides[0];
    a.col = logits->strides[1];
    a.bias = bias ? static_cast<const float*>(bias->data) : nullptr;
    a.T = (int32_t)T;
    a.E = (int32_t)E;
    a.k = (int32_t)k;
    a.groups = groups;
    a.top_groups = top_groups;
    a.group_best = group_best;
    a.half = logits->dtype == CHX_HIP_FLOAT16;
    a.sigmoid = sigmoid != 0;
    a.normalize = normalize != 0;
    a.scale = scale;
    a.experts = static_cast<int32_t*>(experts->data);
    a.weights = static_cast<float*>(weights->data);
    a.order = static_cast<int32_t*>(order->data);
    a.offsets = static_cast<int32_t*>(offsets->data);
    a.counts = static_cast<int32_t*>(workspace);
    a.chunk = rows_of_chunk(T);
    const bool exact = a.bias != nullptr || groups > 1;
    const int32_t chunks = T <= kSingleRows ? 0 : (int32_t)((T + a.chunk - 1) / a.chunk);
    const hipStream_t s = as_stream(stream);
    if (E <= 64) launch_routing<1>(a, exact, chunks, s);
    else if (E <= 128) launch_routing<2>(a, exact, chunks, s);
    else if (E <= 256) launch_routing<4>(a, exact, chunks, s);
    else if (E <= 512) launch_routing<8>(a, exact, chunks, s);
    else launch_routing<16>(a, exact, chunks, s);
    CHX_PROPAGATE(launch_check("routing_kernel"));
    if (chunks == 0) return CHX_HIP_OK;
    routing_order_kernel<<<(unsigned)chunks, 1024, 0, s>>>(a);
    return launch_check("routing_order_kernel");
}

extern "C" int chx_hip_expert_combine(const chx_hip_tensor* x, const chx_hip_tensor* weights, const chx_hip_tensor* r, chx_hip_tensor* y, void* stream) {
    const char* op = "expert combine";
    CHX_PROPAGATE(check_float(x, op, "x"));
    CHX_PROPAGATE(check_float(y, op, "y"));
    CHX_PROPAGATE(check_tensor(weights, op));
    CHX_REQUIRE(weights->ndim == 2 && weights->shape[1] >= 1, "%s: weights must be [rows, k]", op);
    const int64_t T = weights->shape[0], k = weights->shape[1], N = x->shape[1];
    CHX_PROPAGATE(check_dense(weights, CHX_HIP_FLOAT32, T * k, op, "weights"));
    CHX_REQUIRE(k < (1 << 20) && x->shape[0] == T * k, "%s: x must have %lld rows", op, (long long)(T * k));
    CHX_REQUIRE(y->dtype == x->dtype && y->shape[0] == T && y->shape[1] == N, "%s: y must be [%lld, %lld], of the type of x", op, (long long)T, (long long)N);
    if (r != nullptr) {
        CHX_PROPAGATE(check_float(r, op, "r"));
        CHX_REQUIRE(r->dtype == y->dtype && same_shape(*r, *y), "%s: r must have the type and shape of y", op);
    }
    if (T == 0 || N == 0) return CHX_HIP_OK;
    CHX_REQUIRE(elements_apart(*y), "%s: elements of y overlap", op);
    CHX_REQUIRE(!arrays_overlap(*x, *y) && !arrays_overlap(*weights, *y), "%s: y overlaps x or weights", op);
    CHX_REQUIRE(r == nullptr || same_array(*r, *y) || !arrays_overlap(*r, *y), "%s: r and y overlap and are not the same array", op);
    CombineArgs a;
    memset(&a, 0, sizeof(a));
    const int64_t es = dtype_size(x->dtype);
    bool wide = N % (16 / es) == 0;
    auto take = [&](const chx_hip_tensor& t, int64_t* row, int64_t* col) {
        *row = t.strides[0];
        *col = t.strides[1];
        wide = wide && aligned(t.data, 16) && (t.shape[0] == 1 || t.strides[0] % 16 == 0) && (N == 1 || t.strides[1] == es);
    };
    take(*x, &a.x_row, &a.x_col);
    take(*y, &a.y_row, &a.y_col);
    if (r) take(*r, &a.r_row, &a.r_col);
    a.x = static_cast<const char*>(x->data);
    a.weights = static_cast<const float*>(weights->data);
    a.r = r ? static_cast<const char*>(r->data) : nullptr;
    a.y = static_cast<char*>(y->data);
    a.N = (int32_t)N;
    a.k = (int32_t)k;
    a.pieces = wide ? N / (16 / es) : N;
    a.total = T * a.pieces;
    const hipStream_t s = as_stream(stream);
    return in_launches((a.total + 255) / 256, "expert_combine_kernel", [&](int64_t first, unsigned count) {
        a.first = first;
        if (es == 2) {
            if (wide) expert_combine_kernel<_Float16, 8><<<count, 256, 0, s>>>(a);
            else expert_combine_kernel<_Float16, 1><<<count, 256, 0, s>>>(a);
        } else {
            if (wide) expert_combine_kernel<float, 4><<<count, 256, 0, s>>>(a);
            else expert_combine_kernel<float, 1><<<count, 256, 0, s>>>(a);
        }
    });
}
