// Log probabilities of given tokens, the entropy of each row of logits, and the best alternatives.
//
//   m = max x;  s = sum exp(x - m);  t = sum (x - m) exp(x - m)          over a row's V logits
//   log p(token) = x[token] - m - log s;   entropy = log s - t / s;      alternatives: the `top` largest logits, the lower index first
//
// Bound by the bytes of the logits: one pass with a running maximum, four loads of 16 bytes a lane under way.  Where rows are few, work-groups share a row and
// a second launch joins their parts, in one order; where they are many and short, each wavefront has a row of its own.
//
// The arithmetic is what comes next: a float16 logit takes 8 issue slots of a lane (4 of them the exponential), which keep the vector
// units busy for 60 us of 4096 rows of 65,536.  Their sums are therefore kept relative to a number M in units of log 2, the rounded m log2(e): y = x log2(e) - M is one fused
// multiply-add that also converts x, exact to its own rounding, and M drops out at the end (whole_row).  (float32 logits may be too large for that product: x - m first.)
//
// The alternatives are found in the same pass.  What is below a threshold cannot be among the `top` best: the top-th largest of the maxima that the
// lanes found in their first 32 logits has top logits at or above it.  32 logits of a lane are compared by their maximum alone; what
// passes goes to a list in LDS, and the lists are ranked at the end by counting, for every entry, those before it.
#include <cfloat>
#include <cmath>
#include <cstring>

#include "chx_internal.h"

namespace chx {
namespace {

constexpr int kMostTop = 64, kWaves = 4;
constexpr int kKept = 256, kList = kKept + 512;  // entries of a wavefront's list: it is cut when there are more than kKept, and 512 more may come in between
constexpr int kLoads = 4;                        // of 16 bytes (float16), 32 (float32): 8 logits each
constexpr int kBlock = 64 * 8 * kLoads;          // logits of a wavefront's step
constexpr int kMostParts = 64;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

struct Sums;

struct LogprobArgs {
    const char* logits;
    int64_t row, col;  // bytes
    const char* tokens;
    int32_t half, token64;
    int64_t token_col;
    int32_t V, top, parts, part;  // part: logits of a part, a multiple of kWaves * kBlock where there are several
    int64_t R;
    float* logprob;
    float* entropy;
    float* top_logprob;
    int64_t* top_token;
    Sums* sums;  // of the parts: [row][part]
    uint64_t* lists;    // [row][part][top], best first, zeros where a part has none
};

__device__ __forceinline__ uint32_t sortable(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);  // (-0 is 0)
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_sortable(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
// Order of the alternatives: the larger logit, then the lower index.
__device__ __forceinline__ uint64_t entry_of(float v, int32_t index) {
    return (uint64_t)sortable(v) << 32 | (uint32_t)~index;
}

// Sums of 2^y and y 2^y over logits x: y = x log2(e) - m for float16, (x - m) log2(e) for float32.
struct Sums {
    float m, s, t;
};
constexpr float kNoMaximum[2] = {-FLT_MAX, -1e6f};  // [kHalf]: below every m, and its differences are finite or give 0

template <bool kHalf>
__device__ __forceinline__ float log2_of(float x, float m) {
    return kHalf ? __builtin_fmaf(x, kLog2e, -m) : (x - m) * kLog2e;
}
template <bool kHalf>
__device__ __forceinline__ float maximum_of(float x) {
    return kHalf ? x * kLog2e : x;
}

// A row's sums when they are whole: s and t relative to the largest logit itself, low: what m lacks of it.  M is the rounded m log2(e), so the largest logit's term is 2^low and not 1;
// left in, a token that is certain had a log probability of up to 1e-7 instead of 0, above 0 as often as below.  The largest logit is the float16 number next to M / log2(e): M is off
// by 2^-24 of itself, and such numbers are 2^-11 apart.
struct Row {
    float m, low, s, t;
};
template <bool kHalf>
__device__ __forceinline__ Row whole_row(const Sums& z) {
    if (!kHalf || z.s == 0.f) return {z.m, 0.f, z.s, z.t};
    const float low = log2_of<true>((float)(_Float16)(z.m * kLn2), z.m), one = __builtin_amdgcn_exp2f(low);
    return {z.m, low, z.s / one, (z.t - low * z.s) / one};  // (of that term alone exactly 1 and 0)
}

// x less the largest logit, as a natural logarithm.
template <bool kHalf>
__device__ __forceinline__ float log_of(float x, const Row& z) {
    return kHalf ? (log2_of<true>(x, z.m) - z.low) * kLn2 : x - z.m;
}

// The sums relative to a larger maximum.
template <bool kHalf>
__device__ __forceinline__ void move_to(Sums& z, float m) {
    const float y = kHalf ? z.m - m : (z.m - m) * kLog2e, f = __builtin_amdgcn_exp2f(y);
    z.t = f == 0.f ? 0.f * z.s : (z.t + y * z.s) * f;  // (y may be -inf; a NaN stays one)
    z.s = z.s * f;
    z.m = m;
}

// Of all lanes, in every lane.
template <bool kHalf>
__device__ __forceinline__ void join_lanes(Sums& z) {
    float m = z.m;
#pragma unroll
    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    move_to<kHalf>(z, m);
#pragma unroll
    for (int d = 32; d; d /= 2) {
        z.s += __shfl_xor(z.s, d);
        z.t += __shfl_xor(z.t, d);
    }
}

// The `top` best of more than that many entries of one wavefront, kept at the front of its list; returns the least of them.  kKept entries are held in
// registers; more of them, which takes logits that rise for thousands, are read again and again, so that the loop over the logits
// does not pay for registers that it hardly ever needs.
template <bool kFew>
__device__ __forceinline__ uint64_t cut_list(uint64_t* list, int32_t count, int32_t top) {
    constexpr int kHeld = kFew ? kKept / 64 : 1;
    const int lane = threadIdx.x & 63;
    uint64_t mine[kHeld];
    if constexpr (kFew) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) mine[i] = 64 * i + lane < count ? list[64 * i + lane] : 0;
    }
    // the top-th largest, bit by bit: no two entries are equal
    uint64_t least = 0;
    for (int b = 63; b >= 0; --b) {
        const uint64_t try_at = least | 1ull << b;
        int n = 0;
        if constexpr (kFew) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(mine[i] >= try_at));
        } else {
            for (int i = lane; i - lane < count; i += 64) n += __popcll(__builtin_amdgcn_ballot_w64(i < count && list[i] >= try_at));
        }
        if (n >= top) least = try_at;
    }
    int32_t at = 0;
    auto keep = [&](uint64_t entry, bool there) {
        const uint64_t kept = __builtin_amdgcn_ballot_w64(there && entry >= least);
        if ((kept >> lane) & 1) list[at + __popcll(kept & ((1ull << lane) - 1))] = entry;
        at += __popcll(kept);
    };
    if constexpr (kFew) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) keep(mine[i], mine[i] != 0);
    } else {
        for (int i = lane; i - lane < count; i += 64) keep(i < count ? list[i] : 0, i < count);  // (never ahead of what is read)
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return least;
}

// How many of a list's entries come before `mine`.
__device__ __forceinline__ int32_t before_in(const uint64_t* list, int32_t count, uint64_t mine) {
    int32_t n = 0;
#pragma unroll 8
    for (int32_t i = 0; i < count; ++i) n += list[i] > mine;
    return n;
}

// A row's token and its logit: two loads one after the other, asked for before the sums are there.
struct Given {
    float logit, in_place_of;  // in_place_of: 0 without a token, NaN for one that the row does not have, else 1
};
template <bool kHalf>
__device__ __forceinline__ Given given(const LogprobArgs& a, int64_t row) {
    if (!a.logprob) return {0.f, 0.f};
    const char* p = a.tokens + row * a.token_col;
    const int64_t token = a.token64 ? *reinterpret_cast<const int64_t*>(p) : *reinterpret_cast<const int32_t*>(p);
    if (token < 0 || token >= a.V) return {0.f, token < 0 ? 0.f : NAN};
    const char* q = a.logits + row * a.row + token * a.col;
    return {kHalf ? (float)*reinterpret_cast<const _Float16*>(q) : *reinterpret_cast<const float*>(q), 1.f};
}

// What is reported for a row: of its token and its entropy by one lane, of an alternative by whoever has it.
template <bool kHalf>
__device__ __forceinline__ void report_row(const LogprobArgs& a, int64_t row, const Row& z, const Given& g) {
    // (no logit above -inf: no token has a probability)
    const bool none = z.s == 0.f;
    const float log_s = none ? 0.f : logf(z.s);
    if (a.logprob) a.logprob[row] = g.in_place_of != 1.f ? g.in_place_of : none ? -INFINITY : log_of<kHalf>(g.logit, z) - log_s;
    const float entropy = none ? 0.f : log_s - kLn2 * z.t / z.s;
    a.entropy[row] = entropy < 0.f ? 0.f : entropy;  // (a NaN stays)
}

template <bool kHalf>
__device__ __forceinline__ void report_best(const LogprobArgs& a, int64_t row, const Row& z, int32_t rank, uint64_t entry) {
    const bool none = z.s == 0.f;
    a.top_logprob[row * a.top + rank] = none ? -INFINITY : log_of<kHalf>(of_sortable((uint32_t)(entry >> 32)), z) - logf(z.s);
    a.top_token[row * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)entry;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

// Eight logits as they lie in memory, from index i on; -inf from `end` on.
template <bool kHalf>
struct Eight {
    u32x4 v[kHalf ? 1 : 2];
    __device__ __forceinline__ void load(const char* p) {
        v[0] = reinterpret_cast<const u32x4_any*>(p)[0];
        if constexpr (!kHalf) v[1] = reinterpret_cast<const u32x4_any*>(p)[1];
    }
    __device__ __forceinline__ void load_some(const char* row, int64_t col, int32_t i, int32_t end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const char* p = row + (int64_t)(i + j) * col;
            if constexpr (kHalf) {
                const uint32_t h = i + j < end ? *reinterpret_cast<const uint16_t*>(p) : 0xfc00u;
                v[0][j / 2] = j & 1 ? v[0][j / 2] | h << 16 : h;
            } else {
                v[j / 4][j & 3] = i + j < end ? *reinterpret_cast<const uint32_t*>(p) : 0xff800000u;
            }
        }
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (kHalf) return (float)__builtin_bit_cast(half8, v[0])[j];
        else return __builtin_bit_cast(float4v, v[j / 4])[j & 3];
    }
    // What was made of these is made again where it is asked for next, and takes no registers until then.
    __device__ __forceinline__ void forget() {
        asm volatile("" : "+v"(v[0]));
        if constexpr (!kHalf) asm volatile("" : "+v"(v[1]));
    }
    // (a NaN may go unnoticed)
    __device__ __forceinline__ float maximum() const {
        if constexpr (kHalf) {
            const half8 h = __builtin_bit_cast(half8, v[0]);
            half2v m = {h[0], h[1]};
#pragma unroll
            for (int j = 2; j < 8; j += 2) m = __builtin_elementwise_max(m, half2v{h[j], h[j + 1]});
            return (float)(m[0] > m[1] ? m[0] : m[1]);
        } else {
            float m = at(0);
#pragma unroll
            for (int j = 1; j < 8; ++j) m = fmaxf(m, at(j));
            return m;
        }
    }
};

// kTeam wavefronts to a row: 4, or 1 where rows are many and short (no parts then).
template <bool kHalf, int kTeam>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_kernel(LogprobArgs a) {
    __shared__ uint64_t lists[kWaves][kList];
    __shared__ int32_t counts[kWaves];
    __shared__ Sums sums[kWaves];
    __shared__ uint32_t maxima[kTeam > 1 ? kWaves : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int member = kTeam > 1 ? wave : 0;
    int64_t row = kTeam > 1 ? blockIdx.x / a.parts : (int64_t)blockIdx.x * kWaves + wave;
    const int32_t part = kTeam > 1 ? blockIdx.x % a.parts : 0;
    if (kTeam == 1 && row >= a.R) return;
    const int32_t begin = part * a.part, end = min(begin + a.part, a.V);
    const char* logits = a.logits + row * a.row;
    uint64_t* list = lists[wave];
    constexpr int kElement = kHalf ? 2 : 4;
    const bool dense = a.col == kElement;
    Sums z = {kNoMaximum[kHalf], 0.f, 0.f};
    int32_t count = 0;
    float below = NAN;  // what is not above it cannot be among the best; a NaN lets everything pass
    bool first = true;
    for (int32_t b = begin + member * kBlock; first || b < end; b += kTeam * kBlock) {
        Eight<kHalf> x[kLoads];
        if (dense && b + kBlock <= end) {
            const char* p = logits + (int64_t)(b + lane * 8) * kElement;
#pragma unroll
            for (int l = 0; l < kLoads; ++l) x[l].load(p + l * 64 * 8 * kElement);
        } else {
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                const int32_t i = b + (l * 64 + lane) * 8;
                if (dense && i + 8 <= end) x[l].load(logits + (int64_t)i * kElement);
                else x[l].load_some(logits, a.col, i, end);
            }
        }
        float best[kLoads];
#pragma unroll
        for (int l = 0; l < kLoads; ++l) best[l] = x[l].maximum();
        const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
        move_to<kHalf>(z, fmaxf(z.m, maximum_of<kHalf>(most)));
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int j = 0; j < kLoads * 8; ++j) {
            const float y = log2_of<kHalf>(x[j / 8].at(j & 7), z.m), e = __builtin_amdgcn_exp2f(y);
            s += e;
            t = __builtin_fmaf(fmaxf(y, -16384.f), e, t);  // (0, not NaN, for a logit of -inf)
        }
        z.s += s;
        z.t += t;
        if (a.top == 0) {
            first = false;
            continue;
        }
        if (first) {
            // the top-th largest of the lanes' maxima, of all wavefronts of the row, or of the maxima of its loads in one: its upper 20 bits, which is
            // a little below
            first = false;
            constexpr int kMaxima = 4;
            static_assert(kTeam == 1 ? kLoads == kMaxima : kTeam == kMaxima, "as many to a lane");
            uint32_t mine[kMaxima];
            if constexpr (kTeam > 1) {
                maxima[wave][lane] = sortable(most);
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kMaxima; ++w) mine[w] = maxima[w][lane];
            } else {
#pragma unroll
                for (int l = 0; l < kMaxima; ++l) mine[l] = sortable(best[l]);
            }
            uint32_t least = 0;
            for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1) {
                int n = 0;
#pragma unroll
                for (int w = 0; w < kMaxima; ++w) n += __popcll(__builtin_amdgcn_ballot_w64(mine[w] >= (least | bit)));
                if (n >= a.top) least |= bit;
            }
            // (what lies next below: below 0 not -0, which equals it; below -inf a NaN)
            below = of_sortable(least == 0x80000000u ? least - 2 : least - 1);
        }
        // (a sum that has become NaN may hide one from the maximum)
        if (__builtin_amdgcn_ballot_w64(!(most <= below) || z.s != z.s)) {
            uint64_t least = 0;
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                if (__builtin_amdgcn_ballot_w64(!(best[l] <= below) || z.s != z.s) == 0) continue;
                if (count > kKept) {
                    least = cut_list<false>(list, count, a.top);
                    count = a.top;
                }
                x[l].forget();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x[l].at(j);
                    const int32_t index = b + (l * 64 + lane) * 8 + j;
                    const uint64_t pass = __builtin_amdgcn_ballot_w64(index < end && !(v <= below));
                    if (pass == 0) continue;
                    if ((pass >> lane) & 1) list[count + __popcll(pass & ((1ull << lane) - 1))] = entry_of(v, index);
                    count += __popcll(pass);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            // (not before the block's end: among equal logits of a block, those with the lower index may come later; in later blocks all are higher)
            if (least != 0) below = of_sortable((uint32_t)(least >> 32));
        }
    }
    Given g;
    if (lane == 0 && member == 0 && a.parts == 1) g = given<kHalf>(a, row);
    join_lanes<kHalf>(z);
    if (count > 64) {
        if (count <= kKept) cut_list<true>(list, count, a.top);
        else cut_list<false>(list, count, a.top);
        count = a.top;
    }
    if constexpr (kTeam == 1) {
        const Row whole = whole_row<kHalf>(z);
        if (lane == 0) report_row<kHalf>(a, row, whole, g);
        const uint64_t mine = lane < count ? list[lane] : 0;
        const int32_t rank = before_in(list, count, mine);
        if (lane < count && rank < a.top) report_best<kHalf>(a, row, whole, rank, mine);
        return;
    }
    if (lane == 0) {
        sums[wave] = z;
        counts[wave] = count;
    }
    __syncthreads();
    z = lane < kTeam ? sums[lane] : Sums{kNoMaximum[kHalf], 0.f, 0.f};
    join_lanes<kHalf>(z);
    const bool one_part = a.parts == 1;
    const Row whole = whole_row<kHalf>(z);
    if (threadIdx.x == 0) {
        if (one_part) report_row<kHalf>(a, row, whole, g);
        else a.sums[blockIdx.x] = z;
    }
    if (a.top == 0) return;
    const uint64_t mine = lane < count ? list[lane] : 0;
    int32_t rank = 0;
#pragma unroll
    for (int w = 0; w < kTeam; ++w) rank += before_in(lists[w], counts[w], mine);
    if (lane < count && rank < a.top) {
        if (one_part) report_best<kHalf>(a, row, whole, rank, mine);
        else a.lists[(int64_t)blockIdx.x * a.top + rank] = mine;
    }
    if (!one_part) {  // a part may have fewer logits than alternatives
        int32_t all = 0;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) all += counts[w];
        if ((int32_t)threadIdx.x >= all && (int32_t)threadIdx.x < a.top) a.lists[(int64_t)blockIdx.x * a.top + threadIdx.x] = 0;
    }
}

// The parts of a row.  The largest of their last entries is a bound for what can be among the best.
template <bool kHalf>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ uint64_t list[kMostParts * kMostTop];
    __shared__ unsigned long long bound;
    __shared__ int32_t count;
    const int lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x;
    const uint64_t* from = a.lists + row * a.parts * a.top;
    const int32_t all = a.parts * a.top;
    Sums z = lane < a.parts ? a.sums[row * a.parts + lane] : Sums{kNoMaximum[kHalf], 0.f, 0.f};
    const uint64_t last = a.top > 0 && lane < a.parts ? from[(lane + 1) * a.top - 1] : 0, first = (int32_t)threadIdx.x < all ? from[threadIdx.x] : 0;
    Given g;
    if (threadIdx.x == 0) {
        g = given<kHalf>(a, row);
        bound = 1;
        count = 0;
    }
    __syncthreads();
    if (threadIdx.x < 64 && last != 0) atomicMax(&bound, (unsigned long long)last);
    __syncthreads();
    for (int32_t i = threadIdx.x; i < all; i += 256) {
        const uint64_t e = i == (int32_t)threadIdx.x ? first : from[i];
        if (e >= bound) list[atomicAdd(&count, 1)] = e;  // (in any order: they are ranked)
    }
    join_lanes<kHalf>(z);  // (each wavefront has all parts)
    const Row whole = whole_row<kHalf>(z);
    if (threadIdx.x == 0) report_row<kHalf>(a, row, whole, g);
    __syncthreads();
    for (int32_t i = threadIdx.x; i < count; i += 256) {
        const uint64_t mine = list[i];
        const int32_t rank = before_in(list, count, mine);
        if (rank < a.top) report_best<kHalf>(a, row, whole, rank, mine);
    }
}

// Parts of a row: as many as give each compute unit four work-groups, each of at least a step of all its wavefronts.
void split(int64_t R, int64_t V, int32_t* parts, int32_t* part) {
    const int64_t step = kWaves * kBlock, steps = (V + step - 1) / step;
    int64_t n = R > 0 ? 1024 / R : 1;
    n = n < 1 ? 1 : n > kMostParts ? kMostParts : n;
    n = n > steps ? steps : n;
    const int64_t each = (steps + n - 1) / n;
    *parts = (int32_t)((steps + each - 1) / each);
    *part = (int32_t)(each * step);
}

int64_t workspace_of(int64_t R, int64_t V, int64_t top) {
    int32_t parts, part;
    split(R, V, &parts, &part);
    return parts == 1 ? 0 : R * parts * (16 + 8 * top);  // (Sums are 12 bytes)
}

template <bool kHalf>
int launch(const LogprobArgs& a, hipStream_t s) {
    // One wavefront to a row of one or two steps.  us as four / as one, 8192 rows of float16 with 5 alternatives: 1000 logits 57 / 17, 4096 59 / 26, 8192 53 / 44
    // (but 66 / 62 with 20, 81 / 150 with 64); 1024 rows of 4096 10.0 / 10.0 (14.8 / 16.4 with 64).
    if (a.V <= kBlock || (a.V <= 2 * kBlock && a.R >= 2048)) {
        token_logprobs_kernel<kHalf, 1><<<(unsigned)((a.R + kWaves - 1) / kWaves), 64 * kWaves, 0, s>>>(a);
        return launch_check("token_logprobs_kernel");
    }
    token_logprobs_kernel<kHalf, kWaves><<<(unsigned)(a.R * a.parts), 64 * kWaves, 0, s>>>(a);
    CHX_PROPAGATE(launch_check("token_logprobs_kernel"));
    if (a.parts == 1) return CHX_HIP_OK;
    token_logprobs_join_kernel<kHalf><<<(unsigned)a.R, 256, 0, s>>>(a);
    return launch_check("token_logprobs_join_kernel");
}

int check_sizes(int64_t R, int64_t V, int64_t top) {
    CHX_REQUIRE(R >= 0 && R < (int64_t(1) << 24), "token logprobs: 2^24 rows or more");
    CHX_REQUIRE(V >= 1 && V < (int64_t(1) << 30), "token logprobs: 1 to 2^30 - 1 logits to a row, not %lld", (long long)V);
    CHX_REQUIRE(top >= 0 && top <= kMostTop && top <= V, "token logprobs: at most %d alternatives, and no more than there are logits, not %lld", kMostTop, (long long)top);
    return CHX_HIP_OK;
}

int check_result(const chx_hip_tensor* t, int32_t dtype, int64_t elements, const char* name) {
    CHX_PROPAGATE(check_tensor(t, name));
    CHX_REQUIRE(t->dtype == dtype && numel(*t) == elements && (elements == 0 || is_contiguous(*t)) && aligned(t->data, (size_t)dtype_size(dtype)), "token logprobs: %s must be %s, contiguous, %lld elements",
                name, dtype_name(dtype), (long long)elements);
    return CHX_HIP_OK;
}

}  // namespace
}  // namespace chx

using namespace chx;

extern "C" int chx_hip_token_logprobs_workspace(int64_t rows, int64_t logits, int64_t top, size_t* bytes) {
    CHX_REQUIRE(bytes != nullptr, "token logprobs: null output");
    CHX_PROPAGATE(check_sizes(rows, logits, top));
    *bytes = (size_t)workspace_of(rows, logits, top);
    return CHX_HIP_OK;
}

extern "C" int chx_hip_token_logprobs(
        const chx_hip_tensor* logits, const chx_hip_tensor* tokens, chx_hip_tensor* logprobs, chx_hip_tensor* entropy, chx_hip_tensor* top_logprobs,
        chx_hip_tensor* top_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    CHX_PROPAGATE(check_tensor(logits, "token logprobs logits"));
    CHX_REQUIRE(logits->dtype == CHX_HIP_FLOAT16 || logits->dtype == CHX_HIP_FLOAT32, "token logprobs: logits must be float16 or float32, not %s", dtype_name(logits->dtype));
    CHX_REQUIRE(logits->ndim == 2, "token logprobs: logits must be a matrix");
    const int64_t es = dtype_size(logits->dtype);
    CHX_REQUIRE(aligned(logits->data, (size_t)es) && logits->strides[0] % es == 0 && logits->strides[1] % es == 0, "token logprobs: logits are not made of whole elements");
    const int64_t R = logits->shape[0], V = logits->shape[1];
    CHX_PROPAGATE(check_tensor(top_logprobs, "top_logprobs"));
    CHX_REQUIRE(top_logprobs->ndim == 2, "token logprobs: top_logprobs must be a matrix");
    const int64_t top = top_logprobs->shape[1];
    CHX_PROPAGATE(check_sizes(R, V, top));
    CHX_PROPAGATE(check_result(entropy, CHX_HIP_FLOAT32, R, "entropy"));
    CHX_PROPAGATE(check_result(top_logprobs, CHX_HIP_FLOAT32, R * top, "top_logprobs"));
    CHX_PROPAGATE(check_result(top_tokens, CHX_HIP_INT64, R * top, "top_tokens"));
    LogprobArgs a;
    memset(&a, 0, sizeof(a));
    CHX_REQUIRE((tokens == nullptr) == (logprobs == nullptr), "token logprobs: tokens and logprobs are given together");
    if (tokens != nullptr) {
        CHX_PROPAGATE(check_tensor(tokens, "tokens"));
        CHX_REQUIRE(tokens->dtype == CHX_HIP_INT32 || tokens->dtype == CHX_HIP_INT64, "token logprobs: tokens must be int32 or int64, not %s", dtype_name(tokens->dtype));
        const int64_t ts = dtype_size(tokens->dtype);
        CHX_REQUIRE(tokens->ndim == 1 && tokens->shape[0] == R && tokens->strides[0] % ts == 0 && aligned(tokens->data, (size_t)ts), "token logprobs: a token for each row is needed");
        CHX_PROPAGATE(check_result(logprobs, CHX_HIP_FLOAT32, R, "logprobs"));
        a.tokens = static_cast<const char*>(tokens->data);
        a.token64 = tokens->dtype == CHX_HIP_INT64;
        a.token_col = tokens->strides[0];
        a.logprob = static_cast<float*>(logprobs->data);
    }
    const int64_t needed = workspace_of(R, V, top);
    CHX_REQUIRE((int64_t)workspace_bytes >= needed && (needed == 0 || (workspace != nullptr && aligned(workspace, 16))),
                "token logprobs: a workspace of %lld bytes, aligned to 16, is needed", (long long)needed);
    if (R == 0) return CHX_HIP_OK;
    a.logits = static_cast<const char*>(logits->data);
    a.row = logits->strides[0];
    a.col = V == 1 ? es : logits->strides[1];
    a.half = logits->dtype == CHX_HIP_FLOAT16;
    a.V = (int32_t)V;
    a.top = (int32_t)top;
    a.R = R;
    split(R, V, &a.parts, &a.part);
    a.entropy = static_cast<float*>(entropy->data);
    a.top_logprob = static_cast<float*>(top_logprobs->data);
    a.top_token = static_cast<int64_t*>(top_tokens->data);
    a.sums = static_cast<Sums*>(workspace);
    a.lists = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + R * a.parts * 16);
    return a.half ? launch<true>(a, as_stream(stream)) : launch<false>(a, as_stream(stream));
}
