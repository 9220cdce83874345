// Log probabilities of given tokens, the entropy of each row of logits, and the best alternatives.
//
//   m = max x;  s = sum exp(x - m);  t = sum (x - m) exp(x - m)          over a row's V logits
//   log p(token) = x[token] - m - log s;   entropy = log s - t / s;      alternatives: the `top` largest logits, the lower index first
//
// Bound by the bytes of the logits: one pass with a running maximum, four loads of 16 bytes a lane under way, in float32.  Where rows are few, work-groups
// share a row and a second launch joins their parts, in one order.
//
// The alternatives are found in the same pass.  A wavefront keeps a threshold below which nothing can be among its `top` best, first from the
// maxima of its lanes (the top-th largest of 64 of them has top logits at or above it), later from what it has gathered; a block of 32 logits a lane is
// compared by its maximum alone, and what passes goes to a list in LDS that is cut to its best when it is full.
#include <cfloat>
#include <cmath>
#include <cstring>

#include "chx_internal.h"

namespace chx {
namespace {

constexpr int kMostTop = 64, kWaves = 4;
constexpr int kKept = 256, kList = kKept + 512;  // entries of a list: it is cut when there are more than kKept, and 512 more may come in between
constexpr int kLoads = 4;               // of 16 bytes (float16), 32 (float32): 8 logits each
constexpr int kBlock = 64 * 8 * kLoads; // logits of a wavefront's step
constexpr int kMostParts = 64;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

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
    float* sums;     // of the parts: [row][part][4]
    uint64_t* lists; // [row][part][top], best first
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

struct Sums {
    float m, s, t;  // t in units of log 2: sum (x - m) log2(e) exp(x - m)
};
// The sums over both, relative to the larger maximum.
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const float ya = (a.m - m) * kLog2e, yb = (b.m - m) * kLog2e;
    const float fa = a.s == 0.f ? 0.f : __builtin_amdgcn_exp2f(ya), fb = b.s == 0.f ? 0.f : __builtin_amdgcn_exp2f(yb);
    Sums r;
    r.m = m;
    r.s = a.s * fa + b.s * fb;
    r.t = (fa == 0.f ? 0.f * a.s : (a.t + ya * a.s) * fa) + (fb == 0.f ? 0.f * b.s : (b.t + yb * b.s) * fb);
    return r;
}

// The `top` best of `count` entries of one wavefront, kept at the front of its list; returns how many there are, and the least of them (0: all are).
__device__ int32_t cut_list(uint64_t* list, int32_t count, int32_t top, uint64_t* least_kept) {
    const int lane = threadIdx.x & 63;
    *least_kept = 0;
    if (count <= top) return count;
    uint64_t mine[kList / 64];
#pragma unroll
    for (int i = 0; i < kList / 64; ++i) mine[i] = 64 * i + lane < count ? list[64 * i + lane] : 0;
    // the top-th largest, bit by bit: no two entries are equal
    uint64_t least = 0;
    for (int b = 63; b >= 0; --b) {
        const uint64_t try_at = least | 1ull << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kList / 64; ++i) {
            if (64 * i >= count) break;
            n += __popcll(__builtin_amdgcn_ballot_w64(mine[i] >= try_at));
        }
        if (n >= top) least = try_at;
    }
    int32_t at = 0;
#pragma unroll
    for (int i = 0; i < kList / 64; ++i) {
        const uint64_t keep = __builtin_amdgcn_ballot_w64(mine[i] >= least);
        if ((keep >> lane) & 1) list[at + __popcll(keep & ((1ull << lane) - 1))] = mine[i];
        at += __popcll(keep);
    }
    *least_kept = least;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return at;
}

// entries[0, count), count <= 64, of one wavefront: best first, zeros behind them up to `top`.
__device__ void sort_list(uint64_t* list, int32_t count, int32_t top) {
    const int lane = threadIdx.x & 63;
    const uint64_t mine = lane < count ? list[lane] : 0;
    int rank = 0;
    for (int i = 0; i < count; ++i) rank += __shfl(mine, i) > mine;
    __builtin_amdgcn_wave_barrier();
    if (lane < top) list[lane < count ? rank : lane] = mine;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The best `top` of `lists` sorted lists of `top` entries, `stride` entries apart; the lanes of one wavefront, lists <= 64.  Lane j gets the j-th.
__device__ uint64_t merge_lists(const uint64_t* list, int32_t lists, int32_t stride, int32_t top) {
    const int lane = threadIdx.x & 63;
    int32_t next = 0;
    uint64_t head = lane < lists && top > 0 ? list[(int64_t)lane * stride] : 0, got = 0;
    for (int j = 0; j < top; ++j) {
        uint64_t best = head;
#pragma unroll
        for (int d = 32; d; d /= 2) {
            const uint64_t other = __shfl_xor(best, d);
            best = other > best ? other : best;
        }
        if (lane == j) got = best;
        if (head == best && best != 0) {
            ++next;
            head = next < top ? list[(int64_t)lane * stride + next] : 0;
        }
    }
    return got;
}

// What is reported for a row, by one wavefront; `best` as from merge_lists.
__device__ void report(const LogprobArgs& a, int64_t row, const Sums& z, uint64_t best) {
    const int lane = threadIdx.x & 63;
    // (no logit above -inf: no token has a probability)
    const bool none = z.s == 0.f;
    const float log_s = none ? 0.f : logf(z.s);
    if (lane == 0) {
        if (a.logprob) {
            const char* p = a.tokens + row * a.token_col;
            const int64_t token = a.token64 ? *reinterpret_cast<const int64_t*>(p) : *reinterpret_cast<const int32_t*>(p);
            float v = 0.f;
            if (token >= a.V) {
                v = NAN;
            } else if (token >= 0) {
                const char* q = a.logits + row * a.row + token * a.col;
                v = none ? -INFINITY : (a.half ? (float)*reinterpret_cast<const _Float16*>(q) : *reinterpret_cast<const float*>(q)) - z.m - log_s;
            }
            a.logprob[row] = v;
        }
        a.entropy[row] = none ? 0.f : log_s - kLn2 * z.t / z.s;
    }
    if (lane < a.top) {
        const float x = of_sortable((uint32_t)(best >> 32));
        a.top_logprob[row * a.top + lane] = none ? -INFINITY : x - z.m - log_s;
        a.top_token[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)best;
    }
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// Eight logits from index i on; -inf from `end` on.
template <bool kHalf>
__device__ __forceinline__ void load8(const char* row, int64_t col, int32_t i, int32_t end, float* x) {
    constexpr int kElement = kHalf ? 2 : 4;
    if (col == kElement && i + 8 <= end) {
        const u32x4_any* p = reinterpret_cast<const u32x4_any*>(row + (int64_t)i * kElement);
        if constexpr (kHalf) {
            const half8 h = __builtin_bit_cast(half8, p[0]);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (float)h[j];
        } else {
            const u32x4_any lo = p[0], hi = p[1];
            __builtin_memcpy(x, &lo, 16);
            __builtin_memcpy(x + 4, &hi, 16);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = -INFINITY;
        if (i + j < end) {
            const char* p = row + (int64_t)(i + j) * col;
            if constexpr (kHalf) x[j] = (float)*reinterpret_cast<const _Float16*>(p);
            else x[j] = *reinterpret_cast<const float*>(p);
        }
    }
}

template <bool kHalf>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_kernel(LogprobArgs a) {
    __shared__ uint64_t lists[kWaves][kList];
    __shared__ Sums sums[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x / a.parts;
    const int32_t part = blockIdx.x % a.parts;
    const int32_t begin = part * a.part, end = min(begin + a.part, a.V);
    const char* logits = a.logits + row * a.row;
    uint64_t* list = lists[wave];
    // (a maximum of the lowest number to begin with: its differences are finite)
    Sums z = {-FLT_MAX, 0.f, 0.f};
    int32_t count = 0;
    float below = NAN;  // what is not above it cannot be among the best; NaN: not known yet
    for (int32_t b = begin + wave * kBlock; b < end; b += kWaves * kBlock) {
        float x[kLoads * 8];
#pragma unroll
        for (int l = 0; l < kLoads; ++l) load8<kHalf>(logits, a.col, b + (l * 64 + lane) * 8, end, x + l * 8);
        float most = x[0];
#pragma unroll
        for (int j = 1; j < kLoads * 8; ++j) most = fmaxf(most, x[j]);
        const float m = fmaxf(z.m, most);
        {
            const float y = (z.m - m) * kLog2e, f = __builtin_amdgcn_exp2f(y);
            z.t = f == 0.f ? 0.f * z.s : (z.t + y * z.s) * f;
            z.s *= f;
            z.m = m;
        }
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int j = 0; j < kLoads * 8; ++j) {
            const float y = (x[j] - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
            s += e;
            t = __builtin_fmaf(fmaxf(y, -16384.f), e, t);  // (0, not NaN, for a logit of -inf)
        }
        z.s += s;
        z.t += t;
        if (a.top == 0) continue;
        if (below != below) {
            // the top-th largest of the lanes' maxima has `top` logits at or above it
            const uint32_t mine = sortable(most);
            int before = 0;
            for (int i = 0; i < 64; ++i) {
                const uint32_t other = __shfl(mine, i);
                before += other > mine || (other == mine && i < lane);
            }
            const uint64_t at = __builtin_amdgcn_ballot_w64(before == a.top - 1);
            const uint32_t key = __builtin_amdgcn_readlane(mine, __builtin_ctzll(at));
            // (what lies next below: below 0 not -0, which equals it; below -inf a NaN, so that everything passes)
            below = of_sortable(key == 0x80000000u ? key - 2 : key - 1);
        }
        // (a sum that has become NaN may hide one from the maximum)
        if (__builtin_amdgcn_ballot_w64(!(most <= below) || z.s != z.s)) {
            uint64_t least = 0;
#pragma unroll 1
            for (int l = 0; l < kLoads; ++l) {
                if (count > kKept) count = cut_list(list, count, a.top, &least);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float v = x[j];
#pragma unroll
                    for (int q = 1; q < kLoads; ++q) v = q == l ? x[q * 8 + j] : v;
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
    // lanes, then wavefronts, in one order
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        Sums o = {__shfl_xor(z.m, d), __shfl_xor(z.s, d), __shfl_xor(z.t, d)};
        z = joined(z, o);
    }
    if (lane == 0) sums[wave] = z;
    if (a.top > 0) {
        uint64_t least;
        count = cut_list(list, count, a.top, &least);
        sort_list(list, count, a.top);
    }
    __syncthreads();
    if (wave != 0) return;
    z = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) z = joined(z, sums[w]);
    const uint64_t best = merge_lists(&lists[0][0], kWaves, kList, a.top);
    if (a.parts == 1) {
        report(a, row, z, best);
        return;
    }
    float* to = a.sums + (row * a.parts + part) * 4;
    if (lane == 0) {
        to[0] = z.m;
        to[1] = z.s;
        to[2] = z.t;
    }
    if (lane < a.top) a.lists[(row * a.parts + part) * a.top + lane] = best;
}

// The parts of a row, by one wavefront.
__global__ __launch_bounds__(64) void token_logprobs_join_kernel(LogprobArgs a) {
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    Sums z = {-FLT_MAX, 0.f, 0.f};
    if (lane < a.parts) {
        const float* from = a.sums + (row * a.parts + lane) * 4;
        z = {from[0], from[1], from[2]};
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        Sums o = {__shfl_xor(z.m, d), __shfl_xor(z.s, d), __shfl_xor(z.t, d)};
        z = joined(z, o);
    }
    report(a, row, z, merge_lists(a.lists + row * a.parts * a.top, a.parts, a.top, a.top));
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
    return parts == 1 ? 0 : R * parts * (16 + 8 * top);
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
    a.sums = static_cast<float*>(workspace);
    a.lists = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + R * a.parts * 16);
    const hipStream_t s = as_stream(stream);
    const unsigned blocks = (unsigned)(R * a.parts);
    if (a.half) token_logprobs_kernel<true><<<blocks, 64 * kWaves, 0, s>>>(a);
    else token_logprobs_kernel<false><<<blocks, 64 * kWaves, 0, s>>>(a);
    CHX_PROPAGATE(launch_check("token_logprobs_kernel"));
    if (a.parts == 1) return CHX_HIP_OK;
    token_logprobs_join_kernel<<<(unsigned)R, 64, 0, s>>>(a);
    return launch_check("token_logprobs_join_kernel");
}
