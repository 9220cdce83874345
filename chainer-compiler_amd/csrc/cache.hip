// A cache of keys and values in pages: rows appended, drafted rows that were accepted moved together, and eviction by accumulated weight.
//
// All of it is bound by the bytes that move (few rows: by the launches).  Work-groups own what they write: in a move within the cache, a work-group has all
// rows of a sequence's head, of keys or values, and a slice of their elements, so that no row is read by one group after another has written it.
#include <algorithm>
#include <cstring>
#include <initializer_list>

#include "cache.h"

namespace chx {

int check_rows(const chx_hip_tensor* t, int ndim, int32_t dtype, const char* what, const char* name) {
    CHX_PROPAGATE(check_tensor(t, name));
    CHX_REQUIRE(t->dtype == CHX_HIP_FLOAT16 || t->dtype == CHX_HIP_FLOAT32, "%s: %s must be float16 or float32, not %s", what, name, dtype_name(t->dtype));
    CHX_REQUIRE(dtype == 0 || t->dtype == dtype, "%s: %s must be %s, as the others are, not %s", what, name, dtype_name(dtype), dtype_name(t->dtype));
    CHX_REQUIRE(t->ndim == ndim, "%s: %s needs %d axes, not %d", what, name, ndim, t->ndim);
    const int64_t es = dtype_size(t->dtype);
    bool whole = aligned(t->data, (size_t)es);
    for (int i = 0; i < ndim; ++i) whole = whole && (t->shape[i] <= 1 || t->strides[i] % es == 0);
    CHX_REQUIRE(whole, "%s: %s is not made of whole elements", what, name);
    CHX_REQUIRE(t->shape[ndim - 1] <= 1 || t->strides[ndim - 1] == es, "%s: the last axis of %s has gaps", what, name);
    return CHX_HIP_OK;
}

int check_numbers(const chx_hip_tensor* t, int ndim, int64_t n0, int64_t n1, const char* what, const char* name) {
    CHX_PROPAGATE(check_tensor(t, name));
    CHX_REQUIRE(t->dtype == CHX_HIP_INT32, "%s: %s must be int32, not %s", what, name, dtype_name(t->dtype));
    CHX_REQUIRE(t->ndim == ndim && (n0 < 0 || t->shape[0] == n0) && (ndim < 2 || n1 < 0 || t->shape[1] == n1), "%s: %s has another shape than the others ask for", what, name);
    CHX_REQUIRE(numel(*t) == 0 || (is_contiguous(*t) && aligned(t->data, 4)), "%s: %s must be contiguous", what, name);
    return CHX_HIP_OK;
}

int check_cache(const chx_hip_tensor* keys, const chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, const char* what, CacheArgs* c) {
    CHX_PROPAGATE(check_rows(keys, 4, 0, what, "keys"));
    CHX_PROPAGATE(check_rows(values, 4, keys->dtype, what, "values"));
    CHX_REQUIRE(same_shape(*keys, *values), "%s: keys and values must have one shape", what);
    CHX_REQUIRE(keys->shape[1] >= 1 && keys->shape[2] >= 1 && keys->shape[3] >= 1 && keys->shape[3] <= 256, "%s: a page needs a place, a head and 1 to 256 elements", what);
    CHX_REQUIRE(keys->shape[0] < (int64_t(1) << 31) && keys->shape[2] < (int64_t(1) << 16), "%s: 2^31 pages or 2^16 heads", what);
    CHX_PROPAGATE(check_tensor(tables, "tables"));
    CHX_REQUIRE(tables->dtype == CHX_HIP_INT32 && tables->ndim == 2, "%s: tables must be an int32 matrix", what);
    CHX_REQUIRE(numel(*tables) == 0 || (aligned(tables->data, 4) && (tables->shape[1] == 1 || tables->strides[1] == 4) && tables->strides[0] % 4 == 0), "%s: a row of tables must be contiguous", what);
    CHX_REQUIRE(tables->shape[0] < (int64_t(1) << 24), "%s: 2^24 sequences", what);
    CHX_REQUIRE(keys->shape[1] < (int64_t(1) << 30) && tables->shape[1] < (int64_t(1) << 30) && tables->shape[1] * keys->shape[1] < (int64_t(1) << 30), "%s: a sequence of 2^30 places", what);
    CHX_PROPAGATE(check_numbers(lengths, 1, tables->shape[0], 0, what, "lengths"));
    memset(c, 0, sizeof(*c));
    c->k = static_cast<char*>(keys->data);
    c->v = static_cast<char*>(values->data);
    c->k_page = stride_of(*keys, 0), c->k_row = stride_of(*keys, 1), c->k_head = stride_of(*keys, 2);
    c->v_page = stride_of(*values, 0), c->v_row = stride_of(*values, 1), c->v_head = stride_of(*values, 2);
    c->tables = static_cast<const int32_t*>(tables->data);
    c->table_row = tables->strides[0] / 4;
    c->lengths = static_cast<const int32_t*>(lengths->data);
    c->B = (int32_t)tables->shape[0];
    c->groups = (int32_t)keys->shape[2];
    c->D = (int32_t)keys->shape[3];
    c->pages = (int32_t)keys->shape[0];
    c->page_rows = (int32_t)keys->shape[1];
    c->by_page = divisor_of(c->page_rows);
    c->places = (int32_t)(tables->shape[1] * keys->shape[1]);
    return CHX_HIP_OK;
}

int check_mass(const chx_hip_tensor* mass, const CacheArgs& c, const char* what) {
    CHX_PROPAGATE(check_tensor(mass, "mass"));
    CHX_REQUIRE(mass->dtype == CHX_HIP_FLOAT32 && mass->ndim == 3, "%s: mass must be float32 with three axes", what);
    CHX_REQUIRE(mass->shape[0] == c.B && mass->shape[1] == c.groups && mass->shape[2] >= c.places, "%s: mass must have a number for each sequence, head and place", what);
    if (numel(*mass) == 0) return CHX_HIP_OK;
    CHX_REQUIRE(aligned(mass->data, 4) && mass->strides[0] % 4 == 0 && mass->strides[1] % 4 == 0 && (mass->shape[2] == 1 || mass->strides[2] == 4), "%s: the last axis of mass has gaps", what);
    CHX_REQUIRE(elements_apart(*mass), "%s: elements of mass overlap", what);
    return CHX_HIP_OK;
}

namespace {

// Whether some sum of steps along the axes, by less than n of each, comes closer to `distance` than an element is long.  Axes by falling distance of their elements, each more than all behind it reach: only
// the two multiples next to what is left can do.
struct Axis {
    int64_t n, stride;
};
bool steps_meet(int64_t distance, const Axis* axes, int count, int64_t element) {
    distance = std::abs(distance);
    if (count == 0) return distance < element;
    const int64_t steps = distance / axes->stride < axes->n - 1 ? distance / axes->stride : axes->n - 1;
    if (steps_meet(distance - steps * axes->stride, axes + 1, count - 1, element)) return true;
    return steps + 1 < axes->n && steps_meet(distance - (steps + 1) * axes->stride, axes + 1, count - 1, element);
}

// Arrays between each other's rows, as keys and values of pages that hold both: of one type, shape and distances, each with its elements apart, without a byte in common.
bool interleaved(const chx_hip_tensor& a, const chx_hip_tensor& b) {
    if (a.dtype != b.dtype || !same_shape(a, b) || !elements_apart(a) || !elements_apart(b)) return false;
    Axis axes[CHX_HIP_MAX_NDIM];
    int count = 0;
    for (int d = 0; d < a.ndim; ++d) {
        if (a.shape[d] == 1) continue;
        if (a.strides[d] != b.strides[d]) return false;
        axes[count++] = {a.shape[d], std::abs(a.strides[d])};
    }
    std::sort(axes, axes + count, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
    return !steps_meet((int64_t)(reinterpret_cast<intptr_t>(a.data) - reinterpret_cast<intptr_t>(b.data)), axes, count, dtype_size(a.dtype));
}

}  // namespace

int check_apart(const Named& written, const Named* others, int count, const char* what) {
    if (written.t == nullptr || numel(*written.t) == 0) return CHX_HIP_OK;
    for (int i = 0; i < count; ++i) {
        if (others[i].t == nullptr || numel(*others[i].t) == 0) continue;
        CHX_REQUIRE(!arrays_overlap(*written.t, *others[i].t) || interleaved(*written.t, *others[i].t), "%s: %s and %s overlap", what, written.name, others[i].name);
    }
    return CHX_HIP_OK;
}

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Bytes of a row that are copied at once: what all distances, addresses and the row itself are multiples of.
int unit_of(std::initializer_list<int64_t> bytes) {
    int64_t all = 16;
    for (int64_t b : bytes) all |= b;
    return (int)(all & -all);
}
int64_t at_of(const void* p) {
    return (int64_t)reinterpret_cast<intptr_t>(p);
}

__device__ __forceinline__ int32_t clamped(int32_t v, int32_t most) {
    return max(0, min(v, most));
}

// ---- append -------------------------------------------------------------------------------------------

struct AppendArgs {
    CacheArgs c;
    const char *k, *v;
    int64_t k_batch, k_token, k_head, v_batch, v_token, v_head;
    const int32_t* counts;
    int32_t T, units;   // units of a row
    int64_t pieces;     // B T groups units
};

// A lane moves one unit of a key and of its value.  64 tokens of 8 heads of 128 elements, float16, 3.3 us; 6 prompts of up to 4096 26 us (117 MB, 4.5 TB/s; a large copy reaches 5.0).
template <typename Unit>
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs a, int64_t first) {
    const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.pieces) return;
    const int64_t row = i / a.units;
    const int32_t u = (int32_t)(i - row * a.units);
    const int64_t bt = row / a.c.groups;
    const int32_t h = (int32_t)(row - bt * a.c.groups), b = (int32_t)(bt / a.T), t = (int32_t)(bt - (int64_t)b * a.T);
    if (a.counts && t >= a.counts[b]) return;
    const int32_t p = clamped(a.c.lengths[b], a.c.places) + t;  // (both below 2^30)
    if (p >= a.c.places) return;
    const Place at = place_of(a.c, b, p);
    if (at.page < 0) return;
    const Unit k = reinterpret_cast<const Unit*>(a.k + b * a.k_batch + t * a.k_token + h * a.k_head)[u];
    const Unit v = reinterpret_cast<const Unit*>(a.v + b * a.v_batch + t * a.v_token + h * a.v_head)[u];
    reinterpret_cast<Unit*>(a.c.k + at.page * a.c.k_page + at.row * a.c.k_row + h * a.c.k_head)[u] = k;
    reinterpret_cast<Unit*>(a.c.v + at.page * a.c.v_page + at.row * a.c.v_row + h * a.c.v_head)[u] = v;
}

// ---- moves within the cache ---------------------------------------------------------------------------

constexpr int32_t kMostAccepted = 256;
constexpr int kSlice = 128;  // bytes of a row that a work-group moves

struct MoveArgs {
    CacheArgs c;
    float* mass;  // null: none
    int64_t mass_batch, mass_head;
    int32_t row_bytes, slices;
    // accepted
    const int32_t* accepted;
    int32_t most;
    int32_t* new_lengths;
    // evicted
    int32_t keep, recent;
    int32_t* lists;  // [B][groups][1 + 2 most]: how many places move, where to, where from
};

// A slice of a head's row at a place; null: no place.
struct Rows {
    char* base;
    int64_t page, row;
};
__device__ __forceinline__ char* row_at(const MoveArgs& a, const Rows& r, int32_t b, int64_t p) {
    if (p < 0 || p >= a.c.places) return nullptr;
    const Place at = place_of(a.c, b, (int32_t)p);
    return at.page < 0 ? nullptr : r.base + at.page * r.page + at.row * r.row;
}

// Drafted rows that were accepted.  A work-group has at most 256 slices of 128 bytes: all are read before the first is written.  blockIdx: sequence, head, then keys' slices, values' slices, mass.
// Bound by the loads that wait for each other (accepted, tables, rows): where a row comes from and goes to is found once, by a lane for each.  5 of 24 rows of 32 sequences, 8 heads of 128 elements, float16, and their mass: 5.3 us; 77 of
// 200 of 13, 5 heads of 75, float32: 7.9.
template <typename Unit>
__global__ __launch_bounds__(256) void cache_accept_kernel(MoveArgs a) {
    __shared__ Unit rows[kMostAccepted * kSlice / sizeof(Unit)];
    __shared__ const char* from_at[kMostAccepted];
    __shared__ char* to_at[kMostAccepted];
    __shared__ int32_t count;
    const int32_t each = 2 * a.slices + (a.mass ? 1 : 0), what = blockIdx.x % each, h = blockIdx.x / each % a.c.groups, b = blockIdx.x / each / a.c.groups;
    const int32_t length = clamped(a.c.lengths[b], a.c.places), i = threadIdx.x;
    if (i == 0) count = a.most;
    const int32_t slice = what % a.slices * kSlice;
    const Rows r = what < a.slices ? Rows{a.c.k + h * a.c.k_head + slice, a.c.k_page, a.c.k_row} : Rows{a.c.v + h * a.c.v_head + slice, a.c.v_page, a.c.v_row};
    __syncthreads();
    int32_t from = -1;
    if (i < a.most) {
        from = a.accepted[(int64_t)b * a.most + i];
        if (from < 0) atomicMin(&count, i);
        const char* at = row_at(a, r, b, (int64_t)length + from);
        char* to = row_at(a, r, b, (int64_t)length + i);
        from_at[i] = to ? at : nullptr;
        to_at[i] = at ? to : nullptr;
    }
    __syncthreads();
    const int32_t n = count;
    if (what == 0 && h == 0 && i == 0) a.new_lengths[b] = min(length + n, a.c.places);
    if (what == 2 * a.slices) {
        float* mass = a.mass + b * a.mass_batch + h * a.mass_head;
        const int64_t p = i < n ? (int64_t)length + from : a.c.places;
        const float v = p < a.c.places ? mass[p] : 0.f;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (p < a.c.places && length + i < a.c.places) mass[length + i] = v;
        return;
    }
    const int32_t bytes = min(kSlice, a.row_bytes - slice), units = bytes / (int32_t)sizeof(Unit);
    constexpr int kAtOnce = 4;
    for (int32_t j0 = i; j0 < n * units; j0 += 256 * kAtOnce) {
        Unit v[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int32_t j = j0 + k * 256;
            const char* at = j < n * units ? from_at[j / units] : nullptr;
            if (at) v[k] = reinterpret_cast<const Unit*>(at)[j % units];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
            if (j0 + k * 256 < n * units) rows[j0 + k * 256] = v[k];  // (also what is not there: it goes nowhere)
    }
    __syncthreads();
    for (int32_t j = i; j < n * units; j += 256) {
        char* to = to_at[j / units];
        if (to) reinterpret_cast<Unit*>(to)[j % units] = rows[j];
    }
}

// ---- eviction -----------------------------------------------------------------------------------------

// Larger numbers first, a NaN before all.
__device__ __forceinline__ uint32_t sortable(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);  // (-0 is 0)
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// The weights as numbers to be compared, four at a time: in LDS where a sequence's fit (kInLds: read once, eight loads of a lane under way), else from memory each time.  Behind the last
// are zeros, which are less than any weight's.
constexpr int32_t kMostInLds = 36 * 1024;
template <bool kInLds>
struct Keys {
    const float* mass;
    u32x4* keys;
    int32_t n;
    // Calls f(key, whether it is one) for all of them, of all lanes of a wavefront at once.
    template <typename F>
    __device__ __forceinline__ void load(F f) {
        constexpr int kAtOnce = 8;
        uint32_t* to = reinterpret_cast<uint32_t*>(keys);
        const int32_t all = (n + 3) / 4 * 4, lane = threadIdx.x & 63;
        for (int32_t i0 = threadIdx.x; i0 - lane < all; i0 += 1024 * kAtOnce) {
            float v[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) v[j] = i0 + j * 1024 < n ? mass[i0 + j * 1024] : 0.f;
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int32_t i = i0 + j * 1024;
                const uint32_t key = i < n ? sortable(v[j]) : 0;
                if (i < all) to[i] = key;
                f(key, i < n);
            }
        }
    }
    __device__ __forceinline__ u32x4 at(int32_t quad) const {
        if constexpr (kInLds) return keys[quad];
        u32x4 k;
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = 4 * quad + j < n ? sortable(mass[4 * quad + j]) : 0;
        return k;
    }
};

// The sum of what the wavefronts before this one have, of 16.
__device__ __forceinline__ int32_t before_wave(const int32_t* of_waves, int wave) {
    const int lane = threadIdx.x & 63;
    int32_t v = lane < wave ? of_waves[lane & 15] : 0;
#pragma unroll
    for (int d = 8; d; d /= 2) v += __shfl_xor(v, d);
    return __builtin_amdgcn_readfirstlane(v);
}

// A head's places that stay: the threshold of the `best` largest of n weights by three histograms of 11, 11 and 10 bits, of equal ones the lower places; then the
// list of moves, places that go in front of best and places that stay behind it, both in ascending order.  One work-group to a head; bound by its instructions where sequences are long (32,768 places: four passes
// over LDS, and one that fills it), by its barriers where they are short.  128 heads of 2080 places, 2048 to stay: 9.5 us; 32 of 32768, 8192 to stay, 28 (22 where nearly none move).  Tables that LDS has no room for: a weight at a time from memory, in each pass; 65536 places,
// 1 head 95 us, 32 heads 103.
template <bool kInLds>
__global__ __launch_bounds__(1024) void cache_choose_kernel(MoveArgs a) {
    extern __shared__ u32x4 choose_lds[];
    constexpr int kWaves = 16, kBins = 2048;
    __shared__ int32_t bins[kBins];
    __shared__ int32_t of_waves[3][kWaves];
    __shared__ int32_t found[3];  // bin, how many are above it, how many are in it
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t h = blockIdx.x % a.c.groups, b = blockIdx.x / a.c.groups;
    const int32_t length = clamped(a.c.lengths[b], a.c.places);
    int32_t* list = a.lists + (int64_t)blockIdx.x * (1 + 2 * a.most);
    if (h == 0 && threadIdx.x == 0) a.new_lengths[b] = min(length, a.keep);
    if (length <= a.keep) {
        if (threadIdx.x == 0) list[0] = 0;
        return;
    }
    const int32_t n = length - a.recent, best = a.keep - a.recent, quads = (n + 3) / 4;
    if (best == 0) {  // (nothing of them stays, and nothing moves)
        if (threadIdx.x == 0) list[0] = 0;
        return;
    }
    Keys<kInLds> keys = {a.mass + b * a.mass_batch + h * a.mass_head, choose_lds, n};
    for (int i = threadIdx.x; i < kBins; i += 1024) bins[i] = 0;
    __syncthreads();
    auto count = [&](uint32_t bin, bool counts) __attribute__((always_inline)) {
        const uint64_t all = __builtin_amdgcn_ballot_w64(counts);
        if (all == 0) return;
        // (equal weights, as of places that nobody has looked at, would queue for one bin)
        const uint32_t its = __builtin_amdgcn_readlane(bin, __builtin_ctzll(all));
        if (__builtin_amdgcn_ballot_w64(counts && bin == its) == all) {
            if (lane == 0) atomicAdd(&bins[its], __popcll(all));
        } else if (counts) {
            atomicAdd(&bins[bin], 1);
        }
    };
    if constexpr (kInLds) keys.load([&](uint32_t key, bool counts) __attribute__((always_inline)) { count(key >> 21, counts); });  // (with the first histogram)
    uint32_t least = 0;      // upper bits of the threshold
    int32_t wanted = best;   // how many with those bits
    bool tie = false;        // whether some that equal the threshold go
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
        const uint32_t above = digit == 0 ? 0 : ~0u << (shift + bits);
        for (int32_t i = threadIdx.x; i - lane < quads && !(kInLds && digit == 0); i += 1024) {
            const u32x4 key = i < quads ? keys.at(i) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) count((key[j] >> shift) & ((1u << bits) - 1), 4 * i + j < n && ((key[j] ^ least) & above) == 0);
        }
        __syncthreads();
        // the bin in which the wanted one is, from above: a lane has two bins, which it clears for the next digit
        const int at = kBins - 2 - 2 * threadIdx.x;
        const int32_t hi = bins[at + 1], lo = bins[at];
        bins[at + 1] = bins[at] = 0;
        int32_t upto = hi + lo;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int32_t o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        if (lane == 63) of_waves[0][wave] = upto;
        __syncthreads();
        upto += before_wave(of_waves[0], wave);
        const int32_t before = upto - hi - lo;
        if (before < wanted && wanted <= before + hi) found[0] = at + 1, found[1] = before, found[2] = hi;
        else if (before + hi < wanted && wanted <= upto) found[0] = at, found[1] = before + hi, found[2] = lo;
        __syncthreads();
        least |= (uint32_t)found[0] << shift;
        wanted -= found[1];
        tie = found[2] != wanted;
    }
    // `wanted` of those that equal the threshold stay, the lower places first; each wavefront has a run of places, a lane four next to each other
    const uint64_t below = (1ull << lane) - 1;
    const int32_t run = (quads + kWaves * 64 - 1) / (kWaves * 64) * 64, from = wave * run, to = min(from + run, quads);
    int32_t equal = 0;
    if (tie) {
        for (int32_t i = from + lane; i - lane < to; i += 64) {
            const u32x4 key = i < to ? keys.at(i) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) equal += __popcll(__builtin_amdgcn_ballot_w64(key[j] == least));
        }
        if (lane == 0) of_waves[0][wave] = equal;
        __syncthreads();
        equal = before_wave(of_waves[0], wave);
    }
    // which of a lane's four stay, which of those that do not are free places, which of those that do go there
    int32_t rank = equal;
    struct Four {
        uint32_t holes, movers;
    };
    auto four_at = [&](int32_t i) __attribute__((always_inline)) {
        const u32x4 key = i < to ? keys.at(i) : u32x4{0, 0, 0, 0};
        uint32_t stays = 0;
        if (tie) {
            uint64_t same[4];
            int32_t mine = rank;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                same[j] = __builtin_amdgcn_ballot_w64(key[j] == least);
                mine += __popcll(same[j] & below);
                rank += __popcll(same[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                stays |= (uint32_t)(key[j] > least || (key[j] == least && mine < wanted)) << j;
                mine += key[j] == least;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) stays |= (uint32_t)(key[j] >= least) << j;
        }
        // (places behind the last do not stay, and are not below best)
        const int32_t first = best - 4 * i;  // of the four, this many are below best
        const uint32_t in_front = first >= 4 ? 15u : first > 0 ? (1u << first) - 1 : 0;
        return Four{i < to ? ~stays & in_front : 0, stays & ~in_front & 15u};
    };
    int32_t holes = 0, movers = 0;
    for (int32_t i = from + lane; i - lane < to; i += 64) {
        const Four f = four_at(i);
        if (kInLds && i < to) keys.keys[i][0] = f.holes << 4 | f.movers;  // (the lane's own, and no longer a key)
        holes += __popc(f.holes);
        movers += __popc(f.movers);
    }
#pragma unroll
    for (int d = 32; d; d /= 2) {
        holes += __shfl_xor(holes, d);
        movers += __shfl_xor(movers, d);
    }
    if (lane == 0) of_waves[1][wave] = holes, of_waves[2][wave] = movers;
    __syncthreads();
    holes = before_wave(of_waves[1], wave);
    movers = before_wave(of_waves[2], wave);
    rank = equal;
    for (int32_t i = from + lane; i - lane < to; i += 64) {
        Four f;
        if constexpr (kInLds) {
            const uint32_t both = i < to ? keys.keys[i][0] : 0;
            f = {both >> 4, both & 15};
        } else {
            f = four_at(i);
        }
        if (__builtin_amdgcn_ballot_w64((f.holes | f.movers) != 0) == 0) continue;
        int32_t hole_at = holes, mover_at = movers;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t of_holes = __builtin_amdgcn_ballot_w64((f.holes >> j) & 1), of_movers = __builtin_amdgcn_ballot_w64((f.movers >> j) & 1);
            hole_at += __popcll(of_holes & below);
            mover_at += __popcll(of_movers & below);
            holes += __popcll(of_holes);
            movers += __popcll(of_movers);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if ((f.holes >> j) & 1) list[1 + hole_at++] = 4 * i + j;
            if ((f.movers >> j) & 1) list[1 + a.most + mover_at++] = 4 * i + j;
        }
    }
    if (threadIdx.x == 1023) list[0] = holes;  // (with those before the last wavefront)
}

// The moves of a head's list, then the latest places behind them, `recent` of them from length - recent to keep - recent: those may overlap themselves, so they go in
// ascending pieces, each read before it is written.  blockIdx as for cache_accept_kernel.  Bound by the look-ups and rows that wait for each other: 16 sequences of 8 heads of 128 elements, float16, cut from
// 2080 to 2048 places, 256 recent: 11 us (37 MB); 4 from 32768 to 8192, 1024 recent: 100 (220 MB, 2.2 TB/s: 160 work-groups, each with a slice's whole list behind each other), and 14.5 (39 MB) where most of
// what has weight lies in front already, as after an earlier cut.
template <typename Unit, int kThreads>
__global__ __launch_bounds__(kThreads) void cache_evict_kernel(MoveArgs a) {
    constexpr int kAtOnce = 4;
    const int32_t each = 2 * a.slices + 1, what = blockIdx.x % each, h = blockIdx.x / each % a.c.groups, b = blockIdx.x / each / a.c.groups;
    const int32_t length = clamped(a.c.lengths[b], a.c.places);
    if (length <= a.keep) return;
    const int32_t* list = a.lists + (int64_t)(b * a.c.groups + h) * (1 + 2 * a.most);
    const int32_t moves = list[0], latest = length - a.recent, to = a.keep - a.recent;
    const int32_t *to_list = list + 1, *from_list = list + 1 + a.most;
    if (what == 2 * a.slices) {
        float* mass = a.mass + b * a.mass_batch + h * a.mass_head;
        for (int32_t i = threadIdx.x; i < moves; i += kThreads) mass[to_list[i]] = mass[from_list[i]];
        for (int32_t i0 = 0; i0 < a.recent; i0 += kThreads) {
            const int32_t i = i0 + threadIdx.x;
            const float v = i < a.recent ? mass[latest + i] : 0.f;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (what is read here, or was above, may be written next)
            __syncthreads();
            if (i < a.recent) mass[to + i] = v;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        for (int32_t i = a.keep + threadIdx.x; i < length; i += kThreads) mass[i] = 0.f;
        return;
    }
    const int32_t slice = what % a.slices * kSlice, bytes = min(kSlice, a.row_bytes - slice), units = bytes / (int32_t)sizeof(Unit);
    const Rows r = what < a.slices ? Rows{a.c.k + h * a.c.k_head + slice, a.c.k_page, a.c.k_row} : Rows{a.c.v + h * a.c.v_head + slice, a.c.v_page, a.c.v_row};
    const int32_t rows = kThreads / units, mine = threadIdx.x / units, u = threadIdx.x % units;  // (units: at most 64)
    struct Piece {
        Unit v[kAtOnce];
        char* to[kAtOnce];
    };
    // the i-th and following ones of `count` rows: read, with where they go, which is asked for at the same time
    auto read = [&](Piece& piece, int32_t i0, int32_t count, auto from, auto to) __attribute__((always_inline)) {
        const char* at[kAtOnce];
        int32_t from_place[kAtOnce], to_place[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int32_t i = i0 + j * rows + mine;
            const bool there = mine < rows && i < count;
            from_place[j] = there ? from(i) : -1;
            to_place[j] = there ? to(i) : -1;
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            at[j] = row_at(a, r, b, from_place[j]);
            piece.to[j] = row_at(a, r, b, to_place[j]);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            if (at[j] == nullptr) piece.to[j] = nullptr;
            else piece.v[j] = reinterpret_cast<const Unit*>(at[j])[u];
        }
    };
    auto write = [&](const Piece& piece) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (piece.to[j]) reinterpret_cast<Unit*>(piece.to[j])[u] = piece.v[j];
    };
    auto read_moved = [&](Piece& piece, int32_t i0) __attribute__((always_inline)) { read(piece, i0, moves, [&](int32_t i) { return from_list[i]; }, [&](int32_t i) { return to_list[i]; }); };
    auto read_latest = [&](Piece& piece, int32_t i0) __attribute__((always_inline)) { read(piece, i0, a.recent, [&](int32_t i) { return latest + i; }, [&](int32_t i) { return to + i; }); };
    // The rows of the list, whose places are apart from those they come from; its last piece with the first of the latest rows, which may go where rows of the list came from.
    const int32_t step = rows * kAtOnce;
    Piece moved, late;
    int32_t i0 = 0;
    for (; i0 + step < moves; i0 += step) {
        read_moved(moved, i0);
        write(moved);
    }
    read_moved(moved, i0);
    read_latest(late, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    write(moved);
    write(late);
    for (i0 = step; i0 < a.recent; i0 += step) {
        read_latest(late, i0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        write(late);
    }
}

// Launches for units of 16, 8, 4 or 2 bytes.
template <typename F>
int by_unit(int unit, F f) {
    switch (unit) {
        case 16: return f(u32x4{});
        case 8: return f(uint64_t{});
        case 4: return f(uint32_t{});
        default: return f(uint16_t{});
    }
}

int unit_of_cache(const CacheArgs& c, int32_t row_bytes) {
    return unit_of({at_of(c.k), at_of(c.v), c.k_page, c.k_row, c.k_head, c.v_page, c.v_row, c.v_head, row_bytes});
}

int check_moves(const chx_hip_tensor* keys, const chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, const chx_hip_tensor* more,
                const chx_hip_tensor* mass, const chx_hip_tensor* new_lengths, const char* what, MoveArgs* a) {
    memset(a, 0, sizeof(*a));
    CHX_PROPAGATE(check_cache(keys, values, tables, lengths, what, &a->c));
    CHX_REQUIRE(numel(*keys) == 0 || (elements_apart(*keys) && elements_apart(*values)), "%s: elements of keys or values overlap", what);
    if (mass) {
        CHX_PROPAGATE(check_mass(mass, a->c, what));
        a->mass = static_cast<float*>(mass->data);
        a->mass_batch = mass->strides[0] / 4;
        a->mass_head = mass->strides[1] / 4;
    }
    CHX_PROPAGATE(check_numbers(new_lengths, 1, a->c.B, 0, what, "new_lengths"));
    const Named all[] = {{values, "values"}, {tables, "tables"}, {lengths, "lengths"}, {more, "accepted"}, {mass, "mass"}, {new_lengths, "new_lengths"}};
    CHX_PROPAGATE(check_apart({keys, "keys"}, all, 6, what));
    CHX_PROPAGATE(check_apart({values, "values"}, all + 1, 5, what));
    CHX_PROPAGATE(check_apart({mass, "mass"}, all + 1, 3, what));
    CHX_PROPAGATE(check_apart({new_lengths, "new_lengths"}, all + 1, 4, what));
    a->new_lengths = static_cast<int32_t*>(new_lengths->data);
    a->row_bytes = a->c.D * dtype_size(keys->dtype);
    a->slices = (a->row_bytes + kSlice - 1) / kSlice;
    CHX_REQUIRE((int64_t)a->c.B * a->c.groups * (2 * a->slices + 1) < (int64_t(1) << 22), "%s: more sequences and heads than one launch has", what);
    return CHX_HIP_OK;
}

int64_t evict_workspace(int64_t sequences, int64_t heads, int64_t places, int64_t keep) {
    // (places that move are at most as many as stay, or as are left)
    const int64_t most = keep < places - keep ? keep : places > keep ? places - keep : 0;
    return 4 * sequences * heads * (1 + 2 * most);
}

}  // namespace
}  // namespace chx

using namespace chx;

extern "C" int chx_hip_cache_append(
        chx_hip_tensor* keys, chx_hip_tensor* values, const chx_hip_tensor* k, const chx_hip_tensor* v, const chx_hip_tensor* tables, const chx_hip_tensor* lengths,
        const chx_hip_tensor* counts, void* stream) {
    const char* what = "cache append";
    AppendArgs a;
    memset(&a, 0, sizeof(a));
    CHX_PROPAGATE(check_cache(keys, values, tables, lengths, what, &a.c));
    CHX_REQUIRE(numel(*keys) == 0 || (elements_apart(*keys) && elements_apart(*values)), "%s: elements of keys or values overlap", what);
    CHX_PROPAGATE(check_rows(k, 4, keys->dtype, what, "k"));
    CHX_PROPAGATE(check_rows(v, 4, keys->dtype, what, "v"));
    CHX_REQUIRE(same_shape(*k, *v) && k->shape[0] == a.c.B && k->shape[2] == a.c.groups && k->shape[3] == a.c.D, "%s: k and v must be [sequences, tokens, heads, elements] as the cache has them", what);
    CHX_REQUIRE(k->shape[1] < (int64_t(1) << 30), "%s: 2^30 tokens", what);
    if (counts) {
        CHX_PROPAGATE(check_numbers(counts, 1, a.c.B, 0, what, "counts"));
        a.counts = static_cast<const int32_t*>(counts->data);
    }
    const Named all[] = {{values, "values"}, {k, "k"}, {v, "v"}, {tables, "tables"}, {lengths, "lengths"}, {counts, "counts"}};
    CHX_PROPAGATE(check_apart({keys, "keys"}, all, 6, what));
    CHX_PROPAGATE(check_apart({values, "values"}, all + 1, 5, what));
    if (numel(*k) == 0 || numel(*keys) == 0 || a.c.places == 0) return CHX_HIP_OK;
    a.k = static_cast<const char*>(k->data);
    a.v = static_cast<const char*>(v->data);
    a.k_batch = stride_of(*k, 0), a.k_token = stride_of(*k, 1), a.k_head = stride_of(*k, 2);
    a.v_batch = stride_of(*v, 0), a.v_token = stride_of(*v, 1), a.v_head = stride_of(*v, 2);
    a.T = (int32_t)k->shape[1];
    const int32_t row_bytes = a.c.D * dtype_size(keys->dtype);
    const int unit = unit_of({unit_of_cache(a.c, row_bytes), at_of(a.k), at_of(a.v), a.k_batch, a.k_token, a.k_head, a.v_batch, a.v_token, a.v_head});
    a.units = row_bytes / unit;
    a.pieces = (int64_t)a.c.B * a.T * a.c.groups * a.units;
    return by_unit(unit, [&](auto u) {
        return in_launches((a.pieces + 255) / 256, "cache_append_kernel",
                           [&](int64_t first, unsigned count) { cache_append_kernel<decltype(u)><<<count, 256, 0, as_stream(stream)>>>(a, first); });
    });
}

extern "C" int chx_hip_cache_accept(
        chx_hip_tensor* keys, chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, const chx_hip_tensor* accepted, chx_hip_tensor* mass,
        chx_hip_tensor* new_lengths, void* stream) {
    const char* what = "cache accept";
    MoveArgs a;
    CHX_PROPAGATE(check_tensor(accepted, "accepted"));
    CHX_PROPAGATE(check_moves(keys, values, tables, lengths, accepted, mass, new_lengths, what, &a));
    CHX_PROPAGATE(check_numbers(accepted, 2, a.c.B, -1, what, "accepted"));
    CHX_REQUIRE(accepted->shape[1] <= kMostAccepted, "%s: at most %d rows of a sequence, not %lld", what, kMostAccepted, (long long)accepted->shape[1]);
    if (a.c.B == 0) return CHX_HIP_OK;
    a.accepted = static_cast<const int32_t*>(accepted->data);
    a.most = (int32_t)accepted->shape[1];
    const unsigned grid = (unsigned)(a.c.B * a.c.groups * (2 * a.slices + (a.mass ? 1 : 0)));
    return by_unit(unit_of_cache(a.c, a.row_bytes), [&](auto u) {
        cache_accept_kernel<decltype(u)><<<grid, 256, 0, as_stream(stream)>>>(a);
        return launch_check("cache_accept_kernel");
    });
}

extern "C" int chx_hip_cache_evict_workspace(int64_t sequences, int64_t heads, int64_t places, int64_t keep, size_t* bytes) {
    CHX_REQUIRE(bytes != nullptr, "cache evict: null output");
    CHX_REQUIRE(sequences >= 0 && heads >= 0 && places >= 0 && sequences < (int64_t(1) << 24) && heads < (int64_t(1) << 16) && places < (int64_t(1) << 30), "cache evict: numbers of a cache out of range");
    CHX_REQUIRE(keep >= 0, "cache evict: keep is negative");
    CHX_REQUIRE(sequences * heads < (int64_t(1) << 22), "cache evict: more sequences and heads than one launch has");
    *bytes = (size_t)evict_workspace(sequences, heads, places, keep);
    return CHX_HIP_OK;
}

extern "C" int chx_hip_cache_evict(
        chx_hip_tensor* keys, chx_hip_tensor* values, const chx_hip_tensor* tables, const chx_hip_tensor* lengths, chx_hip_tensor* mass, int64_t keep, int64_t recent,
        chx_hip_tensor* new_lengths, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "cache evict";
    MoveArgs a;
    CHX_PROPAGATE(check_tensor(mass, "mass"));
    CHX_PROPAGATE(check_moves(keys, values, tables, lengths, nullptr, mass, new_lengths, what, &a));
    CHX_REQUIRE(recent >= 0 && recent <= keep, "%s: 0 to keep places can be recent, not %lld of %lld", what, (long long)recent, (long long)keep);
    const int64_t needed = evict_workspace(a.c.B, a.c.groups, a.c.places, keep);
    CHX_REQUIRE((int64_t)workspace_bytes >= needed && (needed == 0 || (workspace != nullptr && aligned(workspace, 4))), "%s: a workspace of %lld bytes, aligned to 4, is needed", what,
                (long long)needed);
    if (a.c.B == 0) return CHX_HIP_OK;
    a.keep = (int32_t)(keep < a.c.places ? keep : a.c.places);  // (no sequence is longer)
    a.recent = (int32_t)(recent < a.keep ? recent : a.keep);
    a.most = (int32_t)((needed / 4 / ((int64_t)a.c.B * a.c.groups) - 1) / 2);
    a.lists = static_cast<int32_t*>(workspace);
    const bool in_lds = a.c.places <= kMostInLds;
    auto choose = in_lds ? cache_choose_kernel<true> : cache_choose_kernel<false>;
    if (in_lds && a.c.places > 12 * 1024 - 256)  // (has to be asked for, on every device)
        CHX_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(choose), hipFuncAttributeMaxDynamicSharedMemorySize, 4 * kMostInLds));
    choose<<<(unsigned)(a.c.B * a.c.groups), 1024, in_lds ? (4 * a.c.places + 15) / 16 * 16 : 0, as_stream(stream)>>>(a);
    CHX_PROPAGATE(launch_check("cache_choose_kernel"));
    if (a.keep >= a.c.places) return CHX_HIP_OK;
    const unsigned grid = (unsigned)(a.c.B * a.c.groups * (2 * a.slices + 1));
    return by_unit(unit_of_cache(a.c, a.row_bytes), [&](auto u) {
        // (smaller work-groups where there are more than two of the larger ones to a compute unit)
        if (grid > 512) cache_evict_kernel<decltype(u), 512><<<grid, 512, 0, as_stream(stream)>>>(a);
        else cache_evict_kernel<decltype(u), 1024><<<grid, 1024, 0, as_stream(stream)>>>(a);
        return launch_check("cache_evict_kernel");
    });
}
