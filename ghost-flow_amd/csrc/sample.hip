// sample.hip -- tokens from logits: temperature, top-k, top-p and min-p per row, from
// given uniform numbers.
//
//   z_i = (l_i - max l) / T,  w_i = exp z_i
// over a row in the order (larger logit, then lower index): the first k; of those the
// ones with less than p sum w before them (and the first); of those w_i >= min_p.  The
// token is the first of them, by index, whose running sum of w exceeds u times their
// total.
//
// Weights are integers, round(w 2^44): sums are exact in 64 bits (up to 2^19 entries),
// the same in any order.  A border between two tokens is off by what the roundings before
// it add up to: some 2^-35 of the largest weight where they are independent, and n 2^-45 for
// n logits that are equal, 2^-26 at worst (a step of u is 2^-24).  An exponential is a table
// of 2^(j / 128), a polynomial of four terms beyond (2e-15) and the exponent: 17 operations
// without a branch, 9 of them fp64, which this card issues at the rate of fp32.
//
// Two launches.  The first (a workgroup per 4096 logits, read once) leaves the largest of
// every 16, of its 4096 and where it is, and, where the row's settings need the sum of all
// weights, that of its own, under top-p in bins of a 16th of z as well.  The second has a
// workgroup per row:
//  * no filter: the sums find the 4096 that hold the token;
//  * top-k, min_p (pick_from_few): the k-th largest of the 16s' maxima bounds the k-th
//    largest logit from below, so a few groups, found without reading the row, hold all
//    candidates; up to 512 (or what one histogram leaves of more) are put in order, each
//    counting those before it, and of up to 7168 the cut is found by radix (a call for 64
//    rows: top-k 400 of 1644 22 us, in order by counting 100; 1000 of 131072 32);
//  * top-p (pick_by_bins): the bins say which one is cut, one pass over the row collects
//    its logits, and their bits say the cut;
//  * anything else, such as a larger k or one bin of equal logits (pick_from_row): the row
//    is searched whole, by bins, then the cut's 32 bits by eleven, eleven and ten.
//
// Bound by the way through a row's single workgroup, and the first launch of many rows by the
// vector ALU: some 36 instructions to a logit without filters, 12.6 us of issue of the 13.7 that
// the CUs are busy with 256 rows of 50257 (2.5 are an empty launch's; LDS 2.6, half of that
// conflicts of the table's look-ups).  Launches, us: one row of 32000, top-k and top-p, fp32 3.3
// and 12; 64 rows of 131072, settings of all kinds, bf16 10 and 26; 256 rows of 50257 without
// filters, fp32 18 (2.8 TB/s) and 7.  Per stage of top-p over 131072: 3 to the cut cell and
// bin, 9 to list the bin, 5 to the cut's key, 4 to the token.
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace gfh {
namespace {

constexpr int kGroup = 16, kSlice = 4096, kGroups = kSlice / kGroup;  // logits; groups of a slice
constexpr int kMaxSlices = 128;
constexpr int kBins = 512, kCell = 16, kCells = kBins / kCell;  // of a 16th of z; bins summed together
constexpr int kStored = kBins + kCells;  // of a slice
constexpr int kDigits = 2048;    // a radix step
constexpr int kGuess = 1024, kPickThreads = 1024;
constexpr int kPerPick = kSlice / kPickThreads;  // logits of a slice per thread
constexpr int kListed = 7168;  // candidates, or logits of a bin
constexpr int kHot = 4096;     // groups that have candidates
constexpr int kFew = 512;      // candidates that are put in order
constexpr int kTable = 128;
constexpr double kOne = 0x1p44;
static_assert((int64_t)kMaxSlices * kSlice == (int64_t)1 << 19, "sums of that many weights in 64 bits");

struct Slice {
    float most;     // -inf: nothing can be drawn
    int at;         // the first place of it
    uint64_t sum;   // of weights relative to most
};

struct SampleParams {
    const char *logits;
    int64_t ld;  // elements
    int vocab, slices;
    const float *u;
    gfh_sampling set;
    float *maxima;  // [row][slices kGroups], -inf past the vocabulary
    Slice *slice;   // [row][slices]
    uint64_t *bins; // [row][slices][kBins and kCells] sums of weights relative to the slice's most, where Settings::bins
    int32_t *tokens;
    float *logprobs;  // nullable
};

// A row's settings: 0 / 1 / 0 for no top-k, top-p, min-p.
struct Settings {
    float temperature;
    int k;
    double p, min_p;
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.f); }
    // whether the sum of all weights is needed
    __device__ __forceinline__ bool all() const { return !greedy() && !k && (p < 1.0 || !(min_p > 0.0)); }
    __device__ __forceinline__ bool bins(int slices) const { return all() && p < 1.0 && slices > 1; }
    __device__ __forceinline__ float per() const { return 16.f / temperature; }
};
__device__ __forceinline__ Settings settings(const SampleParams &s, int row) {
    // (no branch around a load, so all are on their way at once: u stands in for absent rows)
    const auto given = [&](const float *of, float all) {
        const float x = (of ? of : s.u)[row];
        return of ? x : all;
    };
    const int32_t *const ks = s.set.top_ks ? s.set.top_ks : reinterpret_cast<const int32_t *>(s.u);
    const float temperature = given(s.set.temperatures, s.set.temperature), p = given(s.set.top_ps, s.set.top_p),
                min_p = given(s.set.min_ps, s.set.min_p);
    const int32_t some = ks[row], k = s.set.top_ks ? some : s.set.top_k;
    Settings r;
    r.temperature = temperature;
    r.k = k < 0 || k >= s.vocab ? 0 : k;
    r.p = p < 1.f ? (double)p : 1.0;
    r.min_p = min_p > 0.f ? (double)min_p : 0.0;
    if (r.min_p > 1.0) r.k = 1;  // none but the first
    return r;
}

// exp((l - most) / T) 2^44, rounded, plus 2^52 in the bits of a double, for finite most and
// l below infinity; scale = 128 log2 e / T, table[j] = 2^(j / 128 + 44).
__device__ __forceinline__ uint64_t weight_bits(float l, double most, double scale, const double *table) {
    // (-inf goes to what rounds to 0, and so does NaN, which 0 times it is)
    const double y = fmax(((double)l - most) * scale, -128.0 * 47);
    const double t = y + 0x1.8p52;  // its low bits: y rounded
    const int n = (int)(uint32_t)__double_as_longlong(t);
    const double r = y - (t - 0x1.8p52);  // in 128ths of an octave
    constexpr double c = 0x1.62e42fefa39efp-8;  // ln 2 / 128
    double e = fma(r, c * c * c * c / 24, c * c * c / 6);
    e = fma(r, e, c * c / 2);
    e = fma(r, e, c);
    e = fma(r, e, 1.0);
    // times 2^(n / 128 + 44), the integer part of n / 128 straight into the exponent
    const uint64_t f = __double_as_longlong(table[n & (kTable - 1)]);
    const uint32_t hi = (uint32_t)(f >> 32) + ((uint32_t)(n & -kTable) << 13);
    return __double_as_longlong(fma(e, __longlong_as_double((uint64_t)hi << 32 | (uint32_t)f), 0x1p52));
}
constexpr uint64_t kBitsOfZero = 0x4330000000000000ull;  // of 2^52
__device__ __forceinline__ uint64_t weight(float l, float most, double scale, const double *table) {
    if (most == INFINITY) return l == most ? (uint64_t)1 << 44 : 0;
    return weight_bits(l, (double)most, scale, table) - kBitsOfZero;
}
__device__ __forceinline__ void fill_table(double *table, int tid) {
    if (tid < kTable) table[tid] = exp2(tid * (1.0 / kTable)) * kOne;
}
constexpr double kLog2e = 1.4426950408889634;
__device__ __forceinline__ double weight_scale(float temperature) { return kTable * kLog2e / (double)temperature; }
// exp2 of (a - b) in units of scale, for a <= b; 0 where b alone is infinite
__device__ __forceinline__ double relative(float a, float b, double scale) {
    return a == b ? 1.0 : b == INFINITY || a == -INFINITY ? 0.0 : exp2(((double)a - (double)b) * scale * (1.0 / kTable));
}

// The bin of a logit: 16ths of z on a grid that does not depend on the row, counted from
// the largest's down; not rising with l.  (Where the grid's numbers leave their range all
// have the last.)
__device__ __forceinline__ float grid_of(float l, float per) { return floorf(l * per); }
__device__ __forceinline__ int bin_of(float l, float top, float per) {
    return (int)fmaxf(fminf(top - grid_of(l, per), (float)(kBins - 1)), 0.f);
}
// The highest bin of the grid's cell of kCell bins: where a slice's bins count from, so that
// the cells of slices meet.
__device__ __forceinline__ float cell_top(float bin) { return floorf(bin * (1.f / kCell)) * kCell + (kCell - 1); }

// A group of logits as it lies in memory (rows begin anywhere that their type allows),
// and in fp32: -inf for NaN and from `end` on.  Apart, so that loads can be on their way.
template <typename T>
struct Group {
    static constexpr int E = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    vec v[kGroup / E];

    __device__ __forceinline__ void load(const T *row, int first, int end) {
        if (first + kGroup <= end) {
            load_whole(row + first);
        } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) v[e / E][e % E] = first + e < end ? row[first + e] : (T)-INFINITY;
        }
    }
    __device__ __forceinline__ void load_whole(const T *from) {
#pragma unroll
        for (int i = 0; i < kGroup / E; ++i) v[i] = *reinterpret_cast<const vec *>(from + i * E);
    }
    __device__ __forceinline__ float value(int e) const { return (float)v[e / E][e % E]; }
    __device__ __forceinline__ void values(float (&x)[kGroup]) const {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) {
            x[e] = value(e);
            x[e] = x[e] == x[e] ? x[e] : -INFINITY;
        }
    }
};
template <typename T>
__device__ __forceinline__ void load_group(const T *row, int first, int end, float (&x)[kGroup]) {
    Group<T> g;
    g.load(row, first, end);
    g.values(x);
}

// ---- a wave's lanes, in the VALU: the LDS path's permutes, one after the other, cost more -----
//
// x of the lane that a DPP pattern names; 0 where it names none, and outside the rows of 16.
template <int PATTERN, int ROWS = 0xf, typename T>
__device__ __forceinline__ T from_lane(T x) {
    constexpr int N = sizeof(T) / 4;
    typedef int words __attribute__((ext_vector_type(N)));
    words w;
    if constexpr (N == 1) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), PATTERN, ROWS, 0xf, false));
    } else {
        w = __builtin_bit_cast(words, x);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], PATTERN, ROWS, 0xf, false);
        return __builtin_bit_cast(T, w);
    }
}
template <typename T>
__device__ __forceinline__ T of_lane(T x, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    }
}
// The sum of a lane's x and those of the lanes before it.
template <typename T>
__device__ __forceinline__ T sum_upto(T x) {
    x += from_lane<0x111>(x);       // row_shr:1
    x += from_lane<0x112>(x);       // row_shr:2
    x += from_lane<0x114>(x);       // row_shr:4
    x += from_lane<0x118>(x);       // row_shr:8
    x += from_lane<0x142, 0xa>(x);  // row_bcast:15, to the second and fourth row
    x += from_lane<0x143, 0xc>(x);  // row_bcast:31, to the upper two
    return x;
}
// f over all lanes, in each; every lane has to be active.
template <typename T, typename F>
__device__ __forceinline__ T over_wave(T x, F &&f) {
    x = f(x, from_lane<0xB1>(x));   // quad_perm [1,0,3,2]
    x = f(x, from_lane<0x4E>(x));   // quad_perm [2,3,0,1]
    x = f(x, from_lane<0x141>(x));  // row_half_mirror
    x = f(x, from_lane<0x140>(x));  // row_mirror
    return f(f(of_lane(x, 0), of_lane(x, 16)), f(of_lane(x, 32), of_lane(x, 48)));
}
constexpr auto add = [](auto a, auto b) { return a + b; };
constexpr auto smaller = [](int a, int b) { return min(a, b); };
constexpr auto larger = [](auto a, auto b) { return a > b ? a : b; };

template <typename T>
__global__ __launch_bounds__(kGroups) void sample_slices_kernel(SampleParams s) {
    __shared__ double table[kTable];
    __shared__ uint64_t hist[kBins];
    __shared__ float mosts[4];
    __shared__ int ats[4];
    __shared__ uint64_t sums[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / s.slices, slice = blockIdx.x - row * s.slices;
    const Settings set = settings(s, row);
    const int first = slice * kSlice + tid * kGroup;
    float x[kGroup];
    load_group(reinterpret_cast<const T *>(s.logits) + row * s.ld, first, s.vocab, x);
    fill_table(table, tid);
    for (int i = tid; i < kBins; i += kGroups) hist[i] = 0;
    float most = x[0];
#pragma unroll
    for (int e = 1; e < kGroup; ++e) most = fmaxf(most, x[e]);
    s.maxima[((int64_t)row * s.slices + slice) * kGroups + tid] = most;
    int at = INT_MAX;
#pragma unroll
    for (int e = kGroup - 1; e >= 0; --e) at = x[e] == most ? first + e : at;
    const float highest = over_wave(most, larger);
    at = over_wave(most == highest ? at : INT_MAX, smaller);
    if (lane == 0) mosts[wave] = highest, ats[wave] = at;
    __syncthreads();
    most = mosts[0], at = ats[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (mosts[w] > most) most = mosts[w], at = ats[w];
    uint64_t sum = 0;
    if (set.all()) {
        const bool bins = set.bins(s.slices);
        const double scale = weight_scale(set.temperature);
        const float per = set.per(), top = cell_top(grid_of(most, per));
        if (most < INFINITY && most > -INFINITY) {
            uint64_t w[kGroup];
#pragma unroll
            for (int e = 0; e < kGroup; ++e) w[e] = weight_bits(x[e], (double)most, scale, table) - kBitsOfZero;
#pragma unroll
            for (int e = 0; e < kGroup; ++e) sum += w[e];
            if (bins) {
#pragma unroll
                for (int e = 0; e < kGroup; ++e)
                    if (w[e]) atomicAdd((unsigned long long *)&hist[bin_of(x[e], top, per)], (unsigned long long)w[e]);
            }
        } else if (most == INFINITY) {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) sum += weight(x[e], most, scale, table);
        }
        sum = over_wave(sum, add);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = sums[0] + sums[1] + sums[2] + sums[3];
        if (bins) {
            // (the last bin, of all that lies further down, is no use)
            uint64_t *const to = s.bins + ((int64_t)row * s.slices + slice) * kStored;
            static_assert(kBins == 2 * kGroups && kCell == 16, "eight threads to a cell");
            const uint64_t a = hist[2 * tid], b = 2 * tid + 1 < kBins - 1 ? hist[2 * tid + 1] : 0;
            to[2 * tid] = a, to[2 * tid + 1] = b;
            uint64_t c = a + b;
            c += from_lane<0xB1>(c);
            c += from_lane<0x4E>(c);
            c += from_lane<0x141>(c);
            if (tid % 8 == 0) to[kBins + tid / 8] = c;
        }
    }
    if (tid == 0) s.slice[(int64_t)row * s.slices + slice] = {most, at, sum};
}

// ---- the second launch ------------------------------------------------------------

// Logits that the cut lies among.
struct List {
    __attribute__((aligned(16))) uint32_t key[kListed];
    int at[kListed];
};
// A few of them, in order.
struct Few {
    uint64_t weight[kFew];
    int rank[kFew], order[kFew];
};

struct PickShared {
    double table[kTable];
    uint64_t wave_sums[2][kPickThreads / 64];
    double slice_sums[kMaxSlices];   // running sums of all weights
    double slice_scale[kMaxSlices];  // of a slice's weights in the row's
    double kept[kMaxSlices];
    uint64_t tied[kMaxSlices];
    int slice_cell[kMaxSlices];      // cells from the row's first to its own
    uint32_t count[kDigits];
    __attribute__((aligned(16))) uint64_t sum[kDigits];  // (or doubles, kHot numbers of groups, Few)
    List list;
    int found, n;
    uint32_t edge[2];
    uint64_t found_count, found_sum;
    double above;
};

// The low bits of a key that are the same for all values of a type of one sign.
template <typename T>
constexpr int kZeroBits = std::is_same_v<T, float> ? 0 : std::is_same_v<T, _Float16> ? 13 : 16;

// Inclusive sum over the workgroup's threads, and the total; call after call takes
// the other half of wave_sums, so one barrier does.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, PickShared &sh, int &turn, int tid, uint64_t &total) {
    const int lane = tid & 63, wave = tid >> 6;
    x = sum_upto(x);
    uint64_t *const sums = sh.wave_sums[turn];
    turn ^= 1;
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPickThreads / 64; ++w) {
        before += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    return before + x;
}

// Larger logits have larger keys; all that cannot be drawn the lowest.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t u = __float_as_uint(l == 0.f ? 0.f : l);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// The logit of a complemented key.
__device__ __forceinline__ float logit_of(uint32_t inverse) {
    const uint32_t key = ~inverse;
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct Row {
    float most, top, per;  // largest logit, its bin of the grid, bins to a unit of it
    double scale;
    int k;
    double p, min_p;
    double u;
};

// The logarithm of a token's probability among those of weight `total`.
__device__ __forceinline__ void answer(const SampleParams &s, int row, int token, float l, const Row &r, double total) {
    s.tokens[row] = token;
    if (!s.logprobs) return;
    const double z = l == r.most ? 0.0 : ((double)l - (double)r.most) * (r.scale * (1.0 / (kTable * kLog2e)));
    s.logprobs[row] = (float)(z - log(total / kOne));
}
// floor(u total), below total.
__device__ __forceinline__ uint64_t target_of(double u, uint64_t total) {
    const double t = fmin(fmax(u, 0.0), 1.0) * (double)total;
    const uint64_t n = (uint64_t)t;
    return n < total ? n : total - 1;
}

// The slice that holds the token, by the slices' running sums of what stays, then the token
// in it; stays(l, first, b) says which of a thread's logits do.  A slice far below the largest
// has a sum, if a small one, and no weight that is not 0 here: then the token is the first
// behind it that has one, or, where none does, the last before it.
template <typename T, typename F>
__device__ __forceinline__ void pick_in_slice(const SampleParams &s, int row, const Row &r, PickShared &sh, int &turn,
                                              int tid, const double *sums, F &&stays) {
    const double total = sums[s.slices - 1], aim = fmin(fmax(r.u, 0.0), 1.0) * total;
    if (tid < 64) {
        int n = 0, last = -1;
        for (int i = tid; i < s.slices; i += 64) {
            const double before = i ? sums[i - 1] : 0.0;
            n += sums[i] <= aim;
            last = sums[i] > before ? i : last;
        }
        n = over_wave(n, add);
        last = over_wave(last, larger);
        if (tid == 0) sh.found = min(n, last);
    }
    __syncthreads();
    const int found = sh.found;
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    constexpr int kPer = kPerPick;
    for (int i = 0; i < s.slices; ++i) {  // (ends at the first, or where the row's largest is)
        const bool back = found + i >= s.slices;
        const int slice = back ? s.slices - 1 - i : found + i, first = slice * kSlice + tid * kPer;
        float l[kPer];
        bool in[kPer];
        uint64_t w[kPer], sum = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const float v = first + e < s.vocab ? (float)x[first + e] : -INFINITY;
            l[e] = v == v ? v : -INFINITY;
        }
        stays(l, first, in);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            w[e] = in[e] ? weight(l[e], r.most, r.scale, sh.table) : 0;
            sum += w[e];
        }
        uint64_t all;
        uint64_t before = block_scan(sum, sh, turn, tid, all) - sum;
        if (all == 0) continue;
        const double target = aim - (slice ? sums[slice - 1] : 0.0);
        uint64_t n = back ? all - 1 : i == 0 && target > 0.0 ? (uint64_t)target : 0;
        n = n < all ? n : all - 1;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (before <= n && n < before + w[e]) answer(s, row, first + e, l[e], r, total);
            before += w[e];
        }
        return;
    }
}

// The places of n <= kFew logits in the order, list.key their complemented keys and
// list.at rising: Few::order.  Each counts those before it.
__device__ __forceinline__ void put_in_order(PickShared &sh, Few &few, int n, int tid) {
    int size = 64;
    while (size < n) size <<= 1;
    if (tid < size) {
        few.rank[tid] = 0;
        if (tid >= n) sh.list.key[tid] = ~0u;  // (behind all)
    }
    __syncthreads();
    const int per = size * size / kPickThreads, i = tid % size;
    static_assert(64 * 64 >= 4 * kPickThreads && kFew <= kPickThreads, "four keys at a time");
    typedef uint32_t four __attribute__((ext_vector_type(4)));
    if (i < n) {
        // (equal ones count where they lie before; for most of the list the wave's 64 agree on that)
        const uint32_t mine = sh.list.key[i];
        const int first = tid / size * per, end = first + per, i0 = __builtin_amdgcn_readfirstlane(i & ~63);
        int before = 0;
        const auto count = [&](int from, int to, uint32_t least) {
#pragma unroll 4
            for (int j = from; j < to; j += 4) {
                const four k = *reinterpret_cast<const four *>(&sh.list.key[j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) before += k[e] < least;
            }
        };
        count(first, min(end, i0), mine + 1);
        for (int j = max(first, i0); j < min(end, i0 + 64); j += 4) {
            const four k = *reinterpret_cast<const four *>(&sh.list.key[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) before += k[e] < mine + (uint32_t)(j + e < i);
        }
        count(max(first, i0 + 64), end, mine);
        atomicAdd(&few.rank[i], before);
    }
    __syncthreads();
    if (tid < n) few.order[few.rank[tid]] = tid;
    __syncthreads();
}

// A cut among listed logits: those of complemented keys below lo stay, and the first
// `ties` of those up to hi, which are equal.
struct ListCut {
    uint32_t lo, hi;
    uint64_t ties, sum;  // sum of the weights that stay
    bool open;           // nothing is cut
};

// The first k of n listed logits in the order, of those the ones with less than `limit`
// before them (and the first).  The range of z that they lie in by 2048ths, then the keys
// between the lowest and the highest of the part that holds the cut (mostly one value),
// eleven bits at a time.
template <typename T>
__device__ __forceinline__ ListCut cut_list(const Row &r, PickShared &sh, int &turn, int tid, int n, int bins, uint64_t k,
                                            uint64_t limit) {
    uint64_t count = 0, sum = 0;  // before the part that is looked into
    uint32_t lo = 0, hi = ~0u;
    const float end = r.top + 1.f, per = (float)kDigits / (float)bins;
    for (bool parts = fabsf(r.top) < 0x1p22f && r.per > 0.f;; parts = false) {
        const int shift = max(0, 32 - __builtin_clz((hi - lo) | 1) - 11);
        const auto digit_of = [&](uint32_t key) {
            if (!parts) return (int)((key - lo) >> shift);
            return (int)fminf(fmaxf(fmaf(-logit_of(key), r.per, end) * per, 0.f), (float)(kDigits - 1));
        };
        __syncthreads();
        for (int i = tid; i < kDigits; i += kPickThreads) sh.count[i] = 0, sh.sum[i] = 0;
        if (tid == 0) sh.found = -1, sh.edge[0] = ~0u, sh.edge[1] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kPickThreads) {
            const uint32_t key = sh.list.key[i];
            if (key - lo > hi - lo) continue;
            const int digit = digit_of(key);
            atomicAdd(&sh.count[digit], 1u);
            atomicAdd((unsigned long long *)&sh.sum[digit],
                      (unsigned long long)weight(logit_of(key), r.most, r.scale, sh.table));
        }
        __syncthreads();
        uint64_t total;
        const uint64_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1], s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
        uint64_t cn = count + block_scan(c0 + c1, sh, turn, tid, total) - c0 - c1;
        uint64_t sn = sum + block_scan(s0 + s1, sh, turn, tid, total) - s0 - s1;
        // the first digit that the cut lies in or behind (found by one thread)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint64_t c = e ? c1 : c0, w = e ? s1 : s0;
            const bool open = cn < k && (sn < limit || cn == 0), shut = cn + c >= k || sn + w >= limit;
            if (c && open && shut) sh.found = 2 * tid + e, sh.found_count = cn, sh.found_sum = sn;
            cn += c, sn += w;
        }
        __syncthreads();
        const int at = sh.found;
        if (at < 0) return {~0u, ~0u, 0, sum + total, true};
        count = sh.found_count, sum = sh.found_sum;
        if (parts) {
            for (int i = tid; i < n; i += kPickThreads) {
                const uint32_t key = sh.list.key[i];
                if (digit_of(key) == at) atomicMin(&sh.edge[0], key), atomicMax(&sh.edge[1], key);
            }
            __syncthreads();
            lo = sh.edge[0], hi = sh.edge[1];
        } else {
            lo += (uint32_t)at << shift;
            hi = min(hi, lo + ((1u << shift) - 1));
        }
        if (lo == hi || (!parts && shift <= kZeroBits<T>)) {
            // equal logits, equal weights
            const uint64_t have = sh.count[at], w = sh.sum[at] / have;
            uint64_t ties = min(have, k - count);
            if (w) ties = min(ties, sum < limit ? (limit - sum - 1) / w + 1 : 0);
            if (count + ties == 0) ties = 1;
            return {lo, hi, ties, sum + ties * w, false};
        }
    }
}

// The listed logits of the 2048ths of the range of z up to the one where the first k end, or
// the first with `limit`, are moved together, if they are kFew at most; returns how many are
// listed then.  (They hold all that stays: the cut lies in the last part.)
__device__ __forceinline__ int narrow_list(const Row &r, PickShared &sh, int &turn, int tid, int n, int bins, uint64_t limit) {
    const float end = r.top + 1.f, per = (float)kDigits / (float)bins;
    const auto digit_of = [&](uint32_t key) {
        return (int)fminf(fmaxf(fmaf(-logit_of(key), r.per, end) * per, 0.f), (float)(kDigits - 1));
    };
    for (int i = tid; i < kDigits; i += kPickThreads) sh.count[i] = 0, sh.sum[i] = 0;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    constexpr int kMost = kListed / kPickThreads;
    static_assert(kMost * kPickThreads == kListed);
    const int each = (n + kPickThreads - 1) / kPickThreads, from = tid * each;
    uint32_t key[kMost];
    int at[kMost], digit[kMost];
#pragma unroll
    for (int e = 0; e < kMost; ++e) {
        digit[e] = kDigits;
        if (e >= each || from + e >= n) continue;
        key[e] = sh.list.key[from + e], at[e] = sh.list.at[from + e];
        digit[e] = digit_of(key[e]);
        atomicAdd(&sh.count[digit[e]], 1u);
        if (!r.k)
            atomicAdd((unsigned long long *)&sh.sum[digit[e]],
                      (unsigned long long)weight(logit_of(key[e]), r.most, r.scale, sh.table));
    }
    __syncthreads();
    uint64_t total;
    const uint64_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1], s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
    const uint64_t cn = block_scan(c0 + c1, sh, turn, tid, total), sn = r.k ? 0 : block_scan(s0 + s1, sh, turn, tid, total);
    // the first digit up to which there are enough (found by one thread)
    const uint64_t k = (uint64_t)r.k;
    const bool before = r.k ? cn - c0 - c1 >= k : sn - s0 - s1 >= limit, half = r.k ? cn - c1 >= k : sn - s1 >= limit,
               here = r.k ? cn >= k : sn >= limit;
    if (!before && here) sh.found = half ? 2 * tid : 2 * tid + 1, sh.found_count = half ? cn - c1 : cn;
    __syncthreads();
    if (sh.found < 0 || sh.found_count > kFew) return n;
    const int last = sh.found, left = (int)sh.found_count;
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < kMost; ++e) mine += digit[e] <= last;
    int to = (int)(block_scan(mine, sh, turn, tid, total) - mine);
#pragma unroll
    for (int e = 0; e < kMost; ++e)
        if (digit[e] <= last) sh.list.key[to] = key[e], sh.list.at[to] = at[e], ++to;
    __syncthreads();
    return left;
}

// Candidates, if they are few enough: the logits in bins up to the one that holds
// the k-th largest maximum of a group (top-k), of a quarter of the groups or the
// kGuess-th (top-p, which may need more, so not where all can be listed), or min_p.
// False: not enough, or too many.
template <typename T>
__device__ __forceinline__ bool pick_from_few(const SampleParams &s, int row, const Row &r, PickShared &sh, int tid,
                                              double all) {
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    const float *const maxima = s.maxima + (int64_t)row * s.slices * kGroups;
    const int groups = (s.vocab + kGroup - 1) / kGroup;
    int turn = 0;
    uint64_t total;
    int last = kBins - 1;  // bin of the last candidates
    bool guess = false;
    if (!r.k && r.min_p > 0.0 && fabsf(r.top) < 0x1p22f) {
        const double b = -log(r.min_p) * 16.0 + 3.0;  // (the grid's cell of the largest, and roundings)
        last = (int)fmin(fmax(b, 0.0), (double)(kBins - 1));
    }
    // this thread's groups: whole fours, neighbours, the first kHeld kept in registers
    constexpr int kHeld = 8;
    const int per = ((groups + kPickThreads - 1) / kPickThreads + 3) & ~3, g0 = tid * per, g1 = min(groups, g0 + per);
    int bin[kHeld];
    {
        f32x4 held[kHeld / 4];
#pragma unroll
        for (int i = 0; i < kHeld / 4; ++i)  // (all on their way at once)
            held[i] = *reinterpret_cast<const f32x4 *>(maxima + min(g0 + 4 * i, s.slices * kGroups - 4));
#pragma unroll
        for (int i = 0; i < kHeld; ++i) bin[i] = i < per && g0 + i < g1 ? bin_of(held[i / 4][i % 4], r.top, r.per) : kBins;
    }
    auto each_group = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (bin[i] < kBins) f(g0 + i, bin[i]);
        for (int i = g0 + kHeld; i < g1; ++i) f(i, bin_of(maxima[i], r.top, r.per));
    };
    if (r.k || (r.p < 1.0 && s.vocab > kListed)) {
        const int want = r.k ? r.k : min(kGuess, groups / 4 + 1);
        if (tid < kBins) sh.count[tid] = 0;
        __syncthreads();
        each_group([&](int, int b) { atomicAdd(&sh.count[b], 1u); });
        __syncthreads();
        if (tid < 64) {
            constexpr int kEach = kBins / 64;
            int c[kEach], n = 0, at = kBins - 1;
#pragma unroll
            for (int e = 0; e < kEach; ++e) n += c[e] = (int)sh.count[kEach * tid + e];
            int upto = sum_upto(n) - n;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                at = upto < want && upto + c[e] >= want ? kEach * tid + e : at;
                upto += c[e];
            }
            at = over_wave(at, smaller);
            if (tid == 0) sh.found = at;
        }
        __syncthreads();
        guess = !r.k && sh.found < last;
        last = min(last, sh.found);
    }
    // the groups that have candidates, in their order
    uint64_t mine = 0;
    each_group([&](int, int b) { mine += b <= last; });
    int at = (int)(block_scan(mine, sh, turn, tid, total) - mine);
    if (total > kHot) return false;
    const int hot = (int)total;
    int *const hots = reinterpret_cast<int *>(sh.sum);
    static_assert(sizeof(sh.sum) >= kHot * sizeof(int) && sizeof(sh.sum) >= sizeof(Few), "in place of the sums");
    if (mine) each_group([&](int g, int b) {
        if (b <= last) hots[at++] = g;
    });
    __syncthreads();
    // the candidates, in their order
    int n = 0;
    for (int h0 = 0; h0 < hot; h0 += kPickThreads) {
        float l[kGroup];
        int first = 0;
        uint32_t in = 0;
        if (h0 + tid < hot) {
            first = hots[h0 + tid] * kGroup;
            load_group(x, first, s.vocab, l);
#pragma unroll
            for (int e = 0; e < kGroup; ++e) in |= (uint32_t)(bin_of(l[e], r.top, r.per) <= last && first + e < s.vocab) << e;
        }
        const uint64_t c = __popc(in);
        at = n + (int)(block_scan(c, sh, turn, tid, total) - c);
        n += (int)total;
        if (n > kListed) return false;
#pragma unroll
        for (int e = 0; e < kGroup; ++e)
            if (in >> e & 1) {
                sh.list.key[at] = ~order_key(l[e]);
                sh.list.at[at] = first + e;
                ++at;
            }
    }
    __syncthreads();
    const double least = r.min_p * kOne;
    const auto limit_of = [&](double sum) {
        const double most = r.p * sum;
        return most > 0.0 ? (uint64_t)ceil(most) : 0;
    };
    const uint64_t none = ~(uint64_t)0;
    if (n > kFew && (r.k ? r.k < n && r.k <= kFew : r.p < 1.0) && fabsf(r.top) < 0x1p22f && r.per > 0.f)
        n = narrow_list(r, sh, turn, tid, n, last + 1, r.k ? none : limit_of(all));
    if (n <= kFew) {
        Few &few = *reinterpret_cast<Few *>(sh.sum);
        if (tid < n) few.weight[tid] = weight(logit_of(sh.list.key[tid]), r.most, r.scale, sh.table);
        put_in_order(sh, few, n, tid);
        // how many stay
        const int pos = tid < n ? few.order[tid] : 0;
        uint64_t w = tid < n ? few.weight[pos] : 0;
        const int k = r.k ? min(r.k, n) : n;
        const uint64_t inside = tid < k ? w : 0;  // (a place from k on does not stay anyway)
        uint64_t before = block_scan(inside, sh, turn, tid, total) - inside;
        uint64_t limit = none;
        if (r.p < 1.0) {
            limit = limit_of(r.k ? (double)total : all);
            if (guess && total < limit) return false;  // the next ones would stay too
        }
        const bool stays = tid == 0 || (tid < k && before < limit && (double)w >= least);
        if (tid < n && !stays) few.weight[pos] = 0;
        __syncthreads();
        w = tid < n ? few.weight[tid] : 0;
        before = block_scan(w, sh, turn, tid, total) - w;
        const uint64_t target = target_of(r.u, total);
        if (before <= target && target < before + w)
            answer(s, row, sh.list.at[tid], logit_of(sh.list.key[tid]), r, (double)total);
        return true;
    }
    ListCut cut{~0u, ~0u, 0, 0, true};
    // by k, then by p of what that leaves
#pragma unroll 1
    for (int step = r.k ? 0 : 1; step < (r.p < 1.0 ? 2 : 1); ++step) {
        const uint64_t limit = step ? limit_of(all) : none;
        cut = cut_list<T>(r, sh, turn, tid, n, last + 1, r.k ? (uint64_t)r.k : none, limit);
        if (cut.open && guess && cut.sum < limit) return false;
        all = (double)cut.sum;
    }
    // what stays, in the order of the indices: a thread's places are neighbours
    const int each = (n + kPickThreads - 1) / kPickThreads, from = tid * each, to = min(from + each, n);
    uint64_t equal = 0, sum = 0;
    for (int j = from; j < to; ++j) equal += !cut.open && sh.list.key[j] >= cut.lo && sh.list.key[j] <= cut.hi;
    const uint64_t ahead = block_scan(equal, sh, turn, tid, total) - equal;
    const auto weight_of = [&](int j, uint64_t &rank) {
        const uint32_t key = sh.list.key[j];
        const float l = logit_of(key);
        const bool stays = cut.open || key < cut.lo || (key <= cut.hi && rank++ < cut.ties);
        const uint64_t w = weight(l, r.most, r.scale, sh.table);
        return stays && (l == r.most || (double)w >= least) ? w : 0;
    };
    uint64_t rank = ahead;
#pragma unroll 1
    for (int j = from; j < to; ++j) sum += weight_of(j, rank);
    uint64_t before = block_scan(sum, sh, turn, tid, total) - sum;
    const uint64_t target = target_of(r.u, total);
    if (before <= target && target < before + sum) {
        rank = ahead;
        int j = from;
#pragma unroll 1
        for (;; ++j) {
            before += weight_of(j, rank);
            if (target < before) break;
        }
        answer(s, row, sh.list.at[j], logit_of(sh.list.key[j]), r, (double)total);
    }
    return true;
}

// top-p without top-k: the bins of the first launch say which bin the cut lies in; one
// pass over the row collects that bin's logits.  False: too many in it, or min_p may cut
// before.  (The last bin holds what lies more than 31 below the largest of its slice: 2^19
// e^-31 of the weights at most, less than the 2^-24 that p leaves.)
template <typename T>
__device__ __forceinline__ bool pick_by_bins(const SampleParams &s, int row, const Row &r, PickShared &sh, int tid,
                                             double all) {
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    const uint64_t *const bins = s.bins + (int64_t)row * s.slices * kStored;
    const Slice *const slices = s.slice + (int64_t)row * s.slices;
    if (!(fabsf(r.top) < 0x1p22f)) return false;
    const float top = cell_top(r.top);
    int turn = 0;
    double *const sums = reinterpret_cast<double *>(sh.sum);
    __syncthreads();
    if (tid < s.slices) {
        const float most = slices[tid].most;
        sh.slice_cell[tid] = most > -INFINITY ? (int)fminf(top - cell_top(grid_of(most, r.per)), (float)kBins) / kCell : kCells;
        sh.slice_scale[tid] = relative(most, r.most, r.scale);
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    const double limit = r.p * all;
    // the row's cells, 32 threads to each with every 32nd slice; the first that reaches the limit
    {
        constexpr int kParts = kPickThreads / kCells;
        const int c = tid % kCells;
        double sum = 0.0;
#pragma unroll 4
        for (int i = tid / kCells; i < s.slices; i += kParts) {
            const int at = c - sh.slice_cell[i];
            const uint64_t w = bins[i * kStored + kBins + max(at, 0)];
            sum += at >= 0 ? (double)w * sh.slice_scale[i] : 0.0;
        }
        sums[tid] = sum;
        __syncthreads();
        if (tid < 64) {
            double v = 0.0;
#pragma unroll
            for (int i = 0; i < kParts; ++i) v += sums[i * kCells + c];
            v = tid < kCells ? v : 0.0;
            const double upto = sum_upto(v) - v;
            const uint64_t here = __ballot(v > 0.0 && upto + v >= limit);
            if (tid == 0) sh.found = here ? __builtin_ctzll(here) : -1;
            if (here && tid == __builtin_ctzll(here)) sh.above = upto;
        }
        __syncthreads();
    }
    const int cell = sh.found;
    if (cell < 0) return false;
    // its bins in the same way, 64 threads to each
    {
        constexpr int kParts = kPickThreads / kCell;
        const double before = sh.above;
        const int b = tid % kCell;
        double sum = 0.0;
#pragma unroll 2
        for (int i = tid / kCell; i < s.slices; i += kParts) {
            const int at = cell - sh.slice_cell[i];
            const uint64_t w = bins[i * kStored + max(at, 0) * kCell + b];
            sum += at >= 0 ? (double)w * sh.slice_scale[i] : 0.0;
        }
        sums[tid] = sum;
        __syncthreads();
        if (tid < 64) {
            double v = 0.0;
#pragma unroll
            for (int i = 0; i < kParts / 4; ++i) v += sums[(i * 4 + tid / kCell) * kCell + b];
            v = quarter_sum_f64(v, tid);
            v = tid < kCell ? v : 0.0;
            const double upto = before + (sum_upto(v) - v);
            // (where the last bits say that none does, the last with anything)
            const uint64_t some = __ballot(v > 0.0), here = __ballot(v > 0.0 && upto + v >= limit);
            const int at = here ? __builtin_ctzll(here) : 63 - __builtin_clzll(some | 1);
            if (tid == 0) sh.found = cell * kCell + at;
            if (tid == at) sh.above = upto;
        }
        __syncthreads();
    }
    const int cut = sh.found;
    // min_p may take something of the bins up to this one
    if (r.min_p > 0.0 && !(exp(-(cut + 2) * (1.0 / 16)) >= r.min_p)) return false;
    const double above = sh.above;
    // what stays of every slice in the bins before: 32 lanes each
    for (int i0 = 0; i0 < s.slices; i0 += kPickThreads / 32) {
        const int i = min(i0 + tid / 32, s.slices - 1), c = tid % 32;
        const uint64_t *const of = bins + i * kStored;
        const int at = cell - sh.slice_cell[i];
        static_assert(kCells == 32 && kCell <= 32, "a lane per cell");
        const uint64_t whole = of[kBins + c], some = of[max(at, 0) * kCell + c % kCell];
        uint64_t w = (c < at ? whole : 0) + (at >= 0 && c < cut % kCell ? some : 0);
        w += from_lane<0xB1>(w);
        w += from_lane<0x4E>(w);
        w += from_lane<0x141>(w);
        w += from_lane<0x140>(w);
        w = tid & 32 ? of_lane(w, 32) + of_lane(w, 48) : of_lane(w, 0) + of_lane(w, 16);
        if (c == 0) sh.kept[i] = (double)w * sh.slice_scale[i];
    }
    // The bin's keys are neighbours, from the lowest whose grid number is the bin's to the
    // highest: a wave each looks for where it and the next one begin.
    if (tid < 128) {
        const float from = top - (float)cut + (float)(tid >> 6);
        uint32_t key = 0;  // all less than it are below
        const auto step = [&](int shift, uint32_t lanes) {
            const uint32_t lane = tid & 63, up = key | lane << shift;
            const float l = logit_of(~(up - 1));
            const bool below = l != l ? !(up >> 31) : grid_of(l, r.per) < from;
            key |= (uint32_t)(__popcll(__ballot(lane < lanes && (lane == 0 || below))) - 1) << shift;
        };
        for (int shift = 26; shift > 0; shift -= 6) step(shift, 64);
        step(0, 4);
        if ((tid & 63) == 0) sh.edge[tid >> 6] = key;
    }
    __syncthreads();
    uint32_t lo = sh.edge[0], hi = sh.edge[1] - 1;
    // the places of its logits, in any order, from the groups whose largest reaches it; a wave's
    // next groups are on their way
    List &list = sh.list;
    {
        const int groups = (s.vocab + kGroup - 1) / kGroup, last = groups - 1;
        const float *const maxima = s.maxima + (int64_t)row * s.slices * kGroups;
        const float low = logit_of(~lo), high = logit_of(~hi);
        static_assert(kMaxSlices * kGroups <= 32 * kPickThreads, "a bit per group of a thread");
        uint32_t reach = 0;  // this thread's groups, kPickThreads apart
#pragma unroll 8
        for (int i = 0; i < (groups + kPickThreads - 1) / kPickThreads; ++i) {
            const int g = tid + i * kPickThreads;
            reach |= (uint32_t)(maxima[min(g, last)] >= low && g < groups) << i;
        }
        // Several loads are on their way at once, with no branch around any: a group that is not
        // wanted takes the row's first, one that ends past the row the row's last sixteen.
        constexpr int kAhead = sizeof(T) == 2 ? 8 : 4;
        const int rounds = (groups + kPickThreads - 1) / kPickThreads;
        for (int i0 = 0; i0 < rounds; i0 += kAhead, reach >>= kAhead) {
            if (!__any(reach & ((1u << kAhead) - 1))) continue;
            Group<T> g[kAhead];
            const auto place = [&](int j) { return min((tid + (i0 + j) * kPickThreads) * kGroup, s.vocab - kGroup); };
#pragma unroll
            for (int j = 0; j < kAhead; ++j) g[j].load_whole(x + (reach >> j & 1 ? place(j) : 0));
            uint64_t found[kAhead / 4] = {};  // bits of four groups each
            int mine = 0;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (!__any(reach >> j & 1)) continue;
                uint32_t in = 0;  // (a NaN is in no range)
#pragma unroll
                for (int e = kGroup - 1; e >= 0; --e) {
                    const float l = g[j].value(e);
                    in = in + in + (uint32_t)(l == __builtin_amdgcn_fmed3f(l, low, high));
                }
                const int twice = ((tid + (i0 + j) * kPickThreads) * kGroup - place(j)) & (kGroup - 1);  // of the group before
                in = reach >> j & 1 ? in >> twice << twice : 0;
                found[j / 4] |= (uint64_t)in << (j % 4 * kGroup);
                mine += __popc(in);
            }
            const int upto = sum_upto(mine);
            int at = 0;
            if ((tid & 63) == 63 && upto) at = atomicAdd(&sh.n, upto);
            at = of_lane(at, 63) + upto - mine;
#pragma unroll
            for (int h = 0; h < kAhead / 4; ++h)
                for (; found[h]; found[h] &= found[h] - 1, ++at) {
                    const int bit = __builtin_ctzll(found[h]);
                    if (at < kListed) list.at[at] = place(4 * h + bit / kGroup) + bit % kGroup;
                }
        }
    }
    __syncthreads();
    const int n = sh.n;
    if (n > kListed) return false;
    for (int i = tid; i < n; i += kPickThreads) list.key[i] = order_key((float)x[list.at[i]]);
    // the cut's key: first by 2048ths of the bin, whose lowest and highest keys are what is open
    // then (of one value mostly); eleven bits of that at a time
    double before = above;
    uint64_t ties = 0;
    for (bool parts = true;; parts = false) {
        const int shift = max(0, 32 - __builtin_clz((hi - lo) | 1) - 11);
        const float end = top - (float)cut + 1.f;
        const auto digit_of = [&](uint32_t key) {
            if (!parts) return (int)((hi - key) >> shift);
            return (int)fminf(fmaxf(fmaf(-logit_of(~key), r.per, end) * kDigits, 0.f), (float)(kDigits - 1));
        };
        __syncthreads();
        for (int i = tid; i < kDigits; i += kPickThreads) sh.count[i] = 0, sh.sum[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kPickThreads) {
            const uint32_t key = list.key[i];
            if (key - lo > hi - lo) continue;
            const int digit = digit_of(key);
            atomicAdd(&sh.count[digit], 1u);
            atomicAdd((unsigned long long *)&sh.sum[digit],
                      (unsigned long long)weight(logit_of(~key), r.most, r.scale, sh.table));
        }
        __syncthreads();
        const uint64_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1], s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
        if (tid == 0) sh.found = -1;
        uint64_t total;
        double ahead = before + (double)(block_scan(s0 + s1, sh, turn, tid, total) - s0 - s1);
        // the last digit that something of stays: its first logit has less than the limit before
        // it (or none at all); where the sums' last bits let none stay, the first
        int mine = -1;
        if (c0 && (ahead < limit || ahead == 0.0)) mine = 2 * tid, atomicMax(&sh.found, mine);
        if (c1 && (ahead + (double)s0 < limit || ahead + (double)s0 == 0.0)) mine = 2 * tid + 1, atomicMax(&sh.found, mine);
        __syncthreads();
        const int found = sh.found;
        if (found < 0) return false;
        if (found >> 1 == tid) {
            sh.above = found & 1 ? ahead + (double)s0 : ahead;
            sh.found_count = found & 1 ? c1 : c0;
            sh.found_sum = found & 1 ? s1 : s0;
        }
        __syncthreads();
        before = sh.above;
        if (parts) {
            if (tid == 0) sh.edge[0] = ~0u, sh.edge[1] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kPickThreads) {
                const uint32_t key = list.key[i];
                if (digit_of(key) == found) atomicMin(&sh.edge[0], key), atomicMax(&sh.edge[1], key);
            }
            __syncthreads();
            lo = sh.edge[0], hi = sh.edge[1];
        } else {
            hi -= (uint32_t)found << shift;
            lo = max(lo, hi - ((1u << shift) - 1));
        }
        if (lo == hi || (!parts && shift <= kZeroBits<T>)) {
            // one value: equal logits, equal weights
            const uint64_t w = sh.found_sum / sh.found_count;
            ties = sh.found_count;
            if (w) ties = min(ties, before < limit ? (uint64_t)ceil(fmin((limit - before) / (double)w, 0x1p40)) : (uint64_t)0);
            ties = max(ties, (uint64_t)1);
            break;
        }
    }
    // what stays of it, slice by slice; of equal ones the first by their index
    if (tid < s.slices) sh.tied[tid] = 0, sh.count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPickThreads) {
        const uint32_t key = list.key[i];
        const int slice = list.at[i] / kSlice;
        if (key > hi)
            atomicAdd((unsigned long long *)&sh.tied[slice], (unsigned long long)weight(logit_of(~key), r.most, r.scale, sh.table));
        else if (key >= lo)
            atomicAdd(&sh.count[slice], 1u);
    }
    __syncthreads();
    const uint64_t equal = sh.found_sum / sh.found_count;
    if (tid < 64) {
        double upto = 0.0;
        uint32_t ranks = 0;
        for (int i0 = 0; i0 < s.slices; i0 += 64) {
            const bool in = i0 + tid < s.slices;
            const uint32_t c = in ? sh.count[i0 + tid] : 0;
            const uint32_t rank = sum_upto(c) + ranks - c;  // equal ones in the slices before
            const uint64_t stay = rank < ties ? min((uint64_t)c, ties - rank) : 0;
            double v = in ? sh.kept[i0 + tid] + (double)(sh.tied[i0 + tid] + stay * equal) : 0.0;
            ranks = of_lane(rank + c, 63);
            v = sum_upto(v);
            if (in) sh.kept[i0 + tid] = upto + v, sh.count[i0 + tid] = rank;
            upto += of_lane(v, 63);
        }
    }
    __syncthreads();
    // (a thread's logits are neighbours, and so are the threads: a scan counts the equal ones)
    pick_in_slice<T>(s, row, r, sh, turn, tid, sh.kept, [&](const float (&l)[kPerPick], int first, bool (&stays)[kPerPick]) {
        uint64_t c = 0, total;
#pragma unroll
        for (int e = 0; e < kPerPick; ++e) {
            const uint32_t key = order_key(l[e]);
            stays[e] = key > hi;
            c += key >= lo && key <= hi;
        }
        uint64_t rank = sh.count[first / kSlice] + block_scan(c, sh, turn, tid, total) - c;
#pragma unroll
        for (int e = 0; e < kPerPick; ++e) {
            const uint32_t key = order_key(l[e]);
            if (key >= lo && key <= hi) stays[e] = rank++ < ties;
        }
    });
    return true;
}

// Where the order (larger first, then lower index) is cut: everything above `key`
// stays, and the first `ties` of those that have it.
struct Cut {
    uint32_t key;
    uint64_t ties, sum;  // sum of the weights that stay
};

// The first `k` of the order, of those the ones with less than `limit` before them
// (and the first), over the whole row: the bin that holds the cut, then its key by
// eleven, eleven and ten bits.
template <typename T>
__device__ __forceinline__ Cut cut_row(const SampleParams &s, int row, const Row &r, PickShared &sh, int &turn, int tid,
                                       uint64_t k, uint64_t limit) {
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    uint64_t count = 0, sum = 0;  // before the part that is looked into
    int bin = 0;
    uint32_t prefix = 0;
    for (int round = 0; round < 4; ++round) {
        const int shift = round == 1 ? 21 : round == 2 ? 10 : 0;
        const uint32_t known = round <= 1 ? 0u : round == 2 ? ~0u << 21 : ~0u << 10;
        __syncthreads();
        for (int i = tid; i < kDigits; i += kPickThreads) sh.count[i] = 0, sh.sum[i] = 0;
        if (tid == 0) sh.found = -1;
        __syncthreads();
        constexpr int kAtOnce = 4;
        typedef T vec __attribute__((ext_vector_type(kAtOnce), aligned(sizeof(T))));
        for (int i0 = tid * kAtOnce; i0 < s.vocab; i0 += kPickThreads * kAtOnce) {
            vec v;
            if (i0 + kAtOnce <= s.vocab) {
                v = *reinterpret_cast<const vec *>(x + i0);
            } else {
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e) v[e] = i0 + e < s.vocab ? x[i0 + e] : (T)-INFINITY;
            }
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                if (i0 + e >= s.vocab) continue;
                const float y = (float)v[e], l = y == y ? y : -INFINITY;
                const int b = bin_of(l, r.top, r.per);
                const uint32_t key = order_key(l);
                int at;
                if (round == 0)
                    at = b;
                else if (b == bin && (key & known) == prefix)
                    at = (int)(~key >> shift & (round == 3 ? 1023u : 2047u));
                else
                    continue;
                atomicAdd(&sh.count[at], 1u);
                atomicAdd((unsigned long long *)&sh.sum[at], (unsigned long long)weight(l, r.most, r.scale, sh.table));
            }
        }
        __syncthreads();
        static_assert(kDigits == 2 * kPickThreads && kBins <= kDigits, "two places per thread");
        uint64_t total;
        const uint64_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1], s0 = sh.sum[2 * tid], s1 = sh.sum[2 * tid + 1];
        uint64_t cn = count + block_scan(c0 + c1, sh, turn, tid, total) - c0 - c1;
        uint64_t sn = sum + block_scan(s0 + s1, sh, turn, tid, total) - s0 - s1;
        // the first bin that the cut lies in or behind (found by one thread); none: the last
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint64_t c = e ? c1 : c0, w = e ? s1 : s0;
            const bool open = cn < k && (sn < limit || cn == 0), shut = cn + c >= k || sn + w >= limit;
            if (c && open && shut) sh.found = 2 * tid + e, sh.found_count = cn, sh.found_sum = sn;
            cn += c, sn += w;
        }
        __syncthreads();
        const int at = sh.found;
        if (at < 0) return {0, ~(uint64_t)0, sum + total};  // everything stays
        count = sh.found_count, sum = sh.found_sum;
        if (round == 0)
            bin = at;
        else
            prefix |= ~(uint32_t)at << shift & (round == 3 ? 1023u : 2047u << shift);
        if (round == 3) {
            const uint64_t have = sh.count[at], w = sh.sum[at] / have;  // equal logits, equal weights
            uint64_t ties = min(have, k - count);
            if (w) ties = min(ties, sum < limit ? (limit - sum - 1) / w + 1 : 0);
            if (count + ties == 0) ties = 1;
            return {prefix, ties, sum + ties * w};
        }
    }
    return {};
}

// The whole row.
template <typename T>
__device__ __forceinline__ void pick_from_row(const SampleParams &s, int row, const Row &r, PickShared &sh, int tid,
                                              double all) {
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    int turn = 0;
    const uint64_t none = ~(uint64_t)0;
    Cut cut{0, none, 0};
    double total = all;
    __syncthreads();
#pragma unroll 1
    for (int step = r.k ? 0 : 1; step < (r.p < 1.0 ? 2 : 1); ++step) {
        const double most = r.p * total;
        const uint64_t limit = step ? most > 0.0 ? (uint64_t)ceil(most) : 0 : none;
        cut = cut_row<T>(s, row, r, sh, turn, tid, r.k ? (uint64_t)r.k : none, limit);
        total = (double)cut.sum;
    }
    // weights that stay, slice by slice in the order of the indices; then the token's slice
    // again
    const double least = r.min_p * kOne;
    constexpr int kPer = kSlice / kPickThreads;
    auto slice_weights = [&](int slice, uint64_t &tied, float (&l)[kPer], uint64_t (&w)[kPer]) __attribute__((always_inline)) {
        const int first = slice * kSlice + tid * kPer;
        uint32_t same = 0;
        uint64_t sum = 0, total;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            float v = first + e < s.vocab ? (float)x[first + e] : -INFINITY;
            l[e] = v == v ? v : -INFINITY;
            const uint32_t key = order_key(l[e]);
            w[e] = 0;
            if (first + e < s.vocab && key >= cut.key) {
                w[e] = weight(l[e], r.most, r.scale, sh.table);
                w[e] = l[e] == r.most || (double)w[e] >= least ? w[e] : 0;
                same |= (uint32_t)(key == cut.key) << e;
            }
        }
        if (cut.ties != none) {
            const uint64_t c = __popc(same);
            uint64_t rank = tied + block_scan(c, sh, turn, tid, total) - c;
            tied += total;
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (same >> e & 1) w[e] = rank++ < cut.ties ? w[e] : 0;
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += w[e];
        return sum;
    };
    uint64_t tied = 0, upto = 0, sum;
    float l[kPer];
    uint64_t w[kPer];
    for (int i = 0; i < s.slices; ++i) {
        uint64_t part;
        if (tid == 0) sh.kept[i] = (double)tied;
        block_scan(slice_weights(i, tied, l, w), sh, turn, tid, part);
        upto += part;
        if (tid == 0) sh.tied[i] = upto;
    }
    __syncthreads();
    const uint64_t target = target_of(r.u, upto);
    int slice = 0;
    while (sh.tied[slice] <= target) ++slice;  // (ends: target < the last)
    const uint64_t start = slice ? sh.tied[slice - 1] : 0;
    tied = (uint64_t)sh.kept[slice];
    sum = slice_weights(slice, tied, l, w);
    uint64_t part;
    uint64_t before = start + block_scan(sum, sh, turn, tid, part) - sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (before <= target && target < before + w[e]) answer(s, row, slice * kSlice + tid * kPer + e, l[e], r, (double)upto);
        before += w[e];
    }
}

template <typename T>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleParams s) {
    __shared__ PickShared sh;
    __shared__ float row_most;
    __shared__ int row_at;
    const int tid = threadIdx.x, row = blockIdx.x;
    const Settings set = settings(s, row);
    const double scale = weight_scale(set.temperature);
    fill_table(sh.table, tid);
    // the row's largest, and the running sums of its slices relative to that
    if (tid < 64) {
        const Slice *const sl = s.slice + (int64_t)row * s.slices;
        float most = -INFINITY;
        int at = INT_MAX;
        for (int i = tid; i < s.slices; i += 64) {
            const float m = sl[i].most;
            if (m > most) most = m, at = sl[i].at;
        }
        const float highest = over_wave(most, larger);
        at = over_wave(most == highest ? at : INT_MAX, smaller);
        most = highest;
        if (tid == 0) row_most = most, row_at = at;
        if (set.all()) {
            double before = 0.0;
            for (int i0 = 0; i0 < s.slices; i0 += 64) {
                double w = 0.0;
                if (i0 + tid < s.slices) w = (double)sl[i0 + tid].sum * relative(sl[i0 + tid].most, most, scale);
                w = sum_upto(w);
                if (i0 + tid < s.slices) sh.slice_sums[i0 + tid] = before + w;
                before += of_lane(w, 63);
            }
        }
    }
    __syncthreads();
    const float most = row_most;
    if (!(most > -INFINITY) || set.greedy()) {
        if (tid == 0) {
            const bool any = most > -INFINITY;
            s.tokens[row] = any ? row_at : -1;
            if (s.logprobs) s.logprobs[row] = any ? 0.f : NAN;
        }
        return;
    }
    const float per = set.per();
    const Row r{most, grid_of(most, per), per, scale, set.k, set.p, set.min_p, (double)s.u[row]};
    const double all = set.all() ? sh.slice_sums[s.slices - 1] : 0.0;
    if (!r.k && !(r.p < 1.0) && !(r.min_p > 0.0)) {
        int turn = 0;
        pick_in_slice<T>(s, row, r, sh, turn, tid, sh.slice_sums, [](const float (&)[kPerPick], int, bool (&b)[kPerPick]) {
#pragma unroll
            for (int e = 0; e < kPerPick; ++e) b[e] = true;
        });
        return;
    }
    if (set.bins(s.slices)) {
        if (pick_by_bins<T>(s, row, r, sh, tid, all)) return;
        __syncthreads();
    }
    if (pick_from_few<T>(s, row, r, sh, tid, all)) return;
    pick_from_row<T>(s, row, r, sh, tid, all);
}

int64_t slices_of(int64_t vocab) { return (vocab + kSlice - 1) / kSlice; }

}  // namespace

int64_t sample_max_vocab() { return (int64_t)kMaxSlices * kSlice; }
int64_t sample_blocks(const SampleDesc &d) { return d.rows * slices_of(d.vocab); }
size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    const int64_t slices = slices_of(vocab);
    return (size_t)(rows * slices) * (kGroups * sizeof(float) + sizeof(Slice) + (slices > 1 ? kStored * sizeof(uint64_t) : 0));
}

int launch_sample(const SampleDesc &d, void *workspace, hipStream_t st) {
    SampleParams s{};
    s.logits = static_cast<const char *>(d.logits);
    s.ld = d.ld;
    s.vocab = (int)d.vocab;
    s.slices = (int)slices_of(d.vocab);
    s.u = d.u;
    s.set = d.set;
    s.slice = static_cast<Slice *>(workspace);
    s.maxima = reinterpret_cast<float *>(s.slice + d.rows * s.slices);
    s.bins = reinterpret_cast<uint64_t *>(s.maxima + d.rows * s.slices * kGroups);
    s.tokens = d.tokens;
    s.logprobs = d.logprobs;
    auto go = [&](auto t) -> int {
        using T = decltype(t);
        hipLaunchKernelGGL(sample_slices_kernel<T>, dim3((unsigned)sample_blocks(d)), dim3(kGroups), 0, st, s);
        GFH_TRY(check_launch("sample"));
        hipLaunchKernelGGL(sample_pick_kernel<T>, dim3((unsigned)d.rows), dim3(kPickThreads), 0, st, s);
        return check_launch("sample (pick)");
    };
    if (d.dtype == GFH_F32) return go(float{});
    return d.dtype == GFH_BF16 ? go(__bf16{}) : go(_Float16{});
}

}  // namespace gfh
