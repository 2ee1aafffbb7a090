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
// the same in any order, and a border between two tokens lies within 2^-35 of its
// place whatever the vocabulary, so no u meets another token than in a longer format
// but for one in 10^10.  An exponential is a table of 2^(j / 32), a polynomial of five
// terms beyond (2e-15) and the exponent: some 20 operations, two thirds of them fp64,
// which this card issues at the rate of fp32.
//
// Two launches.  The first (a workgroup per 4096 logits, read once) leaves the largest of
// every 16, of its 4096 and where it is, and the sum of their weights where the row's
// settings need one.  The second has a workgroup per row, which rarely reads the row
// again: the k-th largest of the 16s' maxima bounds the k-th largest logit from below,
// so a few groups hold all candidates; those are sorted.  With no filter the sums find
// the 4096 that hold the token.  A row whose filter keeps more than kCandidates (a
// flat one under top-p) is searched whole: bins, then radix.
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace gfh {
namespace {

constexpr int kGroup = 16, kSlice = 4096, kGroups = kSlice / kGroup;  // logits; groups of a slice
constexpr int kMaxSlices = 128;
constexpr int kBins = 2048, kCandidates = 2048, kGuess = 1024, kPickThreads = 1024;
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
};
__device__ __forceinline__ Settings settings(const SampleParams &s, int row) {
    Settings r;
    r.temperature = s.set.temperatures ? s.set.temperatures[row] : s.set.temperature;
    r.k = s.set.top_ks ? s.set.top_ks[row] : s.set.top_k;
    if (r.k < 0 || r.k >= s.vocab) r.k = 0;
    r.p = s.set.top_ps ? s.set.top_ps[row] : s.set.top_p;
    if (!(r.p < 1.0)) r.p = 1.0;
    r.min_p = s.set.min_ps ? s.set.min_ps[row] : s.set.min_p;
    if (!(r.min_p > 0.0)) r.min_p = 0.0;
    return r;
}

// exp((l - most) / T) 2^44, rounded; scale = 32 log2 e / T, table[j] = 2^(j / 32).
__device__ __forceinline__ uint64_t weight(float l, float most, double scale, const double *table) {
    if (l == most) return (uint64_t)1 << 44;  // (infinite ones too)
    const double y = ((double)l - (double)most) * scale;
    if (!(y > -32.0 * 46)) return 0;  // NaN and -inf too
    const double t = y + 0x1.8p52;
    const int n = (int)(uint32_t)__double_as_longlong(t);
    const double r = (y - (t - 0x1.8p52)) * 0x1.62e42fefa39efp-6;  // ln 2 / 32
    double e = fma(r, 1.0 / 120, 1.0 / 24);
    e = fma(r, e, 1.0 / 6);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    // 2^(n / 32 + 44), then the integer in the low bits of 2^52 + it
    const double f = __longlong_as_double(__double_as_longlong(table[n & 31]) + ((int64_t)((n >> 5) + 44) << 52));
    return (uint64_t)__double_as_longlong(fma(e, f, 0x1p52)) & 0xfffffffffffffull;
}
__device__ __forceinline__ void fill_table(double *table, int tid) {
    if (tid < 32) table[tid] = exp2(tid / 32.0);
}
__device__ __forceinline__ double weight_scale(float temperature) { return 32.0 * 1.4426950408889634 / (double)temperature; }

// The logits of a group: -inf for NaN and from `end` on.
template <typename T>
__device__ __forceinline__ void load_group(const T *row, int first, int end, float (&x)[kGroup]) {
    constexpr int E = 16 / sizeof(T);
    // (rows begin anywhere that their type allows)
    typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    if (first + kGroup <= end) {
#pragma unroll
        for (int i = 0; i < kGroup / E; ++i) {
            const vec v = *reinterpret_cast<const vec *>(row + first + i * E);
#pragma unroll
            for (int e = 0; e < E; ++e) x[i * E + e] = (float)v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) x[e] = first + e < end ? (float)row[first + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kGroup; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
}

template <typename T>
__global__ __launch_bounds__(kGroups) void sample_slices_kernel(SampleParams s) {
    __shared__ double table[32];
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
    float most = x[0];
#pragma unroll
    for (int e = 1; e < kGroup; ++e) most = fmaxf(most, x[e]);
    s.maxima[((int64_t)row * s.slices + slice) * kGroups + tid] = most;
    int at = INT_MAX;
#pragma unroll
    for (int e = kGroup - 1; e >= 0; --e) at = x[e] == most ? first + e : at;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(most, o);
        const int a2 = __shfl_xor(at, o);
        if (m2 > most || (m2 == most && a2 < at)) most = m2, at = a2;
    }
    if (lane == 0) mosts[wave] = most, ats[wave] = at;
    __syncthreads();
    most = mosts[0], at = ats[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (mosts[w] > most) most = mosts[w], at = ats[w];
    uint64_t sum = 0;
    if (set.all()) {
        const double scale = weight_scale(set.temperature);
        if (most > -INFINITY) {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) sum += weight(x[e], most, scale, table);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor((unsigned long long)sum, o);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = sums[0] + sums[1] + sums[2] + sums[3];
    }
    if (tid == 0) s.slice[(int64_t)row * s.slices + slice] = {most, at, sum};
}

// ---- the second launch ------------------------------------------------------------

struct PickShared {
    double table[32];
    uint64_t wave_sums[2][kPickThreads / 64];
    double slice_sums[kMaxSlices];
    uint64_t chunk_sums[kMaxSlices];
    uint32_t count[kBins];
    uint64_t sum[kBins];
    uint64_t key[kCandidates];
    uint64_t weight[kCandidates];
    int index[kCandidates];
    int hot[kCandidates];
    int found;
    uint64_t found_count, found_sum;
};

// Inclusive sum over the workgroup's threads, and the total; call after call takes
// the other half of wave_sums, so one barrier does.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, PickShared &sh, int &turn, int tid, uint64_t &total) {
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, o);
        x += lane >= o ? y : 0;
    }
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

// The bin of a logit: a 64th of z below the largest; not rising with l.
__device__ __forceinline__ int bin_of(float l, float most, float per) {
    if (l == most) return 0;
    return (int)fminf((most - l) * per, (float)(kBins - 1));  // (NaN: the last)
}
// Larger logits have larger keys; all that cannot be drawn the lowest.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t u = __float_as_uint(l == 0.f ? 0.f : l);
    return u >> 31 ? ~u : u | 0x80000000u;
}

struct Row {
    float most, per;  // largest logit; bins to a unit of it
    double scale;
    int k;
    double p, min_p;
    double u;
};

// The logarithm of a token's probability among those of weight `total`.
__device__ __forceinline__ void answer(const SampleParams &s, int row, int token, float l, const Row &r, double total) {
    s.tokens[row] = token;
    if (!s.logprobs) return;
    const double z = l == r.most ? 0.0 : ((double)l - (double)r.most) * (r.scale * (1.0 / (32.0 * 1.4426950408889634)));
    s.logprobs[row] = (float)(z - log(total / kOne));
}
// floor(u total), below total.
__device__ __forceinline__ uint64_t target_of(double u, uint64_t total) {
    const double t = fmin(fmax(u, 0.0), 1.0) * (double)total;
    const uint64_t n = (uint64_t)t;
    return n < total ? n : total - 1;
}

// No filter: the slice by the sums, then the token in it.
template <typename T>
__device__ __forceinline__ void pick_from_all(const SampleParams &s, int row, const Row &r, PickShared &sh, int tid,
                                              double total) {
    // sh.slice_sums: running sums
    if (tid < 64) {
        const double target = fmin(fmax(r.u, 0.0), 1.0) * total;
        int n = 0, last = -1;
        for (int i = tid; i < s.slices; i += 64) {
            const double before = i ? sh.slice_sums[i - 1] : 0.0;
            n += sh.slice_sums[i] <= target;
            last = sh.slice_sums[i] > before ? i : last;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o), last = max(last, __shfl_xor(last, o));
        if (tid == 0) sh.found = min(n, last);
    }
    __syncthreads();
    const int slice = sh.found;
    const double target = fmin(fmax(r.u, 0.0), 1.0) * total - (slice ? sh.slice_sums[slice - 1] : 0.0);
    const T *const x = reinterpret_cast<const T *>(s.logits) + row * s.ld;
    constexpr int kPer = kSlice / kPickThreads;
    const int first = slice * kSlice + tid * kPer;
    float l[kPer];
    uint64_t w[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        l[e] = first + e < s.vocab ? (float)x[first + e] : -INFINITY;
        w[e] = weight(l[e], r.most, r.scale, sh.table);
        sum += w[e];
    }
    int turn = 0;
    uint64_t all;
    uint64_t upto = block_scan(sum, sh, turn, tid, all);
    // (weights so small that all are 0 here: the slice's largest)
    const Slice sl = s.slice[(int64_t)row * s.slices + slice];
    if (all == 0) {
        if (tid == 0) answer(s, row, sl.at, sl.most, r, total);
        return;
    }
    uint64_t n = target > 0.0 ? (uint64_t)target : 0;
    n = n < all ? n : all - 1;
    upto -= sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (upto <= n && n < upto + w[e]) answer(s, row, first + e, l[e], r, total);
        upto += w[e];
    }
}

// Candidates, if they are few enough: the logits in bins up to the one that holds
// the k-th largest maximum of a group (top-k), of a quarter of the groups or the
// kGuess-th (top-p, which may need more), or min_p.  False: not enough, or too many.
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
    if (!r.k && r.min_p > 0.0) {
        const double b = -log(r.min_p) * 64.0 + 2.0;  // (2: the bins' own rounding)
        last = (int)fmin(fmax(b, 0.0), (double)(kBins - 1));
    }
    if (r.k || r.p < 1.0) {
        const int want = r.k ? r.k : min(kGuess, groups / 4 + 1);
        if (want > kCandidates) return false;
        for (int i = tid; i < kBins; i += kPickThreads) sh.count[i] = 0;
        __syncthreads();
        for (int i = tid; i < groups; i += kPickThreads) atomicAdd(&sh.count[bin_of(maxima[i], r.most, r.per)], 1u);
        if (tid == 0) sh.found = kBins - 1;
        __syncthreads();
        const uint32_t a = sh.count[2 * tid], b = sh.count[2 * tid + 1];
        const uint64_t upto = block_scan(a + b, sh, turn, tid, total);
        const int before = (int)(upto - a - b);
        if (before < want && before + (int)a >= want) sh.found = 2 * tid;
        if (before + (int)a < want && (int)upto >= want) sh.found = 2 * tid + 1;
        __syncthreads();
        guess = !r.k && sh.found < last;
        last = min(last, sh.found);
    }
    // the groups that have candidates, in their order
    const int per = (groups + kPickThreads - 1) / kPickThreads;
    uint64_t mine = 0;
    for (int i = tid * per; i < min(groups, (tid + 1) * per); ++i) mine += bin_of(maxima[i], r.most, r.per) <= last;
    uint64_t at = block_scan(mine, sh, turn, tid, total) - mine;
    if (total > kCandidates) return false;
    const int hot = (int)total;
    for (int i = tid * per; mine && i < min(groups, (tid + 1) * per); ++i)
        if (bin_of(maxima[i], r.most, r.per) <= last) sh.hot[at++] = i;
    __syncthreads();
    // the candidates, in their order
    int n = 0;
    for (int h0 = 0; h0 < hot; h0 += kPickThreads) {
        float l[kGroup];
        int first = 0;
        uint32_t in = 0;
        if (h0 + tid < hot) {
            first = sh.hot[h0 + tid] * kGroup;
            load_group(x, first, s.vocab, l);
#pragma unroll
            for (int e = 0; e < kGroup; ++e) in |= (uint32_t)(bin_of(l[e], r.most, r.per) <= last && first + e < s.vocab) << e;
        }
        const uint64_t c = __popc(in);
        at = n + block_scan(c, sh, turn, tid, total) - c;
        n += (int)total;
        if (n > kCandidates) return false;
#pragma unroll
        for (int e = 0; e < kGroup; ++e)
            if (in >> e & 1) {
                sh.key[at] = (uint64_t)~order_key(l[e]) << 32 | (uint32_t)at;
                sh.index[at] = first + e;
                sh.weight[at] = weight(l[e], r.most, r.scale, sh.table);
                ++at;
            }
    }
    // sorted: larger logits first, equal ones as they came
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kPickThreads) sh.key[i] = ~(uint64_t)0;
    for (int b = 2; b <= size; b <<= 1)
        for (int d = b >> 1; d > 0; d >>= 1) {
            __syncthreads();
            const int i = (tid & ~(d - 1)) * 2 + (tid & (d - 1));
            if (i + d < size) {
                const uint64_t p = sh.key[i], q = sh.key[i + d];
                if ((p > q) == !(i & b)) sh.key[i] = q, sh.key[i + d] = p;
            }
        }
    __syncthreads();
    // how many stay
    static_assert(kCandidates == 2 * kPickThreads, "two places per thread");
    int pos[2];
    uint64_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int j = 2 * tid + e;
        pos[e] = j < n ? (int)(uint32_t)sh.key[j] : 0;
        w[e] = j < n ? sh.weight[pos[e]] : 0;
    }
    uint64_t limit = ~(uint64_t)0;
    const int k = r.k ? min(r.k, n) : n;
    uint64_t upto = block_scan((2 * tid < k ? w[0] : 0) + (2 * tid + 1 < k ? w[1] : 0), sh, turn, tid, total);
    if (r.p < 1.0) {
        const double most = r.p * (r.k ? (double)total : all);
        limit = most > 0.0 ? (uint64_t)ceil(most) : 0;
        if (guess && total < limit) return false;  // the next ones would stay too
    }
    // (a thread's sum without the places from k on, which do not stay anyway)
    uint64_t before = upto - (2 * tid < k ? w[0] : 0) - (2 * tid + 1 < k ? w[1] : 0);
    const double least = r.min_p * kOne;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int j = 2 * tid + e;
        const bool stays = j == 0 || (j < k && before < limit && (double)w[e] >= least);
        if (j < n && !stays) sh.weight[pos[e]] = 0;
        before += w[e];
    }
    __syncthreads();
    w[0] = 2 * tid < n ? sh.weight[2 * tid] : 0;
    w[1] = 2 * tid + 1 < n ? sh.weight[2 * tid + 1] : 0;
    upto = block_scan(w[0] + w[1], sh, turn, tid, total);
    const uint64_t target = target_of(r.u, total);
    before = upto - w[0] - w[1];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if (before <= target && target < before + w[e]) {
            const int i = sh.index[2 * tid + e];
            answer(s, row, i, (float)x[i], r, (double)total);
        }
        before += w[e];
    }
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
        for (int i = tid; i < kBins; i += kPickThreads) sh.count[i] = 0, sh.sum[i] = 0;
        if (tid == 0) sh.found = -1;
        __syncthreads();
        for (int i0 = tid * kGroup; i0 < s.vocab; i0 += kPickThreads * kGroup) {
            float l[kGroup];
            load_group(x, i0, s.vocab, l);
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
                if (i0 + e >= s.vocab) continue;
                const int b = bin_of(l[e], r.most, r.per);
                const uint32_t key = order_key(l[e]);
                int at;
                if (round == 0)
                    at = b;
                else if (b == bin && (key & known) == prefix)
                    at = (int)(~key >> shift & (round == 3 ? 1023u : 2047u));
                else
                    continue;
                atomicAdd(&sh.count[at], 1u);
                atomicAdd((unsigned long long *)&sh.sum[at], (unsigned long long)weight(l[e], r.most, r.scale, sh.table));
            }
        }
        __syncthreads();
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
    if (r.k) {
        cut = cut_row<T>(s, row, r, sh, turn, tid, (uint64_t)r.k, none);
        total = (double)cut.sum;
    }
    if (r.p < 1.0) {
        const double most = r.p * total;
        cut = cut_row<T>(s, row, r, sh, turn, tid, r.k ? (uint64_t)r.k : none, most > 0.0 ? (uint64_t)ceil(most) : 0);
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
        if (tid == 0) sh.key[i] = tied;
        block_scan(slice_weights(i, tied, l, w), sh, turn, tid, part);
        upto += part;
        if (tid == 0) sh.chunk_sums[i] = upto;
    }
    __syncthreads();
    const uint64_t target = target_of(r.u, upto);
    int slice = 0;
    while (sh.chunk_sums[slice] <= target) ++slice;  // (ends: target < the last)
    const uint64_t start = slice ? sh.chunk_sums[slice - 1] : 0;
    tied = sh.key[slice];
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
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float m2 = __shfl_xor(most, o);
            const int a2 = __shfl_xor(at, o);
            if (m2 > most || (m2 == most && a2 < at)) most = m2, at = a2;
        }
        if (tid == 0) row_most = most, row_at = at;
        if (set.all()) {
            double before = 0.0;
            for (int i0 = 0; i0 < s.slices; i0 += 64) {
                double w = 0.0;
                if (i0 + tid < s.slices) {
                    const Slice x = sl[i0 + tid];
                    w = x.most == most ? (double)x.sum
                                       : (double)x.sum * exp2(((double)x.most - (double)most) * scale * (1.0 / 32));
                    w = x.most == most || (most < INFINITY && x.most > -INFINITY) ? w : 0.0;
                }
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const double y = __shfl_up(w, o);
                    w += tid >= o ? y : 0.0;
                }
                if (i0 + tid < s.slices) sh.slice_sums[i0 + tid] = before + w;
                before += __shfl(w, 63);
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
    const Row r{most, 64.f / set.temperature, scale, set.k, set.p, set.min_p, (double)s.u[row]};
    const double all = set.all() ? sh.slice_sums[s.slices - 1] : 0.0;
    if (!r.k && !(r.p < 1.0) && !(r.min_p > 0.0))
        pick_from_all<T>(s, row, r, sh, tid, all);
    else if (!pick_from_few<T>(s, row, r, sh, tid, all))
        pick_from_row<T>(s, row, r, sh, tid, all);
}

int64_t slices_of(int64_t vocab) { return (vocab + kSlice - 1) / kSlice; }

}  // namespace

int64_t sample_max_vocab() { return (int64_t)kMaxSlices * kSlice; }
int64_t sample_blocks(const SampleDesc &d) { return d.rows * slices_of(d.vocab); }
size_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    return (size_t)(rows * slices_of(vocab)) * (kGroups * sizeof(float) + sizeof(Slice));
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
