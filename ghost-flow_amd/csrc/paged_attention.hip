// paged_attention.hip -- attention of a ragged batch's new tokens (one each,
// or chunks of a prompt) over a key/value cache in pages (paged_kv.hpp).
//
//   S = scale q . k,  P = softmax over the keys the token sees,  O = P V
//
// A token at position p sees key j of its sequence when j < kv_len, j <= p if
// causal, j > p - window if there is a window; a token that sees none gets 0.
// The G = heads / kv_heads query heads of a key/value head read the same keys,
// so the rows of a product are (token, head of the group) pairs: row R = token
// * G + g, and a tile is BM consecutive rows of one sequence and key/value
// head.  Tiles lie at multiples of BM rows of the whole batch: tile j of
// sequence s has the number j + s, which no other tile has (a sequence starts
// in the tile row where the one before ends, or later), so a workgroup finds
// its sequence with one search for the largest s with offset(s) G / BM + s <=
// number, and the host needs no length.
//
// Softmax online in base 2, statistics and sums in fp32: the running maximum
// is of the raw dot products, a probability is exp2(s c - m c + bias) with c =
// |scale| log2 e (the sign of the scale is on q).  fp32 q: P is carried as three bf16
// pieces, or in fp32.  q of 16 bits: as two pieces of its type in tiles of 16 rows,
// whose matrix units wait for bytes anyway (64 sequences of up to 4096 keys 134.2 us
// with one, 136.3 with two; then O has its own rounding alone), and rounded to the type
// in tiles of 128 rows, where a second piece would be half as many products more: O is
// then off by up to half a step of the type relative to P |V| as well (against 64 bits, root
// mean square of normal inputs: bf16 2.3e-3 where O's rounding alone has 1.7e-3).
// There l sums the rounded P, so the weights that V is taken with add up to one.  The
// bias (14 or 9 for f16, 16 for three pieces) keeps small probabilities normal in
// their 16-bit form and cancels in O / l.  Long axes are split over workgroups; a
// second kernel joins the parts in their order, so results do not depend on timing.
//
// Rows of the cache past the last key and pages outside the cache read as
// zeros.  A masked key must not reach a row even when its value is not
// finite (0 * inf): a tile that holds keys which some of its rows do not see
// is searched for such values, and its workgroup then redoes its rows one by
// one over the keys they see (slow_rows).  So it does where a sum of its own is not
// finite: an infinite V meets pieces of P of either sign and weights that 16 bits
// round to nothing, and V near the largest fp32 weights above 1.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "paged_types.hpp"
#include "split_bf16.hpp"

namespace gfh {
namespace {

using paged::View;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;
typedef __attribute__((address_space(1))) void *glb_ptr_t;

struct AttnParams {
    View c;
    const char *q;
    char *out;
    int64_t ldq, ldo;  // elements between tokens
    float sc2;         // |scale| log2 e
    bool negate;       // scale < 0
    bool causal;
    int window;  // 0: none
    int ntiles, nsplit, chunk;
    int min_rows, max_rows;  // sequences this launch takes: rows = tokens * group
    bool direct;             // see find_rows
    float *acc;   // [row][nsplit][d] parts, where nsplit > 1 (see part_row)
    float2 *ml;   // [row][nsplit] their maximum (scaled) and sum
};

// A workgroup's rows [r0, r1) and the keys [lo, hi) that any of them sees.
struct Rows {
    int r0, r1, base;   // base: the tile's first row, r0 >= base
    int q_last;         // position of the sequence's token t is t + q_last
    int kv_len;
    int lo, hi;
    int part;           // row r has its parts at (r + part) * kv_heads + kvh
};

// Where no sequence of a few-row launch has more than kFewRows rows (p.direct), a
// sequence has at most kFewTiles tiles and the grid counts those; else it counts
// tile numbers.  Parts are laid out for as many rows.  (16 sequences of 24 rows over
// 2000 keys, bf16: 57 us in 128-row tiles, 94 in 16-row ones; of 16 rows 44 and 58 there,
// but 4 of them 31 and 22, and chunks of prompts in one batch with single tokens would
// put those into 128-row tiles.)
constexpr int kFewRows = 16, kFewTiles = 2;

// Tile `number` of sequence s, whose tokens are [o0, o1) and length kv_len.
__device__ __forceinline__ bool rows_at(const AttnParams &p, int number, int s, int bm, int o0, int o1, int kv_len,
                                        Rows &t) {
    const View &c = p.c;
    o1 = max(o0, o1);
    t.base = (number - s) * bm;
    t.r0 = max(o0 * c.group, t.base);
    t.r1 = min(o1 * c.group, t.base + bm);
    const int rows = (o1 - o0) * c.group;
    if (t.r0 >= t.r1 || rows < p.min_rows || rows > p.max_rows) return false;
    t.part = p.direct ? s * kFewRows - o0 * c.group : 0;
    t.kv_len = kv_len;
    t.q_last = t.kv_len - o1;
    if (t.q_last + o0 < 0) paged::raise(c, paged::kBadLength);  // tokens before position 0
    const int first = t.r0 / c.group + t.q_last, last = (t.r1 - 1) / c.group + t.q_last;
    t.hi = max(0, p.causal ? min(t.kv_len, last + 1) : t.kv_len);
    t.lo = p.window ? min(t.hi, max(0, first - p.window + 1)) : 0;
    return true;
}
__device__ __forceinline__ bool rows_of(const AttnParams &p, int number, int s, int bm, Rows &t) {
    return rows_at(p, number, s, bm, paged::offset_at(p.c, s), paged::offset_at(p.c, s + 1), paged::length_at(p.c, s), t);
}
// The tile of a workgroup and its sequence.
__device__ __forceinline__ bool find_rows(const AttnParams &p, int number, int bm, int lane, Rows &t, int &s) {
    const View &c = p.c;
    if (p.direct) {
        s = number / kFewTiles;
        return rows_of(p, paged::offset_at(c, s) * c.group / bm + s + number % kFewTiles, s, bm, t);
    }
    if (c.num_seqs < 64) {  // everything about the batch in one round of loads
        const int off = paged::offset_at(c, min(lane, c.num_seqs));
        const int len = paged::length_at(c, min(lane, c.num_seqs - 1));
        const bool ok = lane < c.num_seqs && (int)((unsigned)(off * c.group) / (unsigned)bm) + lane <= number;
        s = __popcll(__ballot(ok)) - 1;
        if (s < 0) return false;
        return rows_at(p, number, s, bm, __builtin_amdgcn_readlane(off, s), __builtin_amdgcn_readlane(off, s + 1),
                       __builtin_amdgcn_readlane(len, s), t);
    }
    const int n = paged::wave_leading(c.num_seqs, lane, [&](int i) {
        return (int)((unsigned)(paged::offset_at(c, i) * c.group) / (unsigned)bm) + i <= number;
    });
    s = n - 1;
    return n > 0 && rows_of(p, number, s, bm, t);
}
// The splits that have keys (at least one, which writes rows without any).
__device__ __forceinline__ int active_splits(const AttnParams &p, const Rows &t) {
    return max(1, min(p.nsplit, (t.hi - t.lo + p.chunk - 1) / p.chunk));
}

// The keys [jmin, jmax] that row r of the batch sees.
__device__ __forceinline__ void row_keys(const AttnParams &p, const Rows &t, int r, int &jmin, int &jmax) {
    const bool ok = r >= t.r0 && r < t.r1;
    const int pos = r / p.c.group + t.q_last;
    jmax = !ok ? -1 : p.causal ? min(pos, t.kv_len - 1) : t.kv_len - 1;
    jmin = ok && p.window ? pos - p.window + 1 : 0;
}

template <typename T>
__device__ __forceinline__ const T *q_row(const AttnParams &p, int r, int kvh) {
    const int tok = r / p.c.group, g = r - tok * p.c.group;
    return reinterpret_cast<const T *>(p.q) + tok * p.ldq + (int64_t)(kvh * p.c.group + g) * p.c.d;
}
template <typename T>
__device__ __forceinline__ T *out_row(const AttnParams &p, int r, int kvh) {
    const int tok = r / p.c.group, g = r - tok * p.c.group;
    return reinterpret_cast<T *>(p.out) + tok * p.ldo + (int64_t)(kvh * p.c.group + g) * p.c.d;
}
__device__ __forceinline__ int64_t part_row(const AttnParams &p, const Rows &t, int r, int kvh) {
    return (int64_t)(r + t.part) * p.c.hkv + kvh;
}

// The rows of a tile one by one, a wave each, over the keys [b, e) that each
// sees, in fp32 and without a bias: for the inputs named above.  (Other parts of a
// row are 2^bias larger: the maximum says so.)  64 keys at a time: lane j the score of
// key j, then lanes l and l + 64 of V, eight keys' loads on their way at once (a row of
// 16384 keys of 128, bf16: 2.7 ms, with the keys one by one 19).
template <typename TA, typename TC>
__device__ __forceinline__ void slow_rows(const AttnParams &p, const Rows &t, int seq, int kvh, int b, int e,
                                                    int split, bool parts, float bias, int wave, int nwaves,
                                                    int lane) {
    const View &c = p.c;
    const int d0 = lane < c.d ? lane : 0, d1 = lane + 64 < c.d ? lane + 64 : 0;
    for (int r = t.r0 + wave; r < t.r1; r += nwaves) {
        int jmin, jmax;
        row_keys(p, t, r, jmin, jmax);
        const TA *q = q_row<TA>(p, r, kvh);
        const int last = min(e, jmax + 1);
        float acc[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
        for (int j0 = max(b, jmin); j0 < last; j0 += 64) {
            const int j = j0 + lane;
            const bool in = j < last;
            const int pg = in ? paged::page_of(c, j) : 0, page = in ? c.table[seq * c.table_stride + pg] : -1;
            const bool ok = page >= 0 && page < c.num_pages;
            int64_t at = ok ? page * c.page_stride + (int64_t)(j - pg * c.page_size) * c.row_stride + kvh * c.head_stride
                            : 0;
            float s = 0.f;
#pragma unroll 4
            for (int dim = 0; dim < c.d; dim += 8) {
                float qv[8], kv[8];
                load_vec<8>(q + dim, qv);
#pragma unroll
                for (int i = 0; i < 8; ++i) kv[i] = 0.f;  // a page outside the cache
                if (ok) load_vec<8>(reinterpret_cast<const TC *>(c.k) + at + dim, kv);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(p.negate ? -qv[i] : qv[i], kv[i], s);
            }
            s = in ? s * p.sc2 : -INFINITY;
            float m_new = max_nan(m, s);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m_new = max_nan(m_new, __shfl_xor(m_new, o));
            if (m_new == -INFINITY) continue;
            if (m_new != m_new) {  // so is the row
                m = l = acc[0] = acc[1] = m_new;
                break;
            }
            const float alpha = exp2f(m - m_new), w = in ? exp2f(s - m_new) : 0.f;
            l = fmaf(l, alpha, wave_sum(w));
            acc[0] *= alpha, acc[1] *= alpha;
            m = m_new;
            const uint64_t good = __ballot(ok);
            if (!good) continue;
            // (keys without a row load another's, and take nothing of it)
            const int any = __builtin_ctzll(good);
            const int64_t other = (int64_t)__builtin_amdgcn_readlane((int)(at >> 32), any) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane((int)at, any);
            at = ok ? at : other;
            for (int k0 = 0; k0 < min(64, last - j0); k0 += 8) {
                float v0[8], v1[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t row = (int64_t)__builtin_amdgcn_readlane((int)(at >> 32), k0 + i) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)at, k0 + i);
                    const TC *v = reinterpret_cast<const TC *>(c.v) + row;
                    v0[i] = (float)v[d0], v1[i] = (float)v[d1];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool has = good >> (k0 + i) & 1;
                    const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k0 + i));
                    acc[0] = fmaf(wi, has ? v0[i] : 0.f, acc[0]);
                    acc[1] = fmaf(wi, has ? v1[i] : 0.f, acc[1]);
                }
            }
            if (__all((lane >= c.d || acc[0] != acc[0]) && (lane + 64 >= c.d || acc[1] != acc[1]))) break;
        }
        if (parts) {
            const int64_t at = part_row(p, t, r, kvh) * p.nsplit + split;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lane + 64 * i < c.d) p.acc[at * c.d + lane + 64 * i] = acc[i];
            if (lane == 0) p.ml[at] = make_float2(m + bias, l);
        } else {
            const float inv = m == -INFINITY ? 0.f : 1.0f / l;
            TA *o = out_row<TA>(p, r, kvh);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lane + 64 * i < c.d) o[lane + 64 * i] = (TA)(acc[i] * inv);
        }
    }
}

// ---- 16-bit types ---------------------------------------------------------------

template <typename T>
struct Half;
template <>
struct Half<__bf16> {
    typedef bf16x2 v2;
    typedef bf16x4 v4;
    typedef bf16x8 v8;
    static constexpr uint32_t kExp = 0x7f80u;
    static constexpr float kBias = 0.f;
    // c + both halves of w
    static __device__ __forceinline__ float add2(uint32_t w, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), v2{(__bf16)1.f, (__bf16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<_Float16> {
    typedef f16x2 v2;
    typedef f16x4 v4;
    typedef f16x8 v8;
    static constexpr uint32_t kExp = 0x7c00u;
    static constexpr float kBias = 14.f;
    static __device__ __forceinline__ float add2(uint32_t w, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), v2{(_Float16)1.f, (_Float16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// (x, y) as 16-bit pairs: one rounded to nearest (NP = 1), that and what it leaves,
// rounded (2), or their three bf16 pieces (split_bf16.hpp).
template <typename T, int NP>
__device__ __forceinline__ void pieces2(float x, float y, uint32_t (&w)[NP]) {
    if constexpr (NP == 1) {
        const f32x2 v = {x, y};
        w[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename Half<T>::v2));
    } else if constexpr (NP == 2) {
        const f32x2 v = {x, y};
        const auto a = __builtin_convertvector(v, typename Half<T>::v2);
        const f32x2 r = {x - (float)a[0], y - (float)a[1]};
        w[0] = __builtin_bit_cast(uint32_t, a);
        w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, typename Half<T>::v2));
    } else {
        split2(x, y, w[0], w[1], w[2]);
    }
}

// Where a 16-byte chunk of a K or V row lies in LDS: rows of DP elements, the
// chunk's number XORed with bits of its key so that
//  * a K fragment read (16 or 32 keys at one chunk) and
//  * a transposing V read (4 keys x 16 dims per 16 lanes, groups 4 keys or 16
//    dims apart)
// fall on all banks evenly.
template <int DP>
__device__ __forceinline__ int swz_k(int key) {
    return DP == 128 ? key & 15 : (key >> 1) & 7;
}
template <int DP>
__device__ __forceinline__ int swz_v(int key) {
    return DP == 128 ? ((key & 3) << 2) ^ (((key >> 2) & 1) << 1) : (((key >> 1) & 1) << 2) ^ (((key >> 2) & 1) << 1);
}

__device__ __attribute__((aligned(16))) uint32_t g_zero_chunk[4];

constexpr int kMaxPages = 1024;  // page offsets held in LDS: keys per pass >= kMaxPages

// Byte offsets of the pages of keys [b, e) into LDS, -1 for a page outside
// the cache (reported from key lo on: those before are asked for only to begin at a
// whole tile); returns the end of the keys they cover.
__device__ __forceinline__ int stage_pages(const View &c, int seq, int b, int e, int lo, int elem, int64_t *lds, int tid,
                                           int nthreads) {
    const int p0 = paged::page_of(c, b);
    const int n = min(kMaxPages, paged::page_of(c, e - 1) - p0 + 1);
    for (int i = tid; i < n; i += nthreads) {
        const int page = c.table[seq * c.table_stride + p0 + i];
        const bool ok = page >= 0 && page < c.num_pages;
        if (!ok && p0 + i >= paged::page_of(c, lo)) paged::raise(c, paged::kBadPage);
        lds[i] = ok ? page * c.page_stride * elem : -1;
    }
    return (int)min((int64_t)e, (int64_t)(p0 + n) * c.page_size);
}

// One wave's requests for KEYS keys from k0 of K and V straight into LDS (16
// bytes per lane; keys from e on and dims past d read zeros).
template <int DP, int KEYS, int HINT>
__device__ __forceinline__ void request(const View &c, int kvh, const int64_t *pages, int p0, int k0, int e, char *kl,
                                        char *vl, int lane) {
    constexpr int kRowChunks = DP / 8, kRowsPer = 64 / kRowChunks;
    constexpr int kInstr = KEYS / kRowsPer;
    static_assert(kInstr * kRowsPer == KEYS, "whole instructions");
#pragma unroll
    for (int i = 0; i < kInstr; ++i) {
        const int row = i * kRowsPer + lane / kRowChunks, ch = lane % kRowChunks;
        const int key = min(k0 + row, e - 1), pg = paged::page_of(c, key);
        const int64_t off = pages[pg - p0];
        const int64_t at = off + 2 * ((int64_t)(key - pg * c.page_size) * c.row_stride + kvh * c.head_stride);
        const bool ok = k0 + row < e && off >= 0;
        const int ck = ch ^ swz_k<DP>(row), cv = ch ^ swz_v<DP>(row);
        const char *zero = reinterpret_cast<const char *>(g_zero_chunk);
        const char *ks = ok && ck * 8 < c.d ? c.k + at + ck * 16 : zero;
        const char *vs = ok && cv * 8 < c.d ? c.v + at + cv * 16 : zero;
        __builtin_amdgcn_global_load_lds((glb_ptr_t)ks, (lds_ptr_t)(kl + i * 1024), 16, 0, HINT);
        __builtin_amdgcn_global_load_lds((glb_ptr_t)vs, (lds_ptr_t)(vl + i * 1024), 16, 0, HINT);
    }
}

// The chunk kernels' requests for a 64-key tile, 64 / WAVES keys per wave.  Where
// those lie in one page (a whole tile, at a multiple of them) that is one page
// offset per wave, and offsets per lane that do not change; else every row is
// looked up.
template <int DP, int WAVES>
struct Lanes {
    static constexpr int kKeys = 64 / WAVES;
    static constexpr int kRowChunks = DP / 8, kRowsPer = 64 / kRowChunks, kInstr = kKeys / kRowsPer;
    static_assert(kInstr >= 1, "whole instructions per wave");
    uint32_t k[kInstr], v[kInstr];  // bytes from the wave's first row, ~0: zeros
    bool whole;                     // pages hold whole groups of a wave's keys
    bool full;                      // every lane has dims of the head

    __device__ __forceinline__ Lanes(const View &c, int wave, int lane) {
        whole = c.page_size % kKeys == 0 && c.row_stride < (int64_t)1 << 24;
        full = c.d == DP;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const int row = (wave * kInstr + i) * kRowsPer + lane / kRowChunks, ch = lane % kRowChunks;
            const uint32_t at = (uint32_t)(i * kRowsPer + lane / kRowChunks) * (uint32_t)c.row_stride * 2u;
            const int ck = ch ^ swz_k<DP>(row), cv = ch ^ swz_v<DP>(row);
            k[i] = ck * 8 < c.d ? at + ck * 16 : ~0u;
            v[i] = cv * 8 < c.d ? at + cv * 16 : ~0u;
        }
    }
};
// Where the wave's keys of the tile at k0 begin, in bytes from the cache's (same
// for K and V), or -1 where they have to be looked up one by one.
template <int DP, int WAVES>
__device__ __forceinline__ int64_t locate_tile(const View &c, const Lanes<DP, WAVES> &ln, int kvh, const int64_t *pages,
                                               int p0, int k0, int e, int wave) {
    if (!ln.whole || k0 + 64 > e || (k0 & (ln.kKeys - 1)) != 0) return -1;
    const int key = k0 + wave * ln.kKeys, pg = paged::page_of(c, key);
    const int64_t off = pages[pg - p0];
    const int lo = __builtin_amdgcn_readfirstlane((int)off), hi = __builtin_amdgcn_readfirstlane((int)(off >> 32));
    if (hi < 0) return -1;
    return ((int64_t)hi << 32 | (uint32_t)lo) +
           2 * ((int64_t)(key - pg * c.page_size) * c.row_stride + kvh * c.head_stride);
}
// One tile of K or V, located at `at`, into `to`.
template <int DP, int WAVES, bool V>
__device__ __forceinline__ void request_tile(const View &c, const Lanes<DP, WAVES> &ln, int64_t at, int kvh,
                                             const int64_t *pages, int p0, int k0, int e, char *to, int wave, int lane) {
    using L = Lanes<DP, WAVES>;
    const char *const base = V ? c.v : c.k;
    const char *const zero = reinterpret_cast<const char *>(g_zero_chunk);
    if (at >= 0) {
        if (ln.full) {
#pragma unroll
            for (int i = 0; i < L::kInstr; ++i)
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(base + at + (V ? ln.v[i] : ln.k[i])),
                                                 (lds_ptr_t)(to + (wave * L::kInstr + i) * 1024), 16, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < L::kInstr; ++i) {
                const uint32_t x = V ? ln.v[i] : ln.k[i];
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(x != ~0u ? base + at + x : zero),
                                                 (lds_ptr_t)(to + (wave * L::kInstr + i) * 1024), 16, 0, 0);
            }
        }
        return;
    }
#pragma unroll 1
    for (int i = 0; i < L::kInstr; ++i) {
        const int ins = wave * L::kInstr + i;
        const int row = ins * L::kRowsPer + lane / L::kRowChunks, ch = lane % L::kRowChunks;
        const int key = min(k0 + row, e - 1), pg = paged::page_of(c, key);
        const int64_t off = pages[pg - p0];
        const int64_t from = off + 2 * ((int64_t)(key - pg * c.page_size) * c.row_stride + kvh * c.head_stride);
        const int cc = ch ^ (V ? swz_v<DP>(row) : swz_k<DP>(row));
        const char *src = k0 + row < e && off >= 0 && cc * 8 < c.d ? base + from + cc * 16 : zero;
        __builtin_amdgcn_global_load_lds((glb_ptr_t)src, (lds_ptr_t)(to + ins * 1024), 16, 0, 0);
    }
}

template <typename T>
__device__ __forceinline__ typename Half<T>::v4 read_tr(const char *lds) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(typename Half<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                        (__attribute__((address_space(3))) s4 *)(lds)));
}
// Four A operands of a decode tile at once: dims 16 i .. of keys 4 h .. + 3
// and, BYTES further, keys 16 + 4 h .. + 3, at[i] each.  (The builtin waits
// for every request to LDS first, which here are the next tile's; this waits
// for its own reads alone.)
template <int BYTES, typename V8>
__device__ __forceinline__ void read_tr4(const char *lds, const int (&at)[4], V8 (&v)[4]) {
    typedef int i2 __attribute__((ext_vector_type(2)));
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)lds;
    i2 a[4], b[4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %4, %10\n\t"
        "ds_read_b64_tr_b16 %5, %10 offset:%c12\n\t"
        "ds_read_b64_tr_b16 %6, %11\n\t"
        "ds_read_b64_tr_b16 %7, %11 offset:%c12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(a[0]), "=&v"(b[0]), "=&v"(a[1]), "=&v"(b[1]), "=&v"(a[2]), "=&v"(b[2]), "=&v"(a[3]), "=&v"(b[3])
        : "v"(base + at[0]), "v"(base + at[1]), "v"(base + at[2]), "v"(base + at[3]), "n"(BYTES)
        : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = __builtin_bit_cast(V8, __builtin_shufflevector(a[i], b[i], 0, 1, 2, 3));
}
template <typename V8, typename V4>
__device__ __forceinline__ V8 join(V4 a, V4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    constexpr uint32_t e = Half<T>::kExp;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// Whether some element is infinite or NaN: 0 times it is NaN, and so is the sum of all.
template <typename V, int N>
__device__ __forceinline__ bool any_not_finite(const V (&o)[N]) {
    V zero = o[0] * 0.f;
#pragma unroll
    for (int i = 1; i < N; ++i) zero += o[i] * 0.f;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < (int)(sizeof(V) / 4); ++x) sum += zero[x];
    return sum != sum;
}

// Whether x holds in any lane of the workgroup (a barrier on either side: the
// caller may reuse its LDS).
template <int WAVES>
__device__ __forceinline__ bool any_wave(bool x, int *flags, int wave, int lane) {
    const bool mine = __any(x);
    if (lane == 0) flags[wave] = mine;
    __syncthreads();
    bool any = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any |= flags[w] != 0;
    return any;
}

template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// The rows of q as B operands: lane (c, h) holds dims STEP u + 8 h .. + 7 of
// row c, as NP pieces; dims past d and rows out of the tile are zero.
template <typename TA, typename T, int NU, int STEP, int NP>
__device__ __forceinline__ void load_q(const AttnParams &p, const Rows &t, int r, int kvh, int h,
                                       typename Half<T>::v8 (&qf)[NU][NP]) {
    const bool ok = r >= t.r0 && r < t.r1;
    const TA *q = q_row<TA>(p, ok ? r : t.r0, kvh);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int dim = STEP * u + 8 * h;
        float x[8];
        load_vec<8>(q + (dim < p.c.d ? dim : 0), x);
        uint32_t w[NP][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = ok && dim < p.c.d ? x[e] : 0.f;
            x[e] = p.negate ? -x[e] : x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t two[NP];
            pieces2<T, NP>(x[2 * e], x[2 * e + 1], two);
            if constexpr (NP > 1) {
                // an infinite leading piece leaves nothing
                const bool i0 = !(fabsf(x[2 * e]) < INFINITY), i1 = !(fabsf(x[2 * e + 1]) < INFINITY);
                const uint32_t keep = (i0 ? 0u : 0xffffu) | (i1 ? 0u : 0xffff0000u);
#pragma unroll
                for (int n = 1; n < NP; ++n) two[n] &= keep;
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) w[n][e] = two[n];
        }
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const i32x4 v = {(int)w[n][0], (int)w[n][1], (int)w[n][2], (int)w[n][3]};
            qf[u][n] = __builtin_bit_cast(typename Half<T>::v8, v);
        }
    }
}

// The waves' states of a 16-row tile from LDS (rows of DP + 4 floats, their
// maximum and sum) to the tile's rows: thread i takes 4 dims of a row.
template <typename TA, int DP, int WAVES>
__device__ __forceinline__ void join_waves(const AttnParams &p, const Rows &t, int kvh, int split, bool parts,
                                           const float *accs, const float2 *mls, int tid) {
    constexpr int kRow = DP + 4;
    for (int i = tid; i < 16 * DP / 4; i += 64 * WAVES) {
        const int row = i / (DP / 4), dim = 4 * (i % (DP / 4));
        const int rr = t.base + row;
        if (rr < t.r0 || rr >= t.r1 || dim >= p.c.d) continue;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M = max_nan(M, mls[w * 16 + row].x);
        f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float2 x = mls[w * 16 + row];
            const float f = x.x == -INFINITY ? 0.f : exp2f(x.x - M);
            L = fmaf(x.y, f, L);
            A += *reinterpret_cast<const f32x4 *>(accs + (w * 16 + row) * kRow + dim) * f;
        }
        if (parts) {
            const int64_t at = part_row(p, t, rr, kvh) * p.nsplit + split;
            *reinterpret_cast<f32x4 *>(p.acc + at * p.c.d + dim) = A;
            if (dim == 0) p.ml[at] = make_float2(M, L);
        } else {
            const float inv = M == -INFINITY ? 0.f : 1.0f / L;
            const float y[4] = {A[0] * inv, A[1] * inv, A[2] * inv, A[3] * inv};
            store_vec<4>(out_row<TA>(p, rr, kvh) + dim, y);
        }
    }
}

// ---- few rows: decode --------------------------------------------------------------
//
// A tile of 16 rows, WAVES waves that take 32-key tiles in turn, each with a
// ring of two K / V tiles of its own in LDS (no barrier in the loop) and its
// own softmax state; the states are joined in LDS at the end.  S^T = K . Q^T
// on 16x16x32: lane (c = l % 16, h = l / 16) holds keys 16 kb + 4 h + r of row
// c, which are its B operand of O^T = V^T . P^T when V^T takes the keys in the
// same order (two transposing reads: keys 4 h .., 16 + 4 h ..).
//
// Bound by bytes: 64 sequences of 1024 .. 4096 keys, 32 heads over 8 of 128, bf16,
// 659 MB: 131 us (5.0 TB/s) and 4.8 to join; the matrix units have 16 rows for the
// group's 4 and are busy 4.5% of the cycles.
template <typename TA, typename T, int DP, int NP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void paged_decode_kernel(AttnParams p) {
    using H = Half<T>;
    using v8 = typename H::v8;
    constexpr int NU = DP / 32, NB = DP / 16, kTile = 32 * DP * 2;
    constexpr int kOps = 2 * 32 * DP / 512;  // requests per tile and wave
    constexpr int PP = NP > 1 ? NP : 2;      // pieces of P
    constexpr float kBias = NP > 1 ? 16.f : H::kBias;
    // wave, stage, K / V.  (One array for all: with several the compiler tells
    // them apart and waits for every request before any read of the rings.)
    constexpr int kRing = WAVES * 4 * kTile;
    __shared__ __attribute__((aligned(1024))) char lds[kRing + kMaxPages * 8 + 64];
    int64_t *const pages = reinterpret_cast<int64_t *>(lds + kRing);
    int *const flags = reinterpret_cast<int *>(lds + kRing + kMaxPages * 8);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    // Workgroups share no keys here, so they go round the XCDs as they come: a
    // long sequence's then lie on all of them.  (Only a sequence whose rows cross a
    // multiple of 16 has two tiles that walk the same keys: with 7 heads to a group
    // three of eight single tokens.)
    const int id = blockIdx.x;
    const int kvh = id % p.c.hkv, split = (id / p.c.hkv) % p.nsplit, number = id / p.c.hkv / p.nsplit;
    Rows t;
    int seq;
    if (!find_rows(p, number, 16, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    const int b = t.lo + split * p.chunk, e = split == p.nsplit - 1 ? t.hi : min(t.hi, b + p.chunk);

    const int r = t.base + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    v8 qf[NU][NP];
    load_q<TA, T, NU, 32, NP>(p, t, r, kvh, h, qf);
    // keys that every row sees: [all_lo, all_hi)
    int x0, x1, y0, y1;
    row_keys(p, t, t.r0, x0, x1);
    row_keys(p, t, t.r1 - 1, y0, y1);
    const int all_lo = y0, all_hi = x1 + 1;

    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool odd = false;

    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(p.c, pb);
        __syncthreads();  // every wave is done with the pages before
        const int pe = stage_pages(p.c, seq, pb, e, t.lo, 2, pages, tid, 64 * WAVES);
        __syncthreads();
        const int n = (pe - pb + 31) / 32;  // tiles of this pass; this wave's: wave, wave + WAVES, ..
        char *const ring = lds + wave * 4 * kTile;
        if (wave < n)
            request<DP, 32, kNtHint>(p.c, kvh, pages, p0, pb + 32 * wave, pe, ring, ring + kTile, lane);
        int st = 0;
        for (int i = wave; i < n; i += WAVES, st ^= 1) {
            // (past the last tile: the last key again, into the free stage)
            const int k0 = pb + 32 * i, kn = min(k0 + 32 * WAVES, pe - 1);
            __builtin_amdgcn_sched_barrier(0);
            request<DP, 32, kNtHint>(p.c, kvh, pages, p0, kn, pe, ring + (st ^ 1) * 2 * kTile,
                               ring + (st ^ 1) * 2 * kTile + kTile, lane);
            __builtin_amdgcn_sched_barrier(0);
            wait_vm<kOps>();
            __builtin_amdgcn_sched_barrier(0);
            const char *kt = ring + st * 2 * kTile, *vt = kt + kTile;
            f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const v8 kf = *reinterpret_cast<const v8 *>(kt + (kb * 16 + c) * DP * 2 +
                                                                (((4 * u + h) ^ swz_k<DP>(kb * 16 + c)) << 4));
#pragma unroll
                    for (int q = NP - 1; q >= 0; --q) s[kb] = H::mfma16(kf, qf[u][q], s[kb]);
                }
            if (k0 < all_lo || k0 + 32 > min(all_hi, pe)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int j = k0 + 16 * kb + 4 * h + x;
                        s[kb][x] = j >= jmin && j <= jmax && j < pe ? s[kb][x] : -INFINITY;
                    }
                const uint32_t *w = reinterpret_cast<const uint32_t *>(vt);
#pragma unroll 4
                for (int x = 0; x < kTile / 256; ++x) odd |= not_finite<T>(w[x * 64 + lane]);
            }
            float mb = max_nan(max_nan(max_nan(s[0][0], s[0][1]), max_nan(s[0][2], s[0][3])),
                               max_nan(max_nan(s[1][0], s[1][1]), max_nan(s[1][2], s[1][3])));
            const float m_new = max_nan(m, quarter_max_nan(mb));
            // (an infinite key meets q's pieces with either sign, or a zero one)
            if (NP > 1) odd |= jmax >= 0 && m_new != m_new;
            const float mc = m_new == -INFINITY ? 0.f : m_new * p.sc2;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m * p.sc2 - mc);
            float pv[8], sum = 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                pv[x] = __builtin_amdgcn_exp2f(fmaf(s[x >> 2][x & 3], p.sc2, kBias - mc));
                sum += pv[x];
            }
            m = m_new;
#pragma unroll
            for (int i2 = 0; i2 < NB; ++i2) o[i2] *= alpha;
            uint32_t pw[PP][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t two[PP];
                pieces2<T, PP>(pv[2 * x], pv[2 * x + 1], two);
#pragma unroll
                for (int q = 0; q < PP; ++q) pw[q][x] = two[q];
            }
            l = fmaf(l, alpha, sum);
            v8 pf[PP];
#pragma unroll
            for (int q = 0; q < PP; ++q) {
                const i32x4 v = {(int)pw[q][0], (int)pw[q][1], (int)pw[q][2], (int)pw[q][3]};
                pf[q] = __builtin_bit_cast(v8, v);
            }
            const int key = 4 * h + (c >> 2);
#pragma unroll
            for (int i4 = 0; i4 < NB; i4 += 4) {
                int at[4];
                v8 vf[4];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    at[x] = key * DP * 2 + (((2 * (i4 + x) + ((c & 3) >> 1)) ^ swz_v<DP>(key)) << 4) + (c & 1) * 8;
                read_tr4<16 * DP * 2>(vt, at, vf);
#pragma unroll
                for (int q = PP - 1; q >= 0; --q)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[i4 + x] = H::mfma16(vf[x], pf[q], o[i4 + x]);
            }
        }
        wait_vm<0>();  // nothing is still on its way into the ring
        pb = pe;
    }

    // Join the waves: states into LDS (over the rings), then thread i takes
    // 4 dims of a row.
    l = quarter_sum(l);
    const float mt = m == -INFINITY ? m : m * p.sc2;
    odd |= jmax >= 0 && any_not_finite(o);
    constexpr int kRow = DP + 4;
    static_assert(WAVES * 16 * (kRow + 2) * 4 <= kRing, "states over the rings");
    float *const accs = reinterpret_cast<float *>(lds);
    float2 *const mls = reinterpret_cast<float2 *>(accs + WAVES * 16 * kRow);
    if (any_wave<WAVES>(odd, flags, wave, lane)) {
        slow_rows<TA, T>(p, t, seq, kvh, b, e, split, nact > 1, kBias, wave, WAVES, lane);
        return;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) *reinterpret_cast<f32x4 *>(accs + (wave * 16 + c) * kRow + 16 * i + 4 * h) = o[i];
    if (h == 0) mls[wave * 16 + c] = make_float2(mt, l);
    __syncthreads();
    join_waves<TA, DP, WAVES>(p, t, kvh, split, nact > 1, accs, mls, tid);
}

// Row r of a chunk tile (lane half h holds dims 32 i + 8 x + 4 h .. + 3) to out or
// to the parts.
template <typename TA, int NB>
__device__ __forceinline__ void store_rows(const AttnParams &p, const Rows &t, int kvh, int r, int h, int split,
                                           bool parts, float m, float l, const f32x16 (&o)[NB]) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if (r < t.r0 || r >= t.r1) return;
    const int64_t at = parts ? part_row(p, t, r, kvh) * p.nsplit + split : 0;
    const float f = parts ? 1.f : m == -INFINITY ? 0.f : 1.0f / l;
    if (parts && h == 0) p.ml[at] = make_float2(m == -INFINITY ? m : m * p.sc2, l);
    TA *const row = out_row<TA>(p, r, kvh);
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int dim = 32 * i + 8 * x + 4 * h;
            if (dim >= p.c.d) continue;
            const float y[4] = {o[i][4 * x] * f, o[i][4 * x + 1] * f, o[i][4 * x + 2] * f, o[i][4 * x + 3] * f};
            if (parts)
                store_vec<4>(p.acc + at * p.c.d + dim, y);
            else
                store_vec<4>(row + dim, y);
        }
}

// ---- many rows: chunks of prompts ---------------------------------------------------
//
// A tile of 128 rows, four waves of 32; K and V tiles of 64 keys, two stages
// in LDS filled while the tile before is computed, one barrier per tile.  S^T =
// K . Q^T on 32x32x16: lane (c = l % 32, h = l / 32) holds keys 32 kb + 8 (r /
// 4) + 4 h + r % 4 of row c; registers 8 t .. 8 t + 7 are its B operand of O^T
// = V^T . P^T for the 16 keys 16 t .. when V^T takes them in that order.
//
// Bound by the matrix units and the vector ALU together: per tile a wave's
// products take 1024 cycles, its 32 weights per lane some 850, and the two
// waves that share a SIMD hide one in the other only in part.  So two
// workgroups stay on a CU for every type, the products issue first, and the
// softmax is kept short (bf16, 2048 tokens over 16384 keys, 32 heads over 8
// of 128, 515 GFLOP; f32 over bf16, 27.5 GFLOP in three pieces each):
//   the maximum followed at every tile, weights added singly    564 us
//   the maximum followed late                                   560
//   16-bit weights added in pairs (l sums what the product sees) 544
//   products at the higher issue priority              514 .. 525, 1 PFLOP/s at best
//   f32: one workgroup per CU, fragments two ahead              168
//   f32: two per CU (q's pieces in 96 registers, one ahead)     119
// Eight waves in two groups that alternate between products and softmax by
// barriers were no faster (559 against 564).
template <typename TA, typename T, int DP, int ND, int NP>
__global__ __launch_bounds__(256, 2) void paged_chunk_kernel(AttnParams p) {
    using H = Half<T>;
    using v8 = typename H::v8;
    constexpr int NU = 2 * ND, NB = ND, kTile = 64 * DP * 2;  // ND: 32-dim blocks computed
    constexpr float kLate = H::kBias != 0.f ? 6.f : 8.f;
    constexpr float kBias = NP > 1 ? 16.f : H::kBias != 0.f ? 9.f : 0.f;
    constexpr int kAheadK = NP > 1 ? 1 : 3, kAheadV = NP > 1 ? 1 : 5;  // steps that fragments are read ahead
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTile + kMaxPages * 8 + 64];  // stage, K / V; pages; flags
    int64_t *const pages = reinterpret_cast<int64_t *>(lds + 4 * kTile);
    int *const flags = reinterpret_cast<int *>(lds + 4 * kTile + kMaxPages * 8);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5;
    const int id = xcd_chunked(blockIdx.x, gridDim.x);
    // (tiles of one key/value head side by side: they read the same keys)
    const int number = p.ntiles - 1 - id % p.ntiles, rest = id / p.ntiles;
    const int split = rest % p.nsplit, kvh = rest / p.nsplit;
    Rows t;
    int seq;
    if (!find_rows(p, number, 128, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    // (from a multiple of a tile, so that whole tiles lie in few pages)
    const int b0 = t.lo & ~63, b = b0 + split * p.chunk, e = split == nact - 1 ? t.hi : b + p.chunk;

    const int r = t.base + 32 * wave + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    v8 qf[NU][NP];
    load_q<TA, T, NU, 16, NP>(p, t, r, kvh, h, qf);
    // this wave's rows, the keys [any_lo, any_hi) that any of them sees and
    // [all_lo, all_hi) that all of them see
    const int w0 = max(t.r0, t.base + 32 * wave), w1 = min(t.r1, t.base + 32 * wave + 32);
    const bool live = w0 < w1;
    const Lanes<DP, 4> ln(p.c, wave, lane);
    int any_lo, any_hi, all_lo, all_hi;
    row_keys(p, t, live ? w0 : t.r0, any_lo, all_hi);
    row_keys(p, t, live ? w1 - 1 : t.r0, all_lo, any_hi);
    ++all_hi, ++any_hi;

    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = 0.f;
    float m = -INFINITY, l = 0.f;
    bool odd = false;

    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(p.c, pb);
        __syncthreads();
        const int pe = stage_pages(p.c, seq, pb, e, t.lo, 2, pages, tid, 256);
        __syncthreads();
        const int n = (pe - pb + 63) / 64;
        auto ask = [&](int k0, int st) __attribute__((always_inline)) {
            char *const to = lds + st * 2 * kTile;
            const int64_t at = locate_tile<DP, 4>(p.c, ln, kvh, pages, p0, k0, pe, wave);
            request_tile<DP, 4, false>(p.c, ln, at, kvh, pages, p0, k0, pe, to, wave, lane);
            request_tile<DP, 4, true>(p.c, ln, at, kvh, pages, p0, k0, pe, to + kTile, wave, lane);
        };
        ask(pb, 0);
        for (int i = 0; i < n; ++i) {
            const int k0 = pb + 64 * i, st = i & 1;
            // The tile is there, and every wave is done with the one before: the
            // next one's requests have the scores and the softmax of this one to
            // arrive in (the compiler waits for them before the transposing
            // reads of V).  Priorities here are a wave's own, within its SIMD.
            wait_vm<0>();
            __syncthreads();
            if (i + 1 < n) ask(k0 + 64, st ^ 1);
            if (!live || k0 >= any_hi || k0 + 64 <= any_lo) continue;
            const char *kt = lds + st * 2 * kTile, *vt = kt + kTile;
            f32x16 s[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) s[kb][x] = 0.f;
            // (fragments are read steps ahead of their products)
            v8 kf[kAheadK + 1][2];
            auto read_k = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    kf[u % (kAheadK + 1)][kb] = *reinterpret_cast<const v8 *>(kt + (kb * 32 + c) * DP * 2 +
                                                                  (((2 * u + h) ^ swz_k<DP>(c)) << 4));
            };
#pragma unroll
            for (int u = 0; u < kAheadK; ++u) read_k(u);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if (u + kAheadK < NU) read_k(u + kAheadK);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = NP - 1; q >= 0; --q)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) s[kb] = H::mfma32(kf[u % (kAheadK + 1)][kb], qf[u][q], s[kb]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (k0 < all_lo || k0 + 64 > min(all_hi, pe)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int j = k0 + 32 * kb + 8 * (x >> 2) + 4 * h + (x & 3);
                        s[kb][x] = j >= jmin && j <= jmax && j < pe ? s[kb][x] : -INFINITY;
                    }
                const uint32_t *w = reinterpret_cast<const uint32_t *>(vt);
#pragma unroll 4
                for (int x = 0; x < kTile / 256; ++x) odd |= not_finite<T>(w[x * 64 + lane]);
            }
            __builtin_amdgcn_s_setprio(0);
            float mb = max_nan(s[0][0], s[1][0]);
#pragma unroll
            for (int x = 1; x < 16; ++x) mb = max_nan(mb, max_nan(s[0][x], s[1][x]));
            {
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mb), __float_as_uint(mb), false, false);
                mb = max_nan(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            }
            const float m_new = max_nan(m, mb);
            // (an infinite key meets q's pieces with either sign, or a zero one)
            if (NP > 1) odd |= jmax >= 0 && m_new != m_new;
            // The maximum moves on only when some row's is 2^kLate behind: weights then
            // reach 2^(kBias + kLate), within fp16's range too, and most tiles leave
            // the sums unscaled.
            if (__any(!((m_new - m) * p.sc2 <= kLate) && m_new != -INFINITY)) {
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * p.sc2);
                l *= alpha;
#pragma unroll
                for (int i2 = 0; i2 < NB; ++i2) o[i2] *= alpha;
                m = m_new;
            }
            const float mc = kBias - (m == -INFINITY ? 0.f : m * p.sc2);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    s[kb][x] = __builtin_amdgcn_exp2f(fmaf(s[kb][x], p.sc2, mc));
                    if (NP > 1) l += s[kb][x];
                }
            __builtin_amdgcn_s_setprio(1);
            // steps: 16 keys from 16 (n / NB), 32 dims from 32 (n % NB)
            const int key = 4 * h + ((lane & 15) >> 2);
            v8 vf[kAheadV + 1];
            auto read_v = [&](int n) __attribute__((always_inline)) {
                const int ch = 4 * (n % NB) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                const char *at = vt + (16 * (n / NB) + key) * DP * 2 + (lane & 1) * 8 + ((ch ^ swz_v<DP>(key)) << 4);
                vf[n % (kAheadV + 1)] = join<v8>(read_tr<T>(at), read_tr<T>(at + 8 * DP * 2));
            };
#pragma unroll
            for (int n = 0; n < kAheadV; ++n) read_v(n);
            v8 pf[NP];
#pragma unroll
            for (int n = 0; n < 4 * NB; ++n) {
                if (n + kAheadV < 4 * NB) read_v(n + kAheadV);
                if (n % NB == 0) {
                    const int kb = n / NB / 2, x = n / NB % 2;
                    uint32_t pw[NP][4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        uint32_t two[NP];
                        pieces2<T, NP>(s[kb][8 * x + 2 * y], s[kb][8 * x + 2 * y + 1], two);
#pragma unroll
                        for (int q = 0; q < NP; ++q) pw[q][y] = two[q];
                        if (NP == 1) l = H::add2(two[0], l);
                    }
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        const i32x4 v = {(int)pw[q][0], (int)pw[q][1], (int)pw[q][2], (int)pw[q][3]};
                        pf[q] = __builtin_bit_cast(v8, v);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = NP - 1; q >= 0; --q) o[n % NB] = H::mfma32(vf[n % (kAheadV + 1)], pf[q], o[n % NB]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        pb = pe;
    }

    odd |= jmax >= 0 && any_not_finite(o);
    if (any_wave<4>(odd, flags, wave, lane)) {
        slow_rows<TA, T>(p, t, seq, kvh, b, e, split, nact > 1, kBias, wave, 4, lane);
        return;
    }
    store_rows<TA, NB>(p, t, kvh, r, h, split, nact > 1, m, l, o);
}

// Row r of q, dims 16 u + 4 h .. + 3 per step u; zeros for rows outside the tile.
template <int NU>
__device__ __forceinline__ void load_q_f32(const AttnParams &p, const Rows &t, int r, int kvh, int h, f32x4 (&qv)[NU]) {
    const bool ok = r >= t.r0 && r < t.r1;
    const float *q = q_row<float>(p, ok ? r : t.r0, kvh);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int dim = 16 * u + 4 * h;
        const f32x4 x = *reinterpret_cast<const f32x4 *>(q + (dim < p.c.d ? dim : 0));
        qv[u] = ok && dim < p.c.d ? (p.negate ? -x : x) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
}

// ---- fp32 cache -------------------------------------------------------------------
//
// A tile of 16 rows, four waves that take 16-key tiles in turn and both products
// on f32 MFMA (16x16x4).  K: whole rows straight to LDS, a ring of two tiles per
// wave; product e of step u takes dim 16 u + 4 h + e of quarter h on both sides.
// V straight into registers, 256 bytes of a row at once: lane (c, h) loads dims 64 v
// + 4 c .. + 3 of key 4 h + x, and product (v, e, x) takes dim 64 v + 4 i + e as its
// row i.  The next tile is on its way while this one is computed.
//
// Bound by bytes: 4 sequences of 1314 .. 2047 keys, 32 heads of 128, 213 MB: 49 us
// (4.4 TB/s) and 4.7 to join.  K in registers as well was 53.
template <int DP>
__global__ __launch_bounds__(256, 2) void paged_f32_kernel(AttnParams p) {
    constexpr int NU = DP / 16, NV = DP / 64, kRow = DP + 4;
    constexpr int kTile = 16 * DP * 4, kStates = 4 * 2 * kTile;  // K of four waves, two tiles each; then the states
    static_assert(kStates >= 4 * 16 * kRow * 4, "the states fit");
    constexpr int kPer = 256 / DP, kInstr = 16 / kPer;  // rows per request, requests per tile
    __shared__ __attribute__((aligned(1024))) char lds[kStates + 4 * 16 * 8 + kMaxPages * 8 + 64];
    float *const accs = reinterpret_cast<float *>(lds);
    float2 *const mls = reinterpret_cast<float2 *>(lds + kStates);
    int64_t *const pages = reinterpret_cast<int64_t *>(lds + kStates + 4 * 16 * 8);
    int *const flags = reinterpret_cast<int *>(lds + kStates + 4 * 16 * 8 + kMaxPages * 8);
    const View &cc = p.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int id = blockIdx.x;
    const int kvh = id % cc.hkv, split = (id / cc.hkv) % p.nsplit, number = id / cc.hkv / p.nsplit;
    Rows t;
    int seq;
    if (!find_rows(p, number, 16, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    const int b = t.lo + split * p.chunk, e = split == p.nsplit - 1 ? t.hi : min(t.hi, b + p.chunk);
    const int r = t.base + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    f32x4 qv[NU];
    load_q_f32<NU>(p, t, r, kvh, h, qv);
    int x0, x1, y0, y1;
    row_keys(p, t, t.r0, x0, x1);
    row_keys(p, t, t.r1 - 1, y0, y1);
    const int all_lo = y0, all_hi = x1 + 1;

    f32x4 o[NV][4];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[v][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool odd = false;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    struct Tile {
        f32x4 v[4][NV];
    };
    char *const ring = lds + wave * 2 * kTile;
    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(cc, pb);
        __syncthreads();
        const int pe = stage_pages(cc, seq, pb, e, t.lo, 4, pages, tid, 256);
        __syncthreads();
        // byte offset of key j's row and head, -1 past the keys or outside the cache
        auto row_at = [&](int j) __attribute__((always_inline)) -> int64_t {
            const int jc = min(j, pe - 1), pg = paged::page_of(cc, jc);
            const int64_t off = pages[pg - p0];
            return j < pe && off >= 0
                       ? off + 4 * ((int64_t)(jc - pg * cc.page_size) * cc.row_stride + kvh * cc.head_stride)
                       : -1;
        };
        const f32x4 *const zeros = reinterpret_cast<const f32x4 *>(g_zero_chunk);
        auto load = [&](int k0, Tile &f, char *to) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kInstr; ++i) {
                const int row = i * kPer + lane / (DP / 4), ch = lane % (DP / 4) ^ row;
                const int64_t ka = row_at(k0 + row);
                const char *const from = ka >= 0 && 4 * ch < cc.d ? cc.k + ka + 16 * ch
                                                                  : reinterpret_cast<const char *>(g_zero_chunk);
                __builtin_amdgcn_global_load_lds((glb_ptr_t)from, (lds_ptr_t)(to + i * 1024), 16, 0, kNtHint);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t va = row_at(k0 + 4 * h + x);
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int dim = 64 * v + 4 * c;
                    f.v[x][v] = __builtin_nontemporal_load(
                        va >= 0 && dim < cc.d ? reinterpret_cast<const f32x4 *>(cc.v + va + 4 * dim) : zeros);
                }
            }
        };
        int k0 = pb + 16 * wave;
        // (two tiles in turn, without a copy that would wait for the next one)
        auto step = [&](const Tile &now, Tile &next, int st) __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            load(k0 + 64, next, ring + (st ^ 1) * kTile);
            __builtin_amdgcn_sched_barrier(0);
            wait_vm<kInstr + 4 * NV>();
            __builtin_amdgcn_sched_barrier(0);
            const char *const kt = ring + st * kTile + c * DP * 4;
            f32x4 s = zero;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const f32x4 kf = *reinterpret_cast<const f32x4 *>(kt + (((4 * u + h) ^ c) << 4));
#pragma unroll
                for (int x = 0; x < 4; ++x) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x], qv[u][x], s, 0, 0, 0);
            }
            if (k0 < all_lo || k0 + 16 > min(all_hi, pe)) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int j = k0 + 4 * h + x;
                    s[x] = j >= jmin && j <= jmax && j < pe ? s[x] : -INFINITY;
#pragma unroll
                    for (int v = 0; v < NV; ++v)
#pragma unroll
                        for (int y = 0; y < 4; ++y) odd |= !(fabsf(now.v[x][v][y]) < INFINITY);
                }
            }
            const float m_new = max_nan(m, quarter_max_nan(max_nan(max_nan(s[0], s[1]), max_nan(s[2], s[3]))));
            const float mc = m_new == -INFINITY ? 0.f : m_new * p.sc2;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m * p.sc2 - mc);
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], p.sc2, -mc));
                sum += s[x];
            }
            l = fmaf(l, alpha, sum);
            m = m_new;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int y = 0; y < 4; ++y) o[v][y] *= alpha;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        o[v][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(now.v[x][v][y], s[x], o[v][y], 0, 0, 0);
            k0 += 64;
        };
        Tile even, odds;
        if (k0 < pe) load(k0, even, ring);
#pragma unroll 1
        while (k0 < pe) {
            step(even, odds, 0);
            if (k0 >= pe) break;
            step(odds, even, 1);
        }
        wait_vm<0>();  // nothing is on its way into the ring
        pb = pe;
    }
    l = quarter_sum(l);
    if (any_wave<4>(odd, flags, wave, lane)) {
        slow_rows<float, float>(p, t, seq, kvh, b, e, split, nact > 1, 0.f, wave, 4, lane);
        return;
    }
    // o[v][y], register x: dim 64 v + 4 (4 h + x) + y of row c
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4 *>(accs + (wave * 16 + c) * kRow + 64 * v + 16 * h + 4 * x) =
                f32x4{o[v][0][x], o[v][1][x], o[v][2][x], o[v][3][x]};
    if (h == 0) mls[wave * 16 + c] = make_float2(m == -INFINITY ? m : m * p.sc2, l);
    __syncthreads();
    join_waves<float, DP, 4>(p, t, kvh, split, nact > 1, accs, mls, tid);
}

// Prompts: a tile of 64 rows, four waves of 16, K and V tiles of 32 keys in two
// stages that all waves read, the same products as above.  Bound by the f32 matrix
// units: 2048 tokens of 32 heads over 8 of 128, causal, 34 GFLOP 365 us (94 TFLOP/s);
// with 16 rows per workgroup 741, bound by the keys' way from L2.
template <int DP>
__global__ __launch_bounds__(256, 2) void paged_f32_chunk_kernel(AttnParams p) {
    constexpr int NU = DP / 16, NV = DP / 64, kTile = 32 * DP * 4;
    constexpr int kPer = 256 / DP, kInstr = 32 / kPer / 4;  // rows per request, requests per tile and wave
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTile + kMaxPages * 8 + 64];  // stage, K / V; pages; flags
    int64_t *const pages = reinterpret_cast<int64_t *>(lds + 4 * kTile);
    int *const flags = reinterpret_cast<int *>(lds + 4 * kTile + kMaxPages * 8);
    const View &cc = p.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int id = xcd_chunked(blockIdx.x, gridDim.x);
    const int number = p.ntiles - 1 - id % p.ntiles, rest = id / p.ntiles;
    const int split = rest % p.nsplit, kvh = rest / p.nsplit;
    Rows t;
    int seq;
    if (!find_rows(p, number, 64, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    const int b = t.lo + split * p.chunk, e = split == nact - 1 ? t.hi : b + p.chunk;
    const int r = t.base + 16 * wave + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    f32x4 qv[NU];
    load_q_f32<NU>(p, t, r, kvh, h, qv);
    // this wave's rows, the keys that any and that all of them see
    const int w0 = max(t.r0, t.base + 16 * wave), w1 = min(t.r1, t.base + 16 * wave + 16);
    const bool live = w0 < w1;
    int any_lo, any_hi, all_lo, all_hi;
    row_keys(p, t, live ? w0 : t.r0, any_lo, all_hi);
    row_keys(p, t, live ? w1 - 1 : t.r0, all_lo, any_hi);
    ++all_hi, ++any_hi;

    f32x4 o[NV][4];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[v][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool odd = false;
    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(cc, pb);
        __syncthreads();
        const int pe = stage_pages(cc, seq, pb, e, t.lo, 4, pages, tid, 256);
        __syncthreads();
        const int n = (pe - pb + 31) / 32;
        auto ask = [&](int k0, char *to) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kInstr; ++i) {
                const int ins = wave * kInstr + i;
                const int row = ins * kPer + lane / (DP / 4), ch = (lane % (DP / 4)) ^ (row & 15);
                const int key = min(k0 + row, pe - 1), pg = paged::page_of(cc, key);
                const int64_t off = pages[pg - p0];
                const int64_t at = off + 4 * ((int64_t)(key - pg * cc.page_size) * cc.row_stride + kvh * cc.head_stride);
                const bool ok = k0 + row < pe && off >= 0 && 4 * ch < cc.d;
                const char *const zero = reinterpret_cast<const char *>(g_zero_chunk);
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(ok ? cc.k + at + 16 * ch : zero), (lds_ptr_t)(to + ins * 1024),
                                                 16, 0, 0);
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(ok ? cc.v + at + 16 * ch : zero),
                                                 (lds_ptr_t)(to + kTile + ins * 1024), 16, 0, 0);
            }
        };
        ask(pb, lds);
        for (int i = 0; i < n; ++i) {
            const int k0 = pb + 32 * i, st = i & 1;
            // the tile is there, and every wave is done with the one before
            wait_vm<0>();
            __syncthreads();
            if (i + 1 < n) ask(k0 + 32, lds + (st ^ 1) * 2 * kTile);
            if (!live || k0 >= any_hi || k0 + 32 <= any_lo) continue;
            const char *const kt = lds + st * 2 * kTile, *const vt = kt + kTile;
            f32x4 s[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                f32x4 kf[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    kf[kb] = *reinterpret_cast<const f32x4 *>(kt + (16 * kb + c) * DP * 4 + (((4 * u + h) ^ c) << 4));
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        s[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[kb][x], qv[u][x], s[kb], 0, 0, 0);
            }
            if (k0 < all_lo || k0 + 32 > min(all_hi, pe)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int j = k0 + 16 * kb + 4 * h + x;
                        s[kb][x] = j >= jmin && j <= jmax && j < pe ? s[kb][x] : -INFINITY;
                    }
#pragma unroll 4
                for (int x = 0; x < kTile / 1024; ++x) {
                    const f32x4 w = *reinterpret_cast<const f32x4 *>(vt + (x * 64 + lane) * 16);
#pragma unroll
                    for (int y = 0; y < 4; ++y) odd |= !(fabsf(w[y]) < INFINITY);
                }
            }
            const float m_new =
                max_nan(m, quarter_max_nan(max_nan(max_nan(max_nan(s[0][0], s[0][1]), max_nan(s[0][2], s[0][3])),
                                                   max_nan(max_nan(s[1][0], s[1][1]), max_nan(s[1][2], s[1][3])))));
            // (late, as in the 16-bit chunk kernel)
            if (__any(!((m_new - m) * p.sc2 <= 8.f) && m_new != -INFINITY)) {
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * p.sc2);
                l *= alpha;
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int y = 0; y < 4; ++y) o[v][y] *= alpha;
                m = m_new;
            }
            const float mc = m == -INFINITY ? 0.f : m * p.sc2;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    s[kb][x] = __builtin_amdgcn_exp2f(fmaf(s[kb][x], p.sc2, -mc));
                    l += s[kb][x];
                }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        const int key = 4 * h + x;
                        const f32x4 vf = *reinterpret_cast<const f32x4 *>(vt + (16 * kb + key) * DP * 4 +
                                                                          (((16 * v + c) ^ key) << 4));
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            o[v][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[y], s[kb][x], o[v][y], 0, 0, 0);
                    }
        }
        pb = pe;
    }
    l = quarter_sum(l);
#pragma unroll
    for (int v = 0; v < NV; ++v) odd |= jmax >= 0 && any_not_finite(o[v]);
    if (any_wave<4>(odd, flags, wave, lane)) {
        slow_rows<float, float>(p, t, seq, kvh, b, e, split, nact > 1, 0.f, wave, 4, lane);
        return;
    }
    if (r < t.r0 || r >= t.r1) return;
    const bool parts = nact > 1;
    const int64_t at = parts ? part_row(p, t, r, kvh) * p.nsplit + split : 0;
    const float f = parts ? 1.f : m == -INFINITY ? 0.f : 1.0f / l;
    if (parts && h == 0) p.ml[at] = make_float2(m == -INFINITY ? m : m * p.sc2, l);
    float *const row = parts ? p.acc + at * cc.d : out_row<float>(p, r, kvh);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int dim = 64 * v + 16 * h + 4 * x;
            if (dim < cc.d)
                *reinterpret_cast<f32x4 *>(row + dim) = f32x4{o[v][0][x], o[v][1][x], o[v][2][x], o[v][3][x]} * f;
        }
}

// ---- the parts of split rows, in their order ------------------------------------------

// A wave per (token, head), or per row that a sequence of a direct launch can
// have; two dims per lane.
template <typename TA>
__global__ __launch_bounds__(256) void paged_join_kernel(AttnParams p, int bm) {
    const View &c = p.c;
    const int lane = threadIdx.x & 63;
    const int id = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    int s, kvh, r;
    if (p.direct) {  // sequence, row of it, key/value head
        kvh = id % c.hkv;
        s = id / c.hkv / kFewRows;
        if (s >= c.num_seqs) return;
        r = paged::offset_at(c, s) * c.group + id / c.hkv % kFewRows;
        if (r >= paged::offset_at(c, s + 1) * c.group) return;
    } else {
        const int tok = id / c.heads, head = id - tok * c.heads;
        if (tok >= c.tokens) return;
        const int n = paged::wave_leading(c.num_seqs + 1, lane, [&](int i) { return paged::offset_at(c, i) <= tok; });
        if (n == 0 || n > c.num_seqs) return;
        s = n - 1;
        kvh = head / c.group;
        r = tok * c.group + head - kvh * c.group;
    }
    Rows t;
    if (!rows_of(p, r / bm + s, s, bm, t)) return;
    const int nact = active_splits(p, t);
    if (nact <= 1) return;
    const int64_t at = part_row(p, t, r, kvh) * p.nsplit;
    // the largest maximum: 64 splits at a time
    float M = -INFINITY;
    for (int i = lane; i < nact; i += 64) M = max_nan(M, p.ml[at + i].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = max_nan(M, __shfl_xor(M, o));
    const int dim = min(2 * lane, c.d - 2);
    float L = 0.f, a0 = 0.f, a1 = 0.f;
    for (int s0 = 0; s0 < nact; s0 += 8) {
        float2 ml[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t part = at + min(s0 + i, nact - 1);
            ml[i] = p.ml[part];
            v[i] = *reinterpret_cast<const float2 *>(p.acc + part * c.d + dim);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (s0 + i >= nact || ml[i].x == -INFINITY) continue;  // no key of that part is seen
            const float f = exp2f(ml[i].x - M);
            L = fmaf(ml[i].y, f, L);
            a0 = fmaf(v[i].x, f, a0);
            a1 = fmaf(v[i].y, f, a1);
        }
    }
    const float inv = M == -INFINITY ? 0.f : 1.0f / L;
    const float y[2] = {a0 * inv, a1 * inv};
    if (2 * lane < c.d) store_vec<2>(out_row<TA>(p, r, kvh) + dim, y);
}

// What a call launches: a few-row launch, a chunk launch or both.
struct Plan {
    bool few, chunk;
    bool wide;    // the few-row launch has wide workgroups
    int few_max;  // rows of the longest sequence the few-row launch takes
    int chunk_rows;  // of a tile
    int few_split, few_chunk, chunk_split, chunk_chunk;
    int64_t few_parts, chunk_parts;  // rows of parts
    int64_t part_floats;
};

// Waves of a few-row workgroup: two, so that two or more workgroups share a CU;
// as many as the LDS takes where there are too few tiles to fill the CUs and a
// length that such a workgroup walks in a few steps: no split and no second launch
// (12 heads of 64 over 517 keys, f16: 8.6 us and 3.9 to join -> 9.7).
constexpr int kDecodeWaves = 2, kWideWaves64 = 8, kWideWaves128 = 4;
constexpr int kWideKeys = 96;  // per wave
constexpr int kAll = INT32_MAX;

Plan make_plan(const PagedAttnDesc &d) {
    Plan pl{};
    const int64_t group = d.heads / d.kv.kv_heads;
    const int64_t rows = d.tokens * group;
    const bool f32 = d.kv.dtype == GFH_F32;
    pl.few_max = kFewRows;
    const int64_t cus = device_cu_count();
    // the keys that a row of a tile sees at most
    const int64_t sees = std::max<int64_t>(1, d.window > 0 ? std::min(d.max_kv_len, d.window + 127) : d.max_kv_len);
    // Tiles of 16 rows alone where the batch has few and their keys are few too, for
    // they read them once each (us of a call, 16-row tiles / 128-row ones beside them,
    // bf16, 32 heads over 8 of 128: 32 tokens over 500 keys 16 / 22, over 2000 21 / 30,
    // over 8000 64 / 26; 8 times 4 tokens over 2000 24 / 30).
    // fp32: tiles of 64 rows where they fill the CUs (us of a call, 16 rows / 64: 32
    // heads over 8 of 128, a prompt of 128 tokens over 500 keys 34 / 56, 512 64 / 57,
    // 2048 741 / 365, eight of 300 over 600 keys 420 / 238).
    pl.chunk_rows = f32 ? 64 : 128;
    pl.chunk = rows > (sees <= 2048 ? 128 : kFewRows) && d.tokens > d.kv.num_seqs &&
               (!f32 || rows * d.kv.kv_heads >= pl.chunk_rows * cus);
    pl.few = !pl.chunk || d.kv.num_seqs > 1;
    if (!pl.chunk) pl.few_max = kAll;
    auto cut = [&](int64_t tiles, int64_t target, int64_t least, int64_t unit, int &nsplit, int &chunk) {
        const int64_t items = std::max<int64_t>(1, tiles * d.kv.kv_heads);
        int64_t ch = std::max(least, (items * sees + target - 1) / target);
        ch = (ch + unit - 1) / unit * unit;
        nsplit = (int)std::min<int64_t>((sees + ch / 2) / ch, 256);
        nsplit = std::max(nsplit, 1);
        ch = std::max(ch, (sees + nsplit - 1) / nsplit);
        chunk = (int)std::min<int64_t>((ch + unit - 1) / unit * unit, (int64_t)1 << 30);
    };
    const int64_t few_tiles = std::min(d.kv.num_seqs, d.tokens) + (pl.chunk ? 0 : rows / 16);
    // Keys per workgroup of the few-row launch: one round of those that the CUs hold
    // where that is at most 1024 keys, else about 704, for even ends (up to twelve
    // rounds); a row's parts
    // are joined one after the other, so there are no more than a round needs (us of a
    // call, six rounds of at least 128 keys, fp32 384 / this; bf16 and fp32, 32 heads
    // over 8 of 128, lengths between a quarter and all of: one sequence of 16000 37 and
    // 52 / 25 and 45, 8 of 4000 39 and 72 / 27 and 58, 16 of 2000 39 and 55 / 25 and 57,
    // 64 of 2000 85 and 227 / 79 and 180).  (3/4: few_tiles counts tiles that there may
    // be, and lengths are not all the longest.)
    {
        const int64_t items = std::max<int64_t>(1, few_tiles * d.kv.kv_heads);
        int64_t keys = items * sees * 3 / 4 / (2 * cus);
        if (keys > 1024) keys /= (keys + 703) / 704;
        keys = std::max(keys, items * sees / (24 * cus));  // (parts stay some tens of MB at most)
        cut(few_tiles, kAll, std::max<int64_t>(128, keys), 64, pl.few_split, pl.few_chunk);
    }
    const int64_t wide_keys = kWideKeys * (d.kv.head_dim <= 64 ? kWideWaves64 : kWideWaves128);
    pl.wide = !f32 && pl.few_split > 1 && few_tiles * d.kv.kv_heads <= cus &&
              (d.window > 0 ? std::min(d.max_kv_len, d.window + 15) : d.max_kv_len) <= wide_keys;
    if (pl.wide) pl.few_split = 1;
    cut(rows / pl.chunk_rows + 1, (f32 ? 4 : 2) * cus, 512, 64, pl.chunk_split, pl.chunk_chunk);
    // Sequences of few rows go along in the chunk launch where they are few beside
    // its tiles and have few keys to walk (f32 over bf16 / bf16, us of a call, two
    // launches and one): 2048 tokens and 7 single ones of 2048 keys 148 / 90 -> 123 /
    // 63, 1024 and 63 of 1000 keys 153 / 129 -> 136 / 101, 512 and 3 of 2000 keys 60 /
    // 47 -> 59 / 40; but 2000 and one of 8000 keys 148 / 88 -> 337 / 172.
    if (pl.chunk && 64 * d.kv.num_seqs <= rows && std::min<int64_t>(sees, pl.chunk_chunk) <= 2048) pl.few = false;
    auto floats = [&](bool on, int64_t nsplit, int64_t part_rows) {
        return on && nsplit > 1 ? part_rows * nsplit * (d.kv.head_dim + 2) : 0;
    };
    // (one launch after the other uses them)
    pl.few_parts = (pl.chunk ? d.kv.num_seqs * kFewRows : rows) * d.kv.kv_heads;
    pl.chunk_parts = rows * d.kv.kv_heads;
    pl.part_floats = std::max(floats(pl.few, pl.few_split, pl.few_parts), floats(pl.chunk, pl.chunk_split, pl.chunk_parts));
    return pl;
}

}  // namespace

View paged_view(const gfh_paged_kv &kv, int64_t tokens, int64_t heads) {
    View c{};
    c.k = static_cast<char *>(kv.k_pages);
    c.v = static_cast<char *>(kv.v_pages);
    c.num_pages = kv.num_pages;
    c.page_stride = kv.page_stride, c.row_stride = kv.row_stride, c.head_stride = kv.head_stride;
    c.table = kv.page_table;
    c.table_stride = kv.table_stride;
    c.kv_lens = kv.kv_lens, c.q_offsets = kv.q_offsets;
    c.status = kv.status;
    c.page_size = (int)kv.page_size;
    c.page_shift = (kv.page_size & (kv.page_size - 1)) == 0 ? __builtin_ctzll(kv.page_size) : -1;
    c.capacity = (int)(kv.max_pages * kv.page_size);
    c.num_seqs = (int)kv.num_seqs;
    c.tokens = (int)tokens;
    c.heads = (int)heads;
    c.hkv = (int)kv.kv_heads;
    c.group = (int)(heads / kv.kv_heads);
    c.d = (int)kv.head_dim;
    return c;
}

size_t paged_attention_workspace_bytes(const PagedAttnDesc &d) { return (size_t)make_plan(d).part_floats * 4; }

int launch_paged_attention(const PagedAttnDesc &d, void *workspace, hipStream_t s) {
    const Plan pl = make_plan(d);
    AttnParams p{};
    p.c = paged_view(d.kv, d.tokens, d.heads);
    p.q = static_cast<const char *>(d.q);
    p.out = static_cast<char *>(d.out);
    p.ldq = d.ldq, p.ldo = d.ldo;
    // (a scale of 0 keeps masked scores at -inf)
    p.sc2 = d.scale == 0.f ? 1e-38f : std::fabs(d.scale) * 0x1.715476p+0f;
    p.negate = d.scale < 0.f;
    p.causal = d.causal;
    p.window = d.window >= p.c.capacity ? 0 : (int)d.window;
    const int64_t rows = d.tokens * p.c.group;
    auto run = [&](int bm, int nsplit, int chunk, int64_t parts, int min_rows, int max_rows, auto &&kernel) -> int {
        p.direct = max_rows == kFewRows;
        p.ntiles = p.direct ? kFewTiles * (int)d.kv.num_seqs : (int)((rows - 1) / bm + d.kv.num_seqs);
        p.nsplit = nsplit, p.chunk = chunk, p.min_rows = min_rows, p.max_rows = max_rows;
        p.acc = static_cast<float *>(workspace);
        p.ml = reinterpret_cast<float2 *>(p.acc + parts * nsplit * d.kv.head_dim);
        const int64_t blocks = (int64_t)p.ntiles * p.c.hkv * nsplit;
        if (blocks > (int64_t)1 << 23) return set_error(GFH_INVALID_SHAPE, "paged_attention: grid too large");
        kernel(dim3((unsigned)blocks));
        GFH_TRY(check_launch("paged_attention"));
        if (nsplit > 1) {
            const dim3 join((unsigned)(((p.direct ? d.kv.num_seqs * kFewRows * p.c.hkv : d.tokens * d.heads) + 3) / 4));
            if (d.dtype == GFH_F32)
                hipLaunchKernelGGL(paged_join_kernel<float>, join, dim3(256), 0, s, p, bm);
            else if (d.dtype == GFH_BF16)
                hipLaunchKernelGGL(paged_join_kernel<__bf16>, join, dim3(256), 0, s, p, bm);
            else
                hipLaunchKernelGGL(paged_join_kernel<_Float16>, join, dim3(256), 0, s, p, bm);
            GFH_TRY(check_launch("paged_attention (join)"));
        }
        return GFH_SUCCESS;
    };
    const int64_t hd = d.kv.head_dim;
    auto few = [&](dim3 grid) {
        auto go = [&](auto ta, auto t, auto np) {
            using TA = decltype(ta);
            using T = decltype(t);
            constexpr int NP = decltype(np)::value;
            auto width = [&](auto dp, auto w) {
                constexpr int DP = decltype(dp)::value, W = decltype(w)::value;
                hipLaunchKernelGGL((paged_decode_kernel<TA, T, DP, NP, W>), grid, dim3(64 * W), 0, s, p);
            };
            using Two = std::integral_constant<int, kDecodeWaves>;
            if (hd <= 64) {
                using D = std::integral_constant<int, 64>;
                pl.wide ? width(D{}, std::integral_constant<int, kWideWaves64>{}) : width(D{}, Two{});
            } else {
                using D = std::integral_constant<int, 128>;
                pl.wide ? width(D{}, std::integral_constant<int, kWideWaves128>{}) : width(D{}, Two{});
            }
        };
        using One = std::integral_constant<int, 1>;
        using Three = std::integral_constant<int, 3>;
        if (d.kv.dtype == GFH_F32) {
            if (hd <= 64)
                hipLaunchKernelGGL(paged_f32_kernel<64>, grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL(paged_f32_kernel<128>, grid, dim3(256), 0, s, p);
        } else if (d.dtype == GFH_F32)
            go(float{}, __bf16{}, Three{});
        else if (d.dtype == GFH_BF16)
            go(__bf16{}, __bf16{}, One{});
        else
            go(_Float16{}, _Float16{}, One{});
    };
    auto many = [&](dim3 grid) {
        auto go = [&](auto ta, auto t, auto np) {
            using TA = decltype(ta);
            using T = decltype(t);
            constexpr int NP = decltype(np)::value;
            if (hd <= 64)
                hipLaunchKernelGGL((paged_chunk_kernel<TA, T, 64, 2, NP>), grid, dim3(256), 0, s, p);
            else if (hd <= 96)
                hipLaunchKernelGGL((paged_chunk_kernel<TA, T, 128, 3, NP>), grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((paged_chunk_kernel<TA, T, 128, 4, NP>), grid, dim3(256), 0, s, p);
        };
        using One = std::integral_constant<int, 1>;
        using Three = std::integral_constant<int, 3>;
        if (d.kv.dtype == GFH_F32) {
            if (hd <= 64)
                hipLaunchKernelGGL(paged_f32_chunk_kernel<64>, grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL(paged_f32_chunk_kernel<128>, grid, dim3(256), 0, s, p);
        } else if (d.dtype == GFH_F32)
            go(float{}, __bf16{}, Three{});
        else if (d.dtype == GFH_BF16)
            go(__bf16{}, __bf16{}, One{});
        else
            go(_Float16{}, _Float16{}, One{});
    };
    if (pl.chunk)
        GFH_TRY(run(pl.chunk_rows, pl.chunk_split, pl.chunk_chunk, pl.chunk_parts, pl.few ? pl.few_max + 1 : 0, kAll, many));
    if (pl.few) GFH_TRY(run(16, pl.few_split, pl.few_chunk, pl.few_parts, 0, pl.few_max, few));
    return GFH_SUCCESS;
}

}  // namespace gfh
