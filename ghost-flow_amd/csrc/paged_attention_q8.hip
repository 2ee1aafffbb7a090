// paged_attention_q8.hip -- the attention of paged_attention.hip over a cache of 8
// bits: codes c and a step byte per row (paged_quant.hpp), x = (c - 128) s.
//
// The step has four significant bits, so x s' with s' = s / 4 is an f16 exactly: four
// codes become f16 by two byte permutes (0x6400 + c is the f16 1024 + c) and two
// packed fused multiply-adds, (1024 + c) s' - 1152 s', whose one rounding is none.
// Both products then run on f16 matrix instructions on the exact values, with no
// factor per key in the scores or the weights; the two factors of 4 go into the
// softmax's scale and into l.  q is brought to [2^14, 2^15) by a power of two per row:
// bf16 and f16 are then f16 with all their bits down to 2^-39 of the row's largest
// magnitude, fp32 two f16 pieces (22 bits).  P is two f16 pieces, or one where the output's
// own rounding is eight times as coarse (bf16 prompts).
//
// Nothing in the cache is infinite or NaN, whatever its bytes, so keys that a row does
// not see need no look; a row of q that is not finite gets NaN.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_attention.hpp"
#include "paged_quant.hpp"

namespace gfh {
namespace {

struct Q8Params {
    AttnParams a;
    const uint8_t *ks, *vs;
    int64_t scale_page, scale_head;  // bytes
    int side;     // heads of a few-row workgroup, a divisor of its waves
    bool eights;  // 8 keys from a multiple of 8 lie in one page, their step bytes aligned
};

// A row of zeros, for pages outside the cache (and a step byte for it).
#define GFH_MID4 0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u
__device__ __attribute__((aligned(128))) const uint32_t g_mid_row[32] = {GFH_MID4, GFH_MID4, GFH_MID4, GFH_MID4,
                                                                         GFH_MID4, GFH_MID4, GFH_MID4, GFH_MID4};
#undef GFH_MID4

constexpr int kPageSlots = 1024;  // page numbers held in LDS: keys per pass >= kPageSlots

// The pages of keys [b, e) into LDS, -1 for one outside the cache (reported from key
// lo on: those before are asked for only to begin at a whole tile); returns the end of
// the keys they cover.
__device__ __forceinline__ int stage_page_numbers(const View &c, int seq, int b, int e, int lo, int *lds, int tid,
                                                  int nthreads) {
    const int p0 = paged::page_of(c, b);
    const int n = min(kPageSlots, paged::page_of(c, e - 1) - p0 + 1);
    for (int i = tid; i < n; i += nthreads) {
        const int page = c.table[seq * c.table_stride + p0 + i];
        const bool ok = page >= 0 && page < c.num_pages;
        if (!ok && p0 + i >= paged::page_of(c, lo)) paged::raise(c, paged::kBadPage);
        lds[i] = ok ? page : -1;
    }
    return (int)min((int64_t)e, (int64_t)(p0 + n) * c.page_size);
}

// s / 4 and -1152 s / 4 of a step byte, twice each.
struct Step {
    f16x2 f, g;
};
__device__ __forceinline__ float quarter_step(uint32_t b) {
    return __uint_as_float((min(b, (uint32_t)paged::kMaxStep) + (paged::kStepBits - 16)) << 20);
}
__device__ __forceinline__ Step step_pair(float s0, float s1) {
    const f16x2 f = {(_Float16)s0, (_Float16)s1};
    return {f, f * (_Float16)-1152.f};  // (exact: four bits times 9 2^7)
}
// Codes in bytes 0, 1 (HI: 2, 3) of w as f16 values.
template <bool HI>
__device__ __forceinline__ uint32_t values(uint32_t w, const Step &s) {
    const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, s.f, s.g));
}

// The rows of q as B operands: dims dim_of(u) .. + 7 per step u, as NQ f16 pieces of
// q 2^k; `over` takes the maximum over the lanes of a row.  Returns 2^-k, NaN for a
// row that is not finite.
template <typename TA, int NU, int NQ, typename D, typename F>
__device__ __forceinline__ float load_q8(const AttnParams &p, const Rows &t, int r, int kvh, D &&dim_of,
                                         f16x8 (&qf)[NU][NQ], F &&over) {
    const bool ok = r >= t.r0 && r < t.r1;
    const TA *q = q_row<TA>(p, ok ? r : t.r0, kvh);
    float x[NU][8], most = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int dim = dim_of(u);
        load_vec<8>(q + (dim < p.c.d ? dim : 0), x[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[u][e] = ok && dim < p.c.d ? x[u][e] : 0.f;
            most = max_nan(most, fabsf(x[u][e]));
        }
    }
    most = over(most);
    const int k = most > 0.f ? min(14 + 127 - (int)(__float_as_uint(most) >> 23), 100) : 0;
    const bool finite = most < INFINITY;
    float up = finite ? __uint_as_float((uint32_t)(127 + k) << 23) : NAN;
    const float down = finite ? __uint_as_float((uint32_t)(127 - k) << 23) : NAN;
    up = p.negate ? -up : up;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        uint32_t w[NQ][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t two[NQ];
            pieces2<_Float16, NQ>(x[u][2 * e] * up, x[u][2 * e + 1] * up, two);
#pragma unroll
            for (int n = 0; n < NQ; ++n) w[n][e] = two[n];
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const i32x4 v = {(int)w[n][0], (int)w[n][1], (int)w[n][2], (int)w[n][3]};
            qf[u][n] = __builtin_bit_cast(f16x8, v);
        }
    }
    return down;
}
// The softmax's factor of a row whose q was scaled by 1 / down.  Kept finite, as 0 times it has to
// be 0, and above 0, as a masked score's -inf times it has to be -inf: sums of products here are
// below 2^35, which 1e-38 takes to nothing.  (A NaN passes either comparison.)
__device__ __forceinline__ float row_scale(const AttnParams &p, float down) {
    const float s = p.sc2 * (4.f * down);
    return s > 3e38f ? 3e38f : s < 1e-38f ? 1e-38f : s;
}

__device__ __forceinline__ f16x8 as_operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const i32x4 v = {(int)a, (int)b, (int)c, (int)d};
    return __builtin_bit_cast(f16x8, v);
}

// ---- few rows: decode --------------------------------------------------------------
//
// A tile of 16 rows of pp.side neighbouring key/value heads, whose rows of the cache
// lie side by side; WAVES / side waves of a head take 32-key tiles in turn, each with
// its own softmax state, and the states of a head are joined in LDS at the end.  Codes go from
// memory straight into the registers of the lane that multiplies them: lane (c = l %
// 16, h = l / 16) has
//   K: dims 64 i + 16 h .. + 15 of keys 8 (c / 4) + c % 4 and + 4 (rows c of two blocks), so
//      row 4 h + x of block kb is key 8 h + 4 kb + x, and lane h has keys 8 h .. + 7 of S^T;
//   V: dims DP / 16 c .. of those keys 8 h .. + 7: the byte permutes that make f16 of
//      codes also bring the same dim of two keys side by side, so V needs no
//      transposition elsewhere.  Row i of block b of O^T is dim DP / 16 i + b.
// The next tile's K is asked for when this one's has been multiplied, V likewise: half
// a tile per wave is on its way at any time, in registers that are free anyway.
//
// Bound by bytes, and by their latency: 64 sequences of up to 4096 keys, 32 heads over 8 of 128,
// 333 MB: bf16 72 to 79 us (4.2 to 4.6 TB/s) and 5 for the join, fp32 with two workgroups to a CU
// 96 with it; pages of 100 rows, a look-up and a byte of steps per key, 100 and 146.  Two tiles ahead (234 registers) gained nothing, four waves
// per SIMD spill (134 us), loads that stay in the caches took 82.  One token over 517 keys:
// 9.7 us, the way from offsets to length to page to codes and the waves' join.
template <typename TA, int DP, int NQ, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NQ > 1 ? 2 : 3) void paged_q8_decode_kernel(Q8Params pp) {
    using H = Half<_Float16>;
    constexpr int NU = DP / 32, NB = DP / 16, KP = DP / 64, NV = DP / 64;  // NV: dwords of V per key
    constexpr float kBias = H::kBias;
    constexpr int kRow = DP + 4;
    __shared__ __attribute__((aligned(16))) char lds[WAVES * 16 * (kRow + 2) * 4 + kPageSlots * 4];
    float *const accs = reinterpret_cast<float *>(lds);
    float2 *const mls = reinterpret_cast<float2 *>(accs + WAVES * 16 * kRow);
    int *const pages = reinterpret_cast<int *>(lds + WAVES * 16 * (kRow + 2) * 4);
    const AttnParams &p = pp.a;
    const View &cc = p.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    // The workgroups of a tile's heads go to one XCD, as their rows share lines of memory.
    const int groups = cc.hkv / pp.side, units = gridDim.x / groups, even = units & ~7;
    int id = blockIdx.x, first, unit;
    if (id < even * groups) {
        first = (id >> 3) % groups, unit = (id & 7) + 8 * ((id >> 3) / groups);
    } else {
        id -= even * groups;
        first = id % groups, unit = even + id / groups;
    }
    // (parts of one number later: whether a part has keys then does not go by the XCD)
    const int number = unit % p.ntiles, split = unit / p.ntiles;
    const int kvh = first * pp.side + wave % pp.side, sub = wave / pp.side, subs = WAVES / pp.side;
    Rows t;
    int seq;
    if (!find_rows(p, number, 16, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    // (whole tiles: keys before t.lo are masked)
    const int b0 = t.lo & ~31, b = b0 + split * p.chunk, e = split == nact - 1 ? t.hi : b + p.chunk;

    const int r = t.base + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    f16x8 qf[NU][NQ];
    float scl = 0.f;
    // keys that every row sees: [all_lo, all_hi)
    int x0, x1, y0, y1;
    row_keys(p, t, t.r0, x0, x1);
    row_keys(p, t, t.r1 - 1, y0, y1);
    const int all_lo = y0, all_hi = x1 + 1;

    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    typedef uint32_t vrow __attribute__((ext_vector_type(NV)));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    i32x4 kw[2][KP];
    vrow vw[8];
    u32x2 ks, vs;  // step bytes: of the lane's two keys at byte c % 4 of either word; of keys 8 h ..
    const int64_t head = kvh * cc.head_stride, scale_head = kvh * pp.scale_head;
    // dims past the head's: its first ones, which q's zeros or nobody takes
    int kdim[KP];
#pragma unroll
    for (int i = 0; i < KP; ++i) kdim[i] = 64 * i + 16 * h < cc.d ? 64 * i + 16 * h : 0;
    const int vdim = DP / 16 * c < cc.d ? DP / 16 * c : 0;
    const char *const mid = reinterpret_cast<const char *>(g_mid_row);

    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(cc, pb);
        __syncthreads();  // every wave is done with the pages before
        const int pe = stage_page_numbers(cc, seq, pb, e, t.lo, pages, tid, 64 * WAVES);
        __syncthreads();
        // Where a key's row begins, how far the next one is, and its step byte.
        auto at = [&](int key, const char *cache, const uint8_t *bytes, const char *&rows, int64_t &stride,
                      const uint8_t *&steps) __attribute__((always_inline)) {
            const int pg = paged::page_of(cc, key), page = pages[pg - p0], prow = key - pg * cc.page_size;
            const bool ok = page >= 0;
            rows = ok ? cache + page * cc.page_stride + prow * cc.row_stride + head : mid;
            stride = ok ? cc.row_stride : 0;
            steps = ok ? bytes + page * pp.scale_page + scale_head + prow : reinterpret_cast<const uint8_t *>(mid);
        };
        const char *rows;
        const uint8_t *steps;
        int64_t stride;
        auto load_k = [&](int k0) __attribute__((always_inline)) {
            if (pp.eights) {  // a group of 8 keys, from a multiple of 8 (past the end: the last)
                at(min(k0 + 8 * (c >> 2), (pe - 1) & ~7), cc.k, pp.ks, rows, stride, steps);
                rows += (c & 3) * stride;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < KP; ++i)
                        kw[kb][i] = __builtin_nontemporal_load(
                            reinterpret_cast<const i32x4 *>(rows + 4 * kb * stride + kdim[i]));
                ks = *reinterpret_cast<const u32x2 *>(steps);
            } else {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    at(min(k0 + 8 * (c >> 2) + (c & 3) + 4 * kb, pe - 1), cc.k, pp.ks, rows, stride, steps);
#pragma unroll
                    for (int i = 0; i < KP; ++i) kw[kb][i] = *reinterpret_cast<const i32x4 *>(rows + kdim[i]);
                    ks[kb] = (uint32_t)*steps << (8 * (c & 3));
                }
            }
        };
        auto load_v = [&](int k0) __attribute__((always_inline)) {
            if (pp.eights) {
                at(min(k0 + 8 * h, (pe - 1) & ~7), cc.v, pp.vs, rows, stride, steps);
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    vw[x] = __builtin_nontemporal_load(reinterpret_cast<const vrow *>(rows + x * stride + vdim));
                vs = *reinterpret_cast<const u32x2 *>(steps);
            } else {
                vs = u32x2{0u, 0u};
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    at(min(k0 + 8 * h + x, pe - 1), cc.v, pp.vs, rows, stride, steps);
                    vw[x] = *reinterpret_cast<const vrow *>(rows + vdim);
                    vs[x >> 2] |= (uint32_t)*steps << (8 * (x & 3));
                }
            }
        };
        int k0 = pb + 32 * sub;
        if (k0 < pe) load_k(k0), load_v(k0);
        if (pb == b) {  // (while the first tile is on its way)
            const float down = load_q8<TA, NU, NQ>(
                p, t, r, kvh, [&](int u) { return 64 * (u / 2) + 16 * h + 8 * (u % 2); }, qf,
                [](float x) { return quarter_max_nan(x); });
            scl = row_scale(p, down);
        }
#pragma unroll 1
        for (; k0 < pe; k0 += 32 * subs) {
            f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const float sk = quarter_step(ks[kb] >> (8 * (c & 3)) & 0xff);
                const Step st = step_pair(sk, sk);
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    const uint32_t w0 = (uint32_t)kw[kb][u / 2][2 * (u % 2)], w1 = (uint32_t)kw[kb][u / 2][2 * (u % 2) + 1];
                    const f16x8 kf = as_operand(values<false>(w0, st), values<true>(w0, st), values<false>(w1, st),
                                                values<true>(w1, st));
#pragma unroll
                    for (int q = NQ - 1; q >= 0; --q) s[kb] = H::mfma16(kf, qf[u][q], s[kb]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool more = k0 + 32 * subs < pe;
            if (more) load_k(k0 + 32 * subs);
            __builtin_amdgcn_sched_barrier(0);
            if (k0 < all_lo || k0 + 32 > min(all_hi, pe)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int j = k0 + 8 * h + 4 * kb + x;
                        s[kb][x] = j >= jmin && j <= jmax && j < pe ? s[kb][x] : -INFINITY;
                    }
            }
            const float mb = max_nan(max_nan(max_nan(s[0][0], s[0][1]), max_nan(s[0][2], s[0][3])),
                                     max_nan(max_nan(s[1][0], s[1][1]), max_nan(s[1][2], s[1][3])));
            const float m_new = max_nan(m, quarter_max_nan(mb));
            const float mc = m_new == -INFINITY ? 0.f : m_new * scl;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m * scl - mc);
            float pv[8], sum = 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                pv[x] = __builtin_amdgcn_exp2f(fmaf(s[x >> 2][x & 3], scl, kBias - mc));
                sum += pv[x];
            }
            m = m_new;
            l = fmaf(l, alpha, sum);
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= alpha;
            f16x8 pf[2];
            {
                uint32_t pw[2][4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t two[2];
                    pieces2<_Float16, 2>(pv[2 * x], pv[2 * x + 1], two);
                    pw[0][x] = two[0], pw[1][x] = two[1];
                }
                pf[0] = as_operand(pw[0][0], pw[0][1], pw[0][2], pw[0][3]);
                pf[1] = as_operand(pw[1][0], pw[1][1], pw[1][2], pw[1][3]);
            }
            Step vst[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t w = vs[x >> 1] >> (16 * (x & 1));
                vst[x] = step_pair(quarter_step(w & 0xff), quarter_step(w >> 8 & 0xff));
            }
#pragma unroll
            for (int w = 0; w < NV; ++w)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // bytes 2 half, + 1 of keys 2 x and 2 x + 1
                    uint32_t two[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        two[x] = __builtin_amdgcn_perm(vw[2 * x + 1][w], vw[2 * x][w], half ? 0x07030602u : 0x05010400u);
                    const f16x8 va = as_operand(values<false>(two[0], vst[0]), values<false>(two[1], vst[1]),
                                                values<false>(two[2], vst[2]), values<false>(two[3], vst[3]));
                    const f16x8 vb = as_operand(values<true>(two[0], vst[0]), values<true>(two[1], vst[1]),
                                                values<true>(two[2], vst[2]), values<true>(two[3], vst[3]));
                    const int i = 4 * w + 2 * half;
#pragma unroll
                    for (int q = 1; q >= 0; --q) {
                        o[i] = H::mfma16(va, pf[q], o[i]);
                        o[i + 1] = H::mfma16(vb, pf[q], o[i + 1]);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_v(k0 + 32 * subs);
            __builtin_amdgcn_sched_barrier(0);
        }
        pb = pe;
    }

    // Join the waves of a head: o[b], register x is dim DP / 16 (4 h + x) + b of row c.
    l = 0.25f * quarter_sum(l);
    const float mt = m == -INFINITY ? m : m * scl;
    const int state = wave % pp.side * subs + sub;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int i = 0; i < NB; i += 4)
            *reinterpret_cast<f32x4 *>(accs + (state * 16 + c) * kRow + NB * (4 * h + x) + i) =
                f32x4{o[i][x], o[i + 1][x], o[i + 2][x], o[i + 3][x]};
    if (h == 0) mls[state * 16 + c] = make_float2(mt, l);
    __syncthreads();
    const int place = wave % pp.side;
    join_waves<TA, DP>(p, t, kvh, split, nact > 1, accs + place * subs * 16 * kRow, mls + place * subs * 16, subs,
                       sub * 64 + lane);
}

// ---- many rows: chunks of prompts ---------------------------------------------------
//
// A tile of 32 rows per wave, K and V tiles of 64 keys in two stages of LDS, one barrier
// per tile and the products as in paged_attention.hip.  Codes come into registers (16 of K
// and of V per thread and row, a tile ahead), become f16 there and go to LDS as the
// layout of those products wants them.
//
// Bound by the vector ALU and the matrix units together, as the 16-bit kernel is, with some
// 90 vector instructions per wave and tile more for the codes (of 290; half as many in tiles
// of 256 rows): 2048 tokens over 16384 keys, 32 heads over 8 of 128, 515 GFLOP, bf16 537 to 566 us
// from card to card (0.91 to 0.96 PFLOP/s; 542 where a bf16 cache takes 511), f16 738 to 756 (773
// GFLOP with two pieces of P, 1.04), fp32 in two pieces 885 to 904 (1.15).
//
// P is rounded to f16 for bf16 q, and is two pieces (22 bits) for f16 and fp32.  Relative errors
// against 64 bits there (root of the mean square) and us, one piece / two: bf16 1.67e-3 / 1.66e-3,
// the output's own rounding, and 552 / 750; f16 2.94e-4 / 2.07e-4, its own, and 559 / 756: a bf16
// output hides that rounding, an f16 one would be 42% further off.  One piece is also what l sums.
template <typename TA, int DP, int ND, int NQ, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_q8_chunk_kernel(Q8Params pp) {
    using H = Half<_Float16>;
    static_assert(DP % 16 == 0 && (WAVES == 4 || WAVES == 8));
    constexpr int NU = 2 * ND, NB = ND, kTile = 64 * DP * 2;  // ND: 32-dim blocks computed
    constexpr int NP = std::is_same_v<TA, __bf16> ? 1 : 2;    // pieces of P (see above)
    constexpr float kLate = 6.f, kBias = 9.f;
    constexpr int kAheadK = NQ > 1 ? 1 : 2, kAheadV = NQ > 1 ? 1 : 3;  // steps that fragments are read ahead
    constexpr int kRowUnits = DP / 16, kStep = 64 * WAVES / kRowUnits;
    constexpr int kUnits = kStep < 64 ? 64 / kStep : 1;  // of 16 codes, per thread that has one
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTile + kPageSlots * 4];  // stage, K / V; pages
    int *const pages = reinterpret_cast<int *>(lds + 4 * kTile);
    const AttnParams &p = pp.a;
    const View &cc = p.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5;
    const int id = xcd_chunked(blockIdx.x, gridDim.x);
    // (tiles of one key/value head side by side: they read the same keys)
    const int number = p.ntiles - 1 - id % p.ntiles, rest = id / p.ntiles;
    const int split = rest % p.nsplit, kvh = rest / p.nsplit;
    Rows t;
    int seq;
    if (!find_rows(p, number, 32 * WAVES, lane, t, seq)) return;
    const int nact = active_splits(p, t);
    if (split >= nact) return;
    const int b0 = t.lo & ~63, b = b0 + split * p.chunk, e = split == nact - 1 ? t.hi : b + p.chunk;

    const int r = t.base + 32 * wave + c;
    int jmin, jmax;
    row_keys(p, t, r, jmin, jmax);
    f16x8 qf[NU][NQ];
    const float down = load_q8<TA, NU, NQ>(p, t, r, kvh, [&](int u) { return 8 * h + 16 * u; }, qf, [](float x) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return max_nan(__uint_as_float(a[0]), __uint_as_float(a[1]));
    });
    const float scl = row_scale(p, down);
    // this wave's rows, the keys [any_lo, any_hi) that any of them sees and
    // [all_lo, all_hi) that all of them see
    const int w0 = max(t.r0, t.base + 32 * wave), w1 = min(t.r1, t.base + 32 * wave + 32);
    const bool live = w0 < w1;
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

    // this thread's units of a tile: 16 codes from dim 16 uch of key urow + kStep i
    const int urow = tid / kRowUnits, uch = tid % kRowUnits;
    const bool has = kStep <= 64 || urow < 64;
    const int udim = 16 * uch < cc.d ? 16 * uch : 0;  // (past the head's dims: its first, for nobody)
    const char *const mid = reinterpret_cast<const char *>(g_mid_row);
    struct {
        i32x4 k[kUnits], v[kUnits];
        uint32_t ks[kUnits], vs[kUnits];
    } f;

    for (int pb = b; pb < e;) {
        const int p0 = paged::page_of(cc, pb);
        __syncthreads();
        const int pe = stage_page_numbers(cc, seq, pb, e, t.lo, pages, tid, 64 * WAVES);
        __syncthreads();
        const int n = (pe - pb + 63) / 64;
        auto ask = [&](int k0) __attribute__((always_inline)) {
            if (!has) return;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int key = min(k0 + urow + kStep * i, pe - 1), pg = paged::page_of(cc, key);
                const int page = pages[pg - p0], prow = key - pg * cc.page_size;
                const bool ok = page >= 0;
                const int64_t at = page * cc.page_stride + prow * cc.row_stride + kvh * cc.head_stride + udim;
                const int64_t sat = page * pp.scale_page + kvh * pp.scale_head + prow;
                f.k[i] = *reinterpret_cast<const i32x4 *>(ok ? cc.k + at : mid);
                f.v[i] = *reinterpret_cast<const i32x4 *>(ok ? cc.v + at : mid);
                f.ks[i] = ok ? pp.ks[sat] : 0;
                f.vs[i] = ok ? pp.vs[sat] : 0;
            }
        };
        auto put = [&](int st) __attribute__((always_inline)) {
            if (!has) return;
            char *const to = lds + st * 2 * kTile;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int row = urow + kStep * i;
                auto widen = [&](const i32x4 &w, uint32_t byte, char *tile, int swz) __attribute__((always_inline)) {
                    const float s = quarter_step(byte);
                    const Step stp = step_pair(s, s);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t w0 = (uint32_t)w[2 * x], w1 = (uint32_t)w[2 * x + 1];
                        *reinterpret_cast<f16x8 *>(tile + row * DP * 2 + (((2 * uch + x) ^ swz) << 4)) =
                            as_operand(values<false>(w0, stp), values<true>(w0, stp), values<false>(w1, stp),
                                       values<true>(w1, stp));
                    }
                };
                widen(f.k[i], f.ks[i], to, swz_k<DP>(row));
                widen(f.v[i], f.vs[i], to + kTile, swz_v<DP>(row));
            }
        };
        ask(pb);
        put(0);
        if (n > 1) ask(pb + 64);
        for (int i = 0; i < n; ++i) {
            const int k0 = pb + 64 * i, st = i & 1;
            // The tile is there, and every wave is done with the one before, whose
            // place the next one takes.
            __syncthreads();
            if (i + 1 < n) put(st ^ 1);
            if (i + 2 < n) ask(k0 + 128);
            if (!live || k0 >= any_hi || k0 + 64 <= any_lo) continue;
            const char *kt = lds + st * 2 * kTile, *vt = kt + kTile;
            f32x16 s[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) s[kb][x] = 0.f;
            // (fragments are read steps ahead of their products)
            f16x8 kf[kAheadK + 1][2];
            auto read_k = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    kf[u % (kAheadK + 1)][kb] = *reinterpret_cast<const f16x8 *>(kt + (kb * 32 + c) * DP * 2 +
                                                                                 (((2 * u + h) ^ swz_k<DP>(c)) << 4));
            };
#pragma unroll
            for (int u = 0; u < kAheadK; ++u) read_k(u);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if (u + kAheadK < NU) read_k(u + kAheadK);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = NQ - 1; q >= 0; --q)
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
            // The maximum moves on only when some row's is 2^kLate behind.
            if (__any(!((m_new - m) * scl <= kLate) && m_new != -INFINITY)) {
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * scl);
                l *= alpha;
#pragma unroll
                for (int i2 = 0; i2 < NB; ++i2) o[i2] *= alpha;
                m = m_new;
            }
            const float mc = kBias - (m == -INFINITY ? 0.f : m * scl);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    s[kb][x] = __builtin_amdgcn_exp2f(fmaf(s[kb][x], scl, mc));
                    if (NP > 1) l += s[kb][x];
                }
            __builtin_amdgcn_s_setprio(1);
            // steps: 16 keys from 16 (n / NB), 32 dims from 32 (n % NB)
            const int key = 4 * h + ((lane & 15) >> 2);
            f16x8 vf[kAheadV + 1];
            auto read_v = [&](int n) __attribute__((always_inline)) {
                const int ch = 4 * (n % NB) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                const char *at = vt + (16 * (n / NB) + key) * DP * 2 + (lane & 1) * 8 + ((ch ^ swz_v<DP>(key)) << 4);
                vf[n % (kAheadV + 1)] = join<f16x8>(read_tr<_Float16>(at), read_tr<_Float16>(at + 8 * DP * 2));
            };
#pragma unroll
            for (int n = 0; n < kAheadV; ++n) read_v(n);
            f16x8 pf[NP];
#pragma unroll
            for (int n = 0; n < 4 * NB; ++n) {
                if (n + kAheadV < 4 * NB) read_v(n + kAheadV);
                if (n % NB == 0) {
                    const int kb = n / NB / 2, x = n / NB % 2;
                    uint32_t pw[NP][4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        uint32_t two[NP];
                        pieces2<_Float16, NP>(s[kb][8 * x + 2 * y], s[kb][8 * x + 2 * y + 1], two);
#pragma unroll
                        for (int q = 0; q < NP; ++q) pw[q][y] = two[q];
                        if (NP == 1) l = H::add2(two[0], l);
                    }
#pragma unroll
                    for (int q = 0; q < NP; ++q) pf[q] = as_operand(pw[q][0], pw[q][1], pw[q][2], pw[q][3]);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = NP - 1; q >= 0; --q) o[n % NB] = H::mfma32(vf[n % (kAheadV + 1)], pf[q], o[n % NB]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        pb = pe;
    }
    store_rows<TA, NB>(p, t, kvh, r, h, split, nact > 1, m, scl, 0.25f * l, o);
}

// What a call launches: a few-row launch, a chunk launch or both (as in
// paged_attention.hip).
constexpr int64_t kKeptBytes = (int64_t)64 << 20;  // that a call without a workspace finds kept
struct Plan {
    bool few, chunk;
    bool wide;    // the few-row launch has wide workgroups
    int few_max;  // rows of the longest sequence the few-row launch takes
    int side;     // heads of a few-row workgroup
    int chunk_rows;  // of a tile
    int few_split, few_chunk, chunk_split, chunk_chunk;
    int64_t few_parts, chunk_parts;  // rows of parts
    int64_t part_floats;
};

constexpr int kDecodeWaves = 4, kWideWaves = 8;
constexpr int kWideKeys = 96;  // per wave
constexpr int kAll = INT32_MAX;

Plan make_plan(const PagedAttnDesc &d) {
    Plan pl{};
    const int64_t group = d.heads / d.kv.kv_heads;
    const int64_t rows = d.tokens * group;
    const int64_t cus = device_cu_count();
    // the keys that a row of a tile sees at most
    const int64_t sees = std::max<int64_t>(1, d.window > 0 ? std::min(d.max_kv_len, d.window + 127) : d.max_kv_len);
    pl.few_max = kFewRows;
    // Tiles of 128 rows, or of 16 for all.  Over the same keys the first take about 1.6 times
    // the second's time, of which there are up to eight times as many, and 9 us more for
    // their launches: some 100000 keys of 16 rows, 150000 of up to 64 dims.  (us of a call,
    // 128 / 16, bf16, 32 heads over 8 of 128: 32 sequences of 2 tokens over 4000 keys 112 / 70,
    // of 5 115 / 127; 8 of 5 over 600 24 / 14, of 17 23 / 23, of 33 24 / 31; 1 of 65 over 600
    // 24 / 13, of 33 over 4000 25 / 33.)
    {
        const int64_t seqs = d.kv.num_seqs;
        // in quarters; a sequence's last tile is partly empty
        const int64_t small = std::max(4 * seqs, rows / 4 + 3 * seqs), large = std::max(4 * seqs, rows / 32 + 2 * seqs);
        const int64_t keys = d.kv.kv_heads * (sees * 3 / 4);
        pl.chunk = d.tokens > seqs && keys * (5 * small - 8 * large) > 20 * (d.kv.head_dim <= 64 ? 150000 : 100000);
    }
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
    // Keys per workgroup of the few-row launch.  One round of the workgroups that fit the
    // CUs (three; fp32 q's two make more rounds, of as much workspace; lengths are not all
    // the longest: 3/4), where a row's parts, which are joined one after the other, are then
    // at most 32 of at least 256 keys, or 512 where that leaves every CU one (us of a call,
    // 256 / 512: 16 sequences of up to 2000 25.3 / 23.5, 25 of 1558 under a window of 1112, fp32,
    // 28.3 / 25.4; one of 11476, 20 heads over 5 of 80, 18.9 / 21.2).  Four heads to a workgroup
    // (bf16, 32 heads over 8 of 128: 64 sequences of 1024 .. 4096 keys 77 / one head 88, all
    // of 4096 120 / 124), unless their waves then have few tiles each (16 of 500 .. 2000 keys
    // 29 / 24, one of 16384 32 / 22) or one head needs no second part (256 of 175 .. 700 keys
    // 70 / 64).
    {
        const bool apart = d.tokens == d.kv.num_seqs && 16 % group == 0;  // no row beyond a sequence's first tile
        const int64_t tiles = apart ? d.kv.num_seqs : few_tiles, slots = 3 * cus;
        const int64_t most = tiles * d.kv.kv_heads * sees * 3 / 4;
        int64_t keys = most / slots;
        pl.side = 1;
        if (keys >= 1024 && keys * 3 / 2 < sees)
            while (pl.side < kDecodeWaves && d.kv.kv_heads % (2 * pl.side) == 0) pl.side *= 2;
        keys = std::max<int64_t>({pl.side == 1 && most >= 512 * cus ? 512 : 256, keys / pl.side, sees / 32});
        cut(few_tiles, kAll, keys, 64, pl.few_split, pl.few_chunk);
    }
    pl.wide = pl.few_split > 1 && few_tiles * d.kv.kv_heads <= cus &&
              (d.window > 0 ? std::min(d.max_kv_len, d.window + 15) : d.max_kv_len) <= kWideKeys * kWideWaves;
    if (pl.wide) pl.few_split = pl.side = 1;
    // Tiles of 256 rows, whose codes become f16 once for twice as many rows, where they fill
    // the CUs and walk many keys (us of a call, 128 rows / 256, 32 heads over 8 of 128: 2048
    // tokens over 16384 keys bf16 608 / 550, fp32 942 / 902; over 2048 69 / 70 and 96 / 101; six
    // chunks of up to 700 over a window of 1024, fp32, 74 / 90).
    pl.chunk_rows = rows * d.kv.kv_heads >= 256 * cus && sees >= 4096 ? 256 : 128;
    // One round of them on the keys of their rows (two to a CU of 128 rows), or, where these
    // are cut anyway and the parts are few enough for the stream's kept block, two rounds of
    // half as many keys (or one and a half), which even out better (us of a call, one / two: 59
    // sequences of up to 83 tokens over up to 5136 keys, 16 heads over 4 of 64, fp32, 203 / 169;
    // 11 of 183 over 5536, 32 over 8 of 128, bf16, 146 / 130; what was not cut loses by the
    // join: 6 of 700 under a window of 1024, fp32, 75 / 123).
    const int64_t tiles = rows / pl.chunk_rows + 1, round = 256 / pl.chunk_rows * cus;
    cut(tiles, round, 512, 64, pl.chunk_split, pl.chunk_chunk);
    for (int64_t target : {2 * round, 3 * round / 2}) {
        int nsplit, keys;
        cut(tiles, target, 512, 64, nsplit, keys);
        if (pl.chunk_split == 1 || rows * d.kv.kv_heads * nsplit * (d.kv.head_dim + 2) * 4 > kKeptBytes) continue;
        pl.chunk_split = nsplit, pl.chunk_chunk = keys;
        break;
    }
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

size_t paged_attention_q8_workspace_bytes(const PagedAttnDesc &d) { return (size_t)make_plan(d).part_floats * 4; }

int launch_paged_attention_q8(const PagedAttnDesc &d, const gfh_paged_scales &scales, void *workspace, hipStream_t s) {
    const Plan pl = make_plan(d);
    Q8Params pp{};
    AttnParams &p = pp.a;
    p.c = paged_view(d.kv, d.tokens, d.heads);
    p.q = static_cast<const char *>(d.q);
    p.out = static_cast<char *>(d.out);
    p.ldq = d.ldq, p.ldo = d.ldo;
    p.sc2 = std::fabs(d.scale) * 0x1.715476p+0f;
    p.negate = d.scale < 0.f;
    p.causal = d.causal;
    p.window = d.window >= p.c.capacity ? 0 : (int)d.window;
    pp.ks = scales.k, pp.vs = scales.v;
    pp.scale_page = scales.page_stride, pp.scale_head = scales.head_stride;
    pp.eights = d.kv.page_size % 8 == 0 &&
                ((scales.page_stride | scales.head_stride | (int64_t)(uintptr_t)scales.k | (int64_t)(uintptr_t)scales.v) & 7) == 0;
    pp.side = pl.side;
    const int64_t rows = d.tokens * p.c.group;
    auto run = [&](int bm, int nsplit, int chunk, int64_t parts, int min_rows, int max_rows, auto &&kernel) -> int {
        p.direct = max_rows == kFewRows;
        p.ntiles = p.direct ? kFewTiles * (int)d.kv.num_seqs : (int)((rows - 1) / bm + d.kv.num_seqs);
        p.nsplit = nsplit, p.chunk = chunk, p.min_rows = min_rows, p.max_rows = max_rows;
        p.acc = static_cast<float *>(workspace);
        p.ml = reinterpret_cast<float2 *>(p.acc + parts * nsplit * d.kv.head_dim);
        const int64_t blocks = (int64_t)p.ntiles * (p.c.hkv / (bm == 16 ? pp.side : 1)) * nsplit;
        if (blocks > (int64_t)1 << 23) return set_error(GFH_INVALID_SHAPE, "paged_attention_q8: grid too large");
        kernel(dim3((unsigned)blocks));
        GFH_TRY(check_launch("paged_attention_q8"));
        if (nsplit > 1) {
            const dim3 join((unsigned)(((p.direct ? d.kv.num_seqs * kFewRows * p.c.hkv : d.tokens * d.heads) + 3) / 4));
            if (d.dtype == GFH_F32)
                hipLaunchKernelGGL(paged_join_kernel<float>, join, dim3(256), 0, s, p, bm);
            else if (d.dtype == GFH_BF16)
                hipLaunchKernelGGL(paged_join_kernel<__bf16>, join, dim3(256), 0, s, p, bm);
            else
                hipLaunchKernelGGL(paged_join_kernel<_Float16>, join, dim3(256), 0, s, p, bm);
            GFH_TRY(check_launch("paged_attention_q8 (join)"));
        }
        return GFH_SUCCESS;
    };
    const int64_t hd = d.kv.head_dim;
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    auto by_type = [&](auto &&go) {
        if (d.dtype == GFH_F32)
            go(float{}, Two{});
        else if (d.dtype == GFH_BF16)
            go(__bf16{}, One{});
        else
            go(_Float16{}, One{});
    };
    auto few = [&](dim3 grid) {
        by_type([&](auto ta, auto nq) {
            using TA = decltype(ta);
            constexpr int NQ = decltype(nq)::value;
            auto width = [&](auto dp) {
                constexpr int DP = decltype(dp)::value;
                if (pl.wide)
                    hipLaunchKernelGGL((paged_q8_decode_kernel<TA, DP, NQ, kWideWaves>), grid, dim3(64 * kWideWaves), 0, s, pp);
                else
                    hipLaunchKernelGGL((paged_q8_decode_kernel<TA, DP, NQ, kDecodeWaves>), grid, dim3(64 * kDecodeWaves), 0,
                                       s, pp);
            };
            hd <= 64 ? width(std::integral_constant<int, 64>{}) : width(std::integral_constant<int, 128>{});
        });
    };
    auto many = [&](dim3 grid) {
        by_type([&](auto ta, auto nq) {
            using TA = decltype(ta);
            constexpr int NQ = decltype(nq)::value;
            auto tile = [&](auto dp, auto nd) {
                constexpr int DP = decltype(dp)::value, ND = decltype(nd)::value;
                if (pl.chunk_rows == 256)
                    hipLaunchKernelGGL((paged_q8_chunk_kernel<TA, DP, ND, NQ, 8>), grid, dim3(512), 0, s, pp);
                else
                    hipLaunchKernelGGL((paged_q8_chunk_kernel<TA, DP, ND, NQ, 4>), grid, dim3(256), 0, s, pp);
            };
            using D128 = std::integral_constant<int, 128>;
            if (hd <= 64)
                tile(std::integral_constant<int, 64>{}, Two{});
            else if (hd <= 96)
                tile(D128{}, std::integral_constant<int, 3>{});
            else
                tile(D128{}, std::integral_constant<int, 4>{});
        });
    };
    if (pl.chunk)
        GFH_TRY(run(pl.chunk_rows, pl.chunk_split, pl.chunk_chunk, pl.chunk_parts, pl.few ? pl.few_max + 1 : 0, kAll, many));
    if (pl.few) GFH_TRY(run(16, pl.few_split, pl.few_chunk, pl.few_parts, 0, pl.few_max, few));
    return GFH_SUCCESS;
}

}  // namespace gfh
