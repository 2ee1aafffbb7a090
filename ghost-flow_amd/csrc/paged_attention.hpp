// paged_attention.hpp -- what the attention kernels over a paged cache share: a
// workgroup's rows and keys, the parts of split rows, pieces of 16-bit types.
#pragma once

#include <climits>

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

template <typename T>
__device__ __forceinline__ typename Half<T>::v4 read_tr(const char *lds) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(typename Half<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                        (__attribute__((address_space(3))) s4 *)(lds)));
}
template <typename V8, typename V4>
__device__ __forceinline__ V8 join(V4 a, V4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
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

// The states that `waves` waves have of a 16-row tile from LDS (rows of DP + 4 floats, their
// maximum and sum) to the tile's rows: their thread i takes 4 dims of a row.
template <typename TA, int DP>
__device__ __forceinline__ void join_waves(const AttnParams &p, const Rows &t, int kvh, int split, bool parts,
                                           const float *accs, const float2 *mls, int waves, int tid) {
    constexpr int kRow = DP + 4;
    for (int i = tid; i < 16 * DP / 4; i += 64 * waves) {
        const int row = i / (DP / 4), dim = 4 * (i % (DP / 4));
        const int rr = t.base + row;
        if (rr < t.r0 || rr >= t.r1 || dim >= p.c.d) continue;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < waves; ++w) M = max_nan(M, mls[w * 16 + row].x);
        f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < waves; ++w) {
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

// Row r of a chunk tile (lane half h holds dims 32 i + 8 x + 4 h .. + 3) to out or
// to the parts.
template <typename TA, int NB>
__device__ __forceinline__ void store_rows(const AttnParams &p, const Rows &t, int kvh, int r, int h, int split,
                                           bool parts, float m, float sc2, float l, const f32x16 (&o)[NB]) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if (r < t.r0 || r >= t.r1) return;
    const int64_t at = parts ? part_row(p, t, r, kvh) * p.nsplit + split : 0;
    const float f = parts ? 1.f : m == -INFINITY ? 0.f : 1.0f / l;
    if (parts && h == 0) p.ml[at] = make_float2(m == -INFINITY ? m : m * sc2, l);
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

}  // namespace
}  // namespace gfh
