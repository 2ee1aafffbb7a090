// paged_append_norm.hip -- the append of paged_append.hip with norms of queries and
// keys on the way, and into a cache of 8 bits (paged_quant.hpp).
//
// For a head's dims x of a query or key, with weights w:
//   r = 1 / sqrt(mean(x^2) + eps),  y = (x r) w
// then the rotation of paged_append.hip on y, rounded once to q's or the cache's
// type, or turned into codes.  The sum of squares is taken in fp64 and r rounded to
// fp32, so it does not depend on the order of the sum; y and the rotation round every
// fp32 operation by itself (no contraction), so codes do not depend on the compiler.
//
// A head lies in a group of lanes (a power of two) that holds all its dims in
// registers: the norm and the largest magnitude are a few lane swaps each, and
// everything is read and written once.
//
// Bound by bytes where there are many tokens (16000 of 32 heads over 8 of 128, fp32 into
// codes: 73 to 77 us; 20000 of 16 over 4, bf16 with norms: 145 MB in 36 us, 4.0 TB/s), by the way
// from offsets to length to page where there are few (64 tokens 5.5 us).  A wave's values are
// on their way while it finds its page (after it: 38.5 instead of 36.4 us).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "paged_quant.hpp"
#include "paged_types.hpp"

namespace gfh {
namespace {

using paged::View;

struct AppendNormParams {
    View c;
    const char *q, *k, *v;
    char *q_out;
    int64_t ldq, ldqo, ldk, ldv;  // elements between tokens
    const float *cos, *sin;
    const float *q_norm, *k_norm;
    double eps, inv_d;
    uint8_t *k_scales, *v_scales;
    int64_t scale_page, scale_head;  // bytes between pages, heads; rows are adjacent
    int rot;  // rotated dims R, 0 without tables
    int interleaved;
    int units;  // of a head
    int shift;  // log2 of a head's lanes
    int waves;  // per token
};

// x over a group of 2^shift lanes (at most 16) in every lane of it; swaps of
// neighbours, pairs, quads (mirrored) and halves of 16
template <typename T, typename F>
__device__ __forceinline__ T over_group(T x, int shift, F &&f) {
    auto swapped = [](T v, auto ctrl) __attribute__((always_inline)) {
        constexpr int C = decltype(ctrl)::value;
        if constexpr (sizeof(T) == 8) {
            const uint64_t u = __builtin_bit_cast(uint64_t, v);
            const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, C, 0xf, 0xf, false);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), C, 0xf, 0xf, false);
            return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
        } else {
            return dpp_mov<C>(v);
        }
    };
    if (shift > 0) x = f(x, swapped(x, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
    if (shift > 1) x = f(x, swapped(x, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
    if (shift > 2) x = f(x, swapped(x, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    if (shift > 3) x = f(x, swapped(x, std::integral_constant<int, 0x140>{}));  // row_mirror
    return x;
}

template <int W>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&x)[W], float step) {
    static_assert(W % 4 == 0);
    typedef uint32_t vec __attribute__((ext_vector_type(W / 4)));
    vec v;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= paged::code_of(x[4 * i + e], step) << (8 * e);
        v[i] = w;
    }
    *reinterpret_cast<vec *>(p) = v;
}

// N elements on their way: loaded here, fp32 when they are first needed.
template <typename T, int N>
struct Run {
    static constexpr int kPer = N * sizeof(T) <= 16 ? N : 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kPer)));
    vec v[N / kPer] = {};

    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N / kPer; ++i) v[i] = reinterpret_cast<const vec *>(p)[i];
    }
    __device__ __forceinline__ void values(float (&x)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)v[i / kPer][i % kPer];
    }
};

// W pairs: 2 W elements of a head.  TA: activations, TC: cache (uint8_t: codes).
template <typename TA, typename TC, int W>
__global__ __launch_bounds__(256) void paged_append_norm_kernel(AppendNormParams p) {
#pragma clang fp contract(off)
    constexpr bool kCodes = std::is_same_v<TC, uint8_t>;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int t = wave / p.waves, part = wave % p.waves;
    if (t >= p.c.tokens) return;
    // (lanes without a unit go along with zeros: their group's swaps need them)
    const int heads_per = 64 >> p.shift, i = lane & ((1 << p.shift) - 1);
    const int head = part * heads_per + (lane >> p.shift);  // heads of q, then k, then v
    const int hq = p.q ? p.c.heads : 0;
    const bool live = head < hq + 2 * p.c.hkv && i < p.units;
    const bool is_q = head < hq, is_v = head >= hq + p.c.hkv;
    const int kvh = is_q ? 0 : is_v ? head - hq - p.c.hkv : head - hq;
    const TA *src;
    if (is_q)
        src = reinterpret_cast<const TA *>(p.q) + t * p.ldq + (int64_t)head * p.c.d;
    else if (is_v)
        src = reinterpret_cast<const TA *>(p.v) + t * p.ldv + (int64_t)kvh * p.c.d;
    else
        src = reinterpret_cast<const TA *>(p.k) + t * p.ldk + (int64_t)kvh * p.c.d;
    const int rot = is_v ? 0 : p.rot, turned = rot / (2 * W);  // units that are turned
    const bool turn = i < turned;
    // the unit's two runs of W elements
    const bool split = turn && !p.interleaved;
    const int a0 = split ? i * W : i * 2 * W, b0 = split ? a0 + rot / 2 : a0 + W;
    const float *const norm = is_v ? nullptr : is_q ? p.q_norm : p.k_norm;
    // what does not go by the position is on its way while that is found
    Run<TA, W> raw_a, raw_b;
    Run<float, W> weight_a, weight_b, raw_c, raw_s;
    if (live) {
        raw_a.load(src + a0);
        raw_b.load(src + b0);
        if (norm) {
            weight_a.load(norm + a0);
            weight_b.load(norm + b0);
        }
    }
    const int n = paged::wave_leading(p.c.num_seqs + 1, lane, [&](int s) { return p.c.q_offsets[s] <= t; });
    if (n == 0 || n > p.c.num_seqs) return;  // before the first or behind the last sequence: left as it is
    const int s = n - 1;
    // position: counted from the sequence's end
    const int64_t at = (int64_t)p.c.kv_lens[s] - ((int64_t)p.c.q_offsets[s + 1] - t);
    if (at < 0 || at >= p.c.capacity) {
        if (lane == 0) paged::raise(p.c, paged::kBadLength);
        return;
    }
    const int pos = (int)at;
    if (live && turn) {
        raw_c.load(p.cos + (int64_t)pos * (rot / 2) + i * W);
        raw_s.load(p.sin + (int64_t)pos * (rot / 2) + i * W);
    }
    const int pg = paged::page_of(p.c, pos);
    const int page = p.c.table[s * p.c.table_stride + pg], prow = pos - pg * p.c.page_size;
    const bool page_ok = page >= 0 && page < p.c.num_pages;
    if (!page_ok && lane == 0) paged::raise(p.c, paged::kBadPage);

    float a[W], b[W], c[W], sn[W];
    raw_a.values(a);
    raw_b.values(b);
    raw_c.values(c);
    raw_s.values(sn);
    if (p.q_norm || p.k_norm) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < W; ++e) sum += (double)a[e] * a[e] + (double)b[e] * b[e];
        sum = over_group(sum, p.shift, [](double x, double y) { return x + y; });
        if (live && norm) {
            const float r = (float)rsqrt(fma(sum, p.inv_d, p.eps));
            float wa[W], wb[W];
            weight_a.values(wa);
            weight_b.values(wb);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                a[e] = a[e] * r * wa[e];
                b[e] = b[e] * r * wb[e];
            }
        }
    }
    if (turn && live) {
        if (split) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float x = a[e], y = b[e];
                a[e] = x * c[e] - y * sn[e];
                b[e] = y * c[e] + x * sn[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                // pair e: elements 2e, 2e + 1 of the unit's 2 W
                float &x = 2 * e < W ? a[(2 * e) % W] : b[(2 * e) % W];
                float &y = 2 * e < W ? a[(2 * e + 1) % W] : b[(2 * e + 1) % W];
                const float xv = x, yv = y;
                x = xv * c[e] - yv * sn[e];
                y = yv * c[e] + xv * sn[e];
            }
        }
    }
    float most = 0.f;
    if constexpr (kCodes) {
        bool finite = true;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            most = fmaxf(most, fmaxf(fabsf(a[e]), fabsf(b[e])));
            finite = finite && fabsf(a[e]) <= 127.f * 120.f && fabsf(b[e]) <= 127.f * 120.f;
        }
        most = over_group(most, p.shift, [](float x, float y) { return fmaxf(x, y); });
        if (!finite && live && !is_q) paged::raise(p.c, paged::kBadValue);
    }
    if (!live) return;
    if (is_q) {
        TA *dst = reinterpret_cast<TA *>(p.q_out) + t * p.ldqo + (int64_t)head * p.c.d;
        store_vec<W>(dst + a0, a);
        store_vec<W>(dst + b0, b);
    } else if (page_ok) {
        TC *dst = reinterpret_cast<TC *>(is_v ? p.c.v : p.c.k) + page * p.c.page_stride + (int64_t)prow * p.c.row_stride +
                  (int64_t)kvh * p.c.head_stride;
        if constexpr (kCodes) {
            const int byte = paged::step_byte(most);
            const float step = paged::step_of(byte);
            store_codes<W>(dst + a0, a, step);
            store_codes<W>(dst + b0, b, step);
            if (i == 0) (is_v ? p.v_scales : p.k_scales)[page * p.scale_page + kvh * p.scale_head + prow] = (uint8_t)byte;
        } else {
            store_vec<W>(dst + a0, a);
            store_vec<W>(dst + b0, b);
        }
    }
}

// 8 pairs per lane (16-byte loads of 16-bit types) where the head allows
bool wide_units(const PagedAppendDesc &d) { return d.kv.head_dim % 16 == 0 && (!d.cos || d.rotary_dim % 16 == 0); }
int units_of(const PagedAppendDesc &d) { return (int)d.kv.head_dim / (wide_units(d) ? 16 : 8); }
int shift_of(const PagedAppendDesc &d) {
    int s = 0;
    while ((1 << s) < units_of(d)) ++s;
    return s;
}
int64_t waves_of(const PagedAppendDesc &d) {
    const int64_t per = 64 >> shift_of(d);
    return ((d.q ? d.heads : 0) + 2 * d.kv.kv_heads + per - 1) / per;
}

}  // namespace

int64_t paged_append_norm_blocks(const PagedAppendDesc &d) { return (d.tokens * waves_of(d) + 3) / 4; }

int launch_paged_append_norm(const PagedAppendDesc &d, const PagedNormDesc &n, hipStream_t s) {
    AppendNormParams p{};
    p.c = paged_view(d.kv, d.tokens, d.heads);
    p.q = static_cast<const char *>(d.q);
    p.k = static_cast<const char *>(d.k);
    p.v = static_cast<const char *>(d.v);
    p.q_out = static_cast<char *>(d.q_out);
    p.ldq = d.ldq, p.ldqo = d.ldqo, p.ldk = d.ldk, p.ldv = d.ldv;
    p.cos = d.cos, p.sin = d.sin;
    p.q_norm = n.q_norm, p.k_norm = n.k_norm, p.eps = n.eps;
    p.inv_d = 1.0 / (double)d.kv.head_dim;
    p.k_scales = n.scales.k, p.v_scales = n.scales.v;
    p.scale_page = n.scales.page_stride, p.scale_head = n.scales.head_stride;
    p.rot = d.cos ? (int)d.rotary_dim : 0;
    p.interleaved = d.interleaved;
    p.units = units_of(d);
    p.shift = shift_of(d);
    p.waves = (int)waves_of(d);
    const dim3 grid((unsigned)paged_append_norm_blocks(d));
    auto go = [&](auto ta, auto tc) {
        using TA = decltype(ta);
        using TC = decltype(tc);
        if (wide_units(d))
            hipLaunchKernelGGL((paged_append_norm_kernel<TA, TC, 8>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((paged_append_norm_kernel<TA, TC, 4>), grid, dim3(256), 0, s, p);
    };
    if (d.kv.dtype == GFH_U8) {
        if (d.dtype == GFH_F32)
            go(float{}, uint8_t{});
        else if (d.dtype == GFH_BF16)
            go(__bf16{}, uint8_t{});
        else
            go(_Float16{}, uint8_t{});
    } else if (d.dtype == GFH_F32)
        d.kv.dtype == GFH_F32 ? go(float{}, float{}) : go(float{}, __bf16{});
    else if (d.dtype == GFH_BF16)
        go(__bf16{}, __bf16{});
    else
        go(_Float16{}, _Float16{});
    return check_launch("paged_append_norm");
}

}  // namespace gfh
