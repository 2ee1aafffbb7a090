// paged_append.hip -- new keys and values into their pages, with the rotary
// positions applied on the way, and the queries rotated by the same angles.
//
// For the pair (a, b) = (x[j], x[j + R/2]) of a head's first R dims (half
// split), or (x[2j], x[2j + 1]) (interleaved), at position p:
//   a' = a cos[p, j] - b sin[p, j]      b' = b cos[p, j] + a sin[p, j]
// in fp32 and rounded once to the output's type; dims from R on, and v, are
// copied.  cos / sin are fp32 tables of the positions, so far positions lose
// nothing to an angle held in 32 bits.
//
// Bound by bytes (every value read and written once) for a prompt (412 MB in 76 us,
// 5.4 TB/s), by the chain offsets -> length -> table / angles -> store for a decode
// step (64 tokens: 3.8 us).  A thread holds W pairs, so that both halves of a
// rotated unit are one vector load each; a wave's 64 units are of one token, whose
// sequence the wave finds with one round of loads (paged_kv.hpp).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "paged_types.hpp"

namespace gfh {
namespace {

using paged::View;

struct AppendParams {
    View c;
    const char *q, *k, *v;
    char *q_out;
    int64_t ldq, ldqo, ldk, ldv;  // elements between tokens
    const float *cos, *sin;
    int rot;  // rotated dims R, 0 without tables
    int interleaved;
    int units;  // per head
    int waves;  // per token
};

// W pairs: 2 W elements of a head.  TA: activations, TC: cache.
template <typename TA, typename TC, int W>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int t = wave / p.waves, part = wave % p.waves;
    if (t >= p.c.tokens) return;
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
    const int page = p.c.table[s * p.c.table_stride + paged::page_of(p.c, pos)];
    const bool page_ok = page >= 0 && page < p.c.num_pages;
    if (!page_ok && lane == 0) paged::raise(p.c, paged::kBadPage);
    const int64_t row =
        page * p.c.page_stride + (int64_t)(pos - paged::page_of(p.c, pos) * p.c.page_size) * p.c.row_stride;

    const int u = part * 64 + lane;
    const int hq = p.q ? p.c.heads : 0;
    const int head = u / p.units, i = u - head * p.units;  // heads of q, then k, then v
    if (head >= hq + 2 * p.c.hkv) return;
    const bool is_q = head < hq, is_v = head >= hq + p.c.hkv;
    const TA *src;
    if (is_q)
        src = reinterpret_cast<const TA *>(p.q) + t * p.ldq + (int64_t)head * p.c.d;
    else if (is_v)
        src = reinterpret_cast<const TA *>(p.v) + t * p.ldv + (int64_t)(head - hq - p.c.hkv) * p.c.d;
    else
        src = reinterpret_cast<const TA *>(p.k) + t * p.ldk + (int64_t)(head - hq) * p.c.d;
    const int rot = is_v ? 0 : p.rot, turned = rot / (2 * W);  // units that are turned
    const bool turn = i < turned;
    // the unit's two runs of W elements
    const bool split = turn && !p.interleaved;
    const int a0 = split ? i * W : i * 2 * W, b0 = split ? a0 + rot / 2 : a0 + W;
    float a[W], b[W];
    load_vec<W>(src + a0, a);
    load_vec<W>(src + b0, b);
    if (turn) {
        float c[W], sn[W];
        load_vec<W>(p.cos + (int64_t)pos * (rot / 2) + i * W, c);
        load_vec<W>(p.sin + (int64_t)pos * (rot / 2) + i * W, sn);
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
    if (is_q) {
        TA *dst = reinterpret_cast<TA *>(p.q_out) + t * p.ldqo + (int64_t)head * p.c.d;
        store_vec<W>(dst + a0, a);
        store_vec<W>(dst + b0, b);
    } else if (page_ok) {
        TC *dst = reinterpret_cast<TC *>(is_v ? p.c.v : p.c.k) + row +
                  (int64_t)(is_v ? head - hq - p.c.hkv : head - hq) * p.c.head_stride;
        store_vec<W>(dst + a0, a);
        store_vec<W>(dst + b0, b);
    }
}

// 8 pairs per thread (16-byte loads of 16-bit types) where the head allows
bool wide_units(const PagedAppendDesc &d) { return d.kv.head_dim % 16 == 0 && (!d.cos || d.rotary_dim % 16 == 0); }
int units_of(const PagedAppendDesc &d) { return (int)d.kv.head_dim / (wide_units(d) ? 16 : 8); }
int64_t waves_of(const PagedAppendDesc &d) {
    return (((d.q ? d.heads : 0) + 2 * d.kv.kv_heads) * units_of(d) + 63) / 64;
}

}  // namespace

int64_t paged_append_blocks(const PagedAppendDesc &d) { return (d.tokens * waves_of(d) + 3) / 4; }

int launch_paged_append(const PagedAppendDesc &d, hipStream_t s) {
    AppendParams p{};
    p.c = paged_view(d.kv, d.tokens, d.heads);
    p.q = static_cast<const char *>(d.q);
    p.k = static_cast<const char *>(d.k);
    p.v = static_cast<const char *>(d.v);
    p.q_out = static_cast<char *>(d.q_out);
    p.ldq = d.ldq, p.ldqo = d.ldqo, p.ldk = d.ldk, p.ldv = d.ldv;
    p.cos = d.cos, p.sin = d.sin;
    p.rot = d.cos ? (int)d.rotary_dim : 0;
    p.interleaved = d.interleaved;
    const bool wide = wide_units(d);
    p.units = units_of(d);
    p.waves = (int)waves_of(d);
    const dim3 grid((unsigned)paged_append_blocks(d));
    auto go = [&](auto ta, auto tc) {
        using TA = decltype(ta);
        using TC = decltype(tc);
        if (wide)
            hipLaunchKernelGGL((paged_append_kernel<TA, TC, 8>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((paged_append_kernel<TA, TC, 4>), grid, dim3(256), 0, s, p);
    };
    if (d.dtype == GFH_F32)
        d.kv.dtype == GFH_F32 ? go(float{}, float{}) : go(float{}, __bf16{});
    else if (d.dtype == GFH_BF16)
        go(__bf16{}, __bf16{});
    else
        go(_Float16{}, _Float16{});
    return check_launch("paged_append");
}

}  // namespace gfh
