// paged_read.hip -- cached rows as dense values: the inverse of the append.
//
// Row t of k_out and v_out is what the cache holds at the position that token t of
// the batch has (paged_kv.hpp), so a batch whose sequences have as many tokens as
// positions reads them whole.  8-bit rows come back as (c - 128) s (paged_quant.hpp),
// exact in fp32 and rounded once to a 16-bit type; other types are converted.
//
// Bound by bytes.  A wave has one token, or up to four of few heads, and finds their
// places once; a lane takes 16 bytes of the output per step, so that stores cover whole
// lines, with kAhead steps' loads on their way at once.  Stores are nontemporal: nothing
// reads them here, and lines of the cache stay (16 sequences of up to 4096 positions, 8
// heads of 128, codes to fp32, 349 MB: 52 us, 6.7 TB/s as part of the codes is in the last
// cache; 512 positions 4.0 us).
#include "common.hpp"
#include "kernels.hpp"
#include "paged_kv.hpp"
#include "paged_quant.hpp"
#include "paged_types.hpp"

namespace gfh {
namespace {

using paged::View;

struct ReadParams {
    View c;
    char *k_out, *v_out;
    int64_t ldk, ldv;  // elements between tokens
    const uint8_t *k_scales, *v_scales;
    int64_t scale_page, scale_head;
    int each;  // tokens of a wave, neighbours: 1, 2 or 4
};

// MANY: up to four tokens to a wave, p.each.
template <typename TC, typename TO, bool MANY>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadParams p) {
    constexpr bool kCodes = std::is_same_v<TC, uint8_t>;
    constexpr int E = 16 / sizeof(TO) < 8 ? 4 : 8, kAhead = 4;
    const int lane = threadIdx.x & 63;
    const int t0 = __builtin_amdgcn_readfirstlane((int)(((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (MANY ? p.each : 1)));
    if (t0 >= p.c.tokens) return;
    // the tokens' places; a neighbour's is mostly in the same sequence, which is known
    constexpr int kMost = MANY ? 4 : 1;
    int live = 0, ok = 0;  // a bit for each
    int pages[kMost], prow[kMost];
    int64_t row[kMost], steps[kMost];
    int n = 0, next = 0, len = 0;  // sequences from the first that begin up to a token; where the nth begins
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int t = t0 + j;
        pages[j] = -1, prow[j] = 0;
        if (j > 0 && (j >= p.each || t >= p.c.tokens)) continue;
        if (j == 0 || (n <= p.c.num_seqs && next <= t)) {
            n = paged::wave_leading(p.c.num_seqs + 1, lane, [&](int s) { return p.c.q_offsets[s] <= t; });
            next = p.c.q_offsets[min(n, p.c.num_seqs)];
            len = p.c.kv_lens[min(max(n, 1), p.c.num_seqs) - 1];
        }
        if (n == 0 || n > p.c.num_seqs) continue;  // before the first or behind the last sequence
        const int64_t at = (int64_t)len - ((int64_t)next - t);
        if (at < 0 || at >= p.c.capacity) {
            if (lane == 0) paged::raise(p.c, paged::kBadLength);
            continue;
        }
        live |= 1 << j;
        const int pos = (int)at, pg = paged::page_of(p.c, pos);
        pages[j] = p.c.table[(n - 1) * p.c.table_stride + pg], prow[j] = pos - pg * p.c.page_size;
    }
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int page = __builtin_amdgcn_readfirstlane(pages[j]);
        const bool in = page >= 0 && page < p.c.num_pages;
        if (!in && (live >> j & 1) && lane == 0) paged::raise(p.c, paged::kBadPage);
        ok |= (int)in << j;
        row[j] = page * p.c.page_stride + (int64_t)prow[j] * p.c.row_stride;
        steps[j] = page * p.scale_page + prow[j];
    }
    const int per = p.c.d / E, half = p.c.hkv * per;  // units of a head; of k, then as many of v
    const int units = 2 * half * (MANY ? p.each : 1);
    // (by value: an index that is not constant would put the four into memory)
    auto of = [](int64_t a, int64_t b, int64_t c, int64_t d, int j) { return j & 2 ? j & 1 ? d : c : j & 1 ? b : a; };
    constexpr int k1 = MANY ? 1 : 0, k2 = MANY ? 2 : 0, k3 = MANY ? 3 : 0;
    typedef TC raw __attribute__((ext_vector_type(E), aligned(E * sizeof(TC) < 16 ? E * sizeof(TC) : 16)));
    for (int u0 = lane; u0 < units; u0 += 64 * kAhead) {
        raw v[kAhead];
        uint32_t bytes[kAhead];
        TO *to[kAhead];
        // (nothing that is loaded is looked at before all is on its way)
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            // (of one token the last again: every lane then loads, or none)
            const int all = MANY ? u0 + 64 * a : min(u0 + 64 * a, units - 1), j = MANY ? (all >= 2 * half) + (all >= 4 * half) + (all >= 6 * half) : 0,
                      u = all - 2 * half * j;
            const bool here = u0 + 64 * a < units && live >> j & 1, good = (!MANY || all < units) && ok >> j & 1;
            const bool is_v = u >= half;
            const int uu = is_v ? u - half : u, head = uu / per, dim = (uu - head * per) * E;
            to[a] = reinterpret_cast<TO *>(is_v ? p.v_out : p.k_out) + (t0 + j) * (is_v ? p.ldv : p.ldk) +
                    (int64_t)head * p.c.d + dim;
            if (!here) to[a] = nullptr;
            v[a] = raw(kCodes ? (TC)128 : (TC)0);  // a page outside the cache reads as zeros
            bytes[a] = 0;
            if (good) {
                const int64_t at = of(row[0], row[k1], row[k2], row[k3], j);
                v[a] = *reinterpret_cast<const raw *>(reinterpret_cast<const TC *>(is_v ? p.c.v : p.c.k) + at +
                                                      (int64_t)head * p.c.head_stride + dim);
                if constexpr (kCodes) {
                    const int64_t step = of(steps[0], steps[k1], steps[k2], steps[k3], j);
                    bytes[a] = (is_v ? p.v_scales : p.k_scales)[step + head * p.scale_head];
                }
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (!to[a]) continue;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e)
                x[e] = kCodes ? ((float)v[a][e] - 128.f) * paged::step_of(bytes[a]) : (float)v[a][e];
            store_vec<E, true>(to[a], x);
        }
    }
}

// Tokens of a wave: as many as its four steps of 64 lanes hold, where there are enough
// waves all the same: each has the way from offsets to length to page before it (33000 tokens
// of 4 heads of 64, codes to bf16: one to a wave 27 us, four 15; of 8 heads of 128 one is as
// good).
int tokens_each(const PagedReadDesc &d) {
    const int64_t units = 2 * d.kv.kv_heads * d.kv.head_dim / (d.dtype == GFH_F32 ? 4 : 8);
    return d.tokens < 8192 ? 1 : units <= 64 ? 4 : units <= 128 ? 2 : 1;
}

}  // namespace

int launch_paged_read(const PagedReadDesc &d, hipStream_t s) {
    ReadParams p{};
    p.c = paged_view(d.kv, d.tokens, d.kv.kv_heads);
    p.k_out = static_cast<char *>(d.k_out);
    p.v_out = static_cast<char *>(d.v_out);
    p.ldk = d.ldk, p.ldv = d.ldv;
    p.k_scales = d.scales.k, p.v_scales = d.scales.v;
    p.scale_page = d.scales.page_stride, p.scale_head = d.scales.head_stride;
    p.each = tokens_each(d);
    const dim3 grid((unsigned)((d.tokens + 4 * p.each - 1) / (4 * p.each)));
    auto to = [&](auto tc) {
        auto as = [&](auto out) {
            using TC = decltype(tc);
            using TO = decltype(out);
            if (p.each > 1)
                hipLaunchKernelGGL((paged_read_kernel<TC, TO, true>), grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((paged_read_kernel<TC, TO, false>), grid, dim3(256), 0, s, p);
        };
        if (d.dtype == GFH_F32)
            as(float{});
        else if (d.dtype == GFH_BF16)
            as(__bf16{});
        else
            as(_Float16{});
    };
    if (d.kv.dtype == GFH_U8)
        to(uint8_t{});
    else if (d.kv.dtype == GFH_F32)
        to(float{});
    else if (d.kv.dtype == GFH_BF16)
        to(__bf16{});
    else
        to(_Float16{});
    return check_launch("paged_read");
}

}  // namespace gfh
