// paged_read.hip -- cached rows as dense values: the inverse of the append.
//
// Row t of k_out and v_out is what the cache holds at the position that token t of
// the batch has (paged_kv.hpp), so a batch whose sequences have as many tokens as
// positions reads them whole.  8-bit rows come back as (c - 128) s (paged_quant.hpp),
// exact in fp32 and rounded once to a 16-bit type; other types are converted.
//
// Bound by bytes.  A wave has one token and finds its place once; a lane takes 16
// bytes of the output per step, so that stores cover whole lines, with kAhead steps'
// loads on their way at once.  Stores are nontemporal: nothing reads them here, and lines of
// the cache stay (16 sequences of up to 4096 positions, 8 heads of 128, codes to fp32, 349 MB:
// 51 us, 6.8 TB/s as part of the codes is in the last cache; 512 positions 4.3 us).
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
};

template <typename TC, typename TO>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadParams p) {
    constexpr bool kCodes = std::is_same_v<TC, uint8_t>;
    constexpr int E = 16 / sizeof(TO) < 8 ? 4 : 8, kAhead = 4;
    const int lane = threadIdx.x & 63;
    const int t = __builtin_amdgcn_readfirstlane((int)((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (t >= p.c.tokens) return;
    const int n = paged::wave_leading(p.c.num_seqs + 1, lane, [&](int s) { return p.c.q_offsets[s] <= t; });
    if (n == 0 || n > p.c.num_seqs) return;
    const int s = n - 1;
    const int64_t at = (int64_t)p.c.kv_lens[s] - ((int64_t)p.c.q_offsets[s + 1] - t);
    if (at < 0 || at >= p.c.capacity) {
        if (lane == 0) paged::raise(p.c, paged::kBadLength);
        return;
    }
    const int pos = (int)at, pg = paged::page_of(p.c, pos);
    const int page = p.c.table[s * p.c.table_stride + pg], prow = pos - pg * p.c.page_size;
    const bool ok = page >= 0 && page < p.c.num_pages;
    if (!ok && lane == 0) paged::raise(p.c, paged::kBadPage);
    const int64_t row = page * p.c.page_stride + (int64_t)prow * p.c.row_stride;
    const int per = p.c.d / E, half = p.c.hkv * per;  // units of a head; of k, then as many of v
    for (int u0 = lane; u0 < 2 * half; u0 += 64 * kAhead) {
        float x[kAhead][E];
        TO *to[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int u = min(u0 + 64 * a, 2 * half - 1);
            const bool is_v = u >= half;
            const int uu = is_v ? u - half : u, head = uu / per, dim = (uu - head * per) * E;
            to[a] = reinterpret_cast<TO *>(is_v ? p.v_out : p.k_out) + t * (is_v ? p.ldv : p.ldk) + (int64_t)head * p.c.d + dim;
#pragma unroll
            for (int e = 0; e < E; ++e) x[a][e] = 0.f;
            if (!ok) continue;  // reads as zeros
            const TC *src = reinterpret_cast<const TC *>(is_v ? p.c.v : p.c.k) + row + (int64_t)head * p.c.head_stride + dim;
            if constexpr (kCodes) {
                typedef uint32_t vec __attribute__((ext_vector_type(E / 4)));
                const vec w = *reinterpret_cast<const vec *>(src);
                const float step =
                    paged::step_of((is_v ? p.v_scales : p.k_scales)[page * p.scale_page + head * p.scale_head + prow]);
#pragma unroll
                for (int e = 0; e < E; ++e) x[a][e] = ((float)(w[e / 4] >> (8 * (e % 4)) & 0xff) - 128.f) * step;
            } else {
                load_vec<E>(src, x[a]);
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (u0 + 64 * a < 2 * half) store_vec<E, true>(to[a], x[a]);
    }
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
    const dim3 grid((unsigned)paged_read_blocks(d));
    auto to = [&](auto tc) {
        using TC = decltype(tc);
        if (d.dtype == GFH_F32)
            hipLaunchKernelGGL((paged_read_kernel<TC, float>), grid, dim3(256), 0, s, p);
        else if (d.dtype == GFH_BF16)
            hipLaunchKernelGGL((paged_read_kernel<TC, __bf16>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((paged_read_kernel<TC, _Float16>), grid, dim3(256), 0, s, p);
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
