// w4.hip -- weights of 4 bits in groups: to codes and back, and Linear on them.
//
// A weight W [n, k] is held as codes c [n, k / 2] (two per byte, the even
// column in the low four bits), one fp32 scale per group of `group` columns of
// a row and, if it is asymmetric, one zero point byte per group:
//   W'[i, j] = (c - z) s,   z = 8 where there are no zero points
//   symmetric:  s = max|w| (1/7),                 c = clamp(round(w / s), -8, 7) + 8
//   asymmetric: s = (max(w, 0) - min(w, 0)) (1/15), z = clamp(round(-min(w, 0) / s), 0, 15),
//               c = clamp(round(w / s) + z, 0, 15)
// the int8 scheme (quant_math.hpp: IEEE division by s, round half away from
// zero, NaN counts as 0) on 16 levels, with 0 among them; 1/7 and 1/15 are the
// fp32 constants; a group without a range has s = 1.
//
// Linear: y[m, n] = sum over groups g of s[n, g] sum over j in g of x[m, j]
// (c[n, j] - z[n, g]) + bias[n].  A code becomes an f16 exactly: 0x6400 | c is
// 1024 + c (0x6400 | c << 4 is 1024 + 16 c), and one packed f16 operation takes
// 1024 + z off, nine instructions for eight codes.  The scale multiplies a
// group's finished sum in fp32.  Three kernels: VALU for one or two rows of x (fp32:
// four), a stream of W for up to 16 rows of 16 bits, tiles for the rest.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "paged_types.hpp"
#include "quant_math.hpp"

namespace gfh {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- to codes and back ----------------------------------------------------------

#pragma clang fp contract(off)

struct W4Params {
    const float *w;
    uint8_t *codes;
    float *scales;
    uint8_t *zps;
    float *out;
    int64_t n, k, groups;
    int group;
    int lanes, lane_bits;  // per group (a power of two up to 64), and its logarithm
};

__device__ __forceinline__ void w4_params(float lo, float hi, bool asym, float &s, int &z) {
    z = 8;
    if (asym) {
        lo = fminf(lo, 0.f), hi = fmaxf(hi, 0.f);
        s = (hi - lo) * (1.0f / 15.0f);
        if (s == 0.f) s = 1.f;
        z = min(max(qmath::sat_f32_to_i32(roundf(-lo / s)), 0), 15);
    } else {
        s = fmaxf(fabsf(lo), fabsf(hi)) * (1.0f / 7.0f);
        if (s == 0.f) s = 1.f;
    }
}
__device__ __forceinline__ uint32_t w4_code(float w, float s, int z) {
    const int q = qmath::sat_f32_to_i32(roundf(w / s));
    return (uint32_t)min(max(min(max(q, -16), 16) + z, 0), 15);
}

// Eight codes.  round(w / s) is round(w (1 / s)) wherever the product is further
// from a tie than the two can be apart: up to 16.5, where codes end, each of the
// reciprocal, the product, the sum with 1/2 and w / s itself is off by less than
// 2^-19.9 -- under 2^-17 together.  Where one of a wave's is nearer than 2^-16 (or
// NaN, infinite, or s is so far from 1 that 1 / s is inexact), all divide.
__device__ __forceinline__ uint32_t w4_codes(const float (&v)[8], float s, float inv, bool plain, int z) {
    uint32_t c = 0;
    bool near = !plain;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float t = v[e] * inv, a = fabsf(t) + 0.5f, f = floorf(a);
        near |= !(fabsf(a - f - 0.5f) < 0.5f - 0x1p-16f);
        const int q = (int)copysignf(fminf(f, 16.f), t);
        c |= (uint32_t)min(max(q + z, 0), 15) << (4 * e);
    }
    if (__any(near)) {
        c = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) c |= w4_code(v[e], s, z) << (4 * e);
    }
    return c;
}

// A group's 8-column units over `lanes` lanes (several each where the group is
// longer), fp32 in, four code bytes per unit out.  Bound by bytes once most codes
// go without a division (4096 x 4096: 17.2 us for 76 MB, 4.4 TB/s, against 21.7 with
// one for every code).
__global__ __launch_bounds__(256) void quantize_w4_kernel(W4Params p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t gi = id >> p.lane_bits, all = p.n * p.groups;
    const int sub = (int)id & (p.lanes - 1);
    const bool ok = gi < all;
    int64_t row = 0, g = 0;
    if (ok) {
        row = all <= UINT32_MAX ? (uint32_t)gi / (uint32_t)p.groups : gi / p.groups;
        g = gi - row * p.groups;
    }
    const int64_t j0 = g * p.group, j1 = min(j0 + p.group, p.k);
    const float *w = p.w + row * p.k;
    float lo = INFINITY, hi = -INFINITY, v[8];
    const bool one = p.group <= 8 * p.lanes;  // the unit stays in registers
    for (int64_t j = j0 + 8 * sub; ok && j < j1; j += 8 * p.lanes) {
        load_vec<8>(w + j, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) lo = fminf(lo, v[e]), hi = fmaxf(hi, v[e]);
    }
    for (int o = p.lanes >> 1; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor(lo, o));
        hi = fmaxf(hi, __shfl_xor(hi, o));
    }
    if (!ok) return;
    if (!(lo <= hi)) lo = hi = 0.f;  // nothing but NaN
    float s;
    int z;
    w4_params(lo, hi, p.zps != nullptr, s, z);
    const float inv = 1.0f / s;
    const bool plain = s > 0x1p-100f && s < 0x1p100f;
    for (int64_t j = j0 + 8 * sub; j < j1; j += 8 * p.lanes) {
        if (!one) load_vec<8>(w + j, v);
        *reinterpret_cast<uint32_t *>(p.codes + (row * p.k + j) / 2) = w4_codes(v, s, inv, plain, z);
    }
    if (sub == 0) {
        p.scales[gi] = s;
        if (p.zps) p.zps[gi] = (uint8_t)z;
    }
}

// Eight columns per thread and turn.  Bound by bytes (4096 x 4096: 15.4 us, 76 MB).
__global__ __launch_bounds__(256) void dequantize_w4_kernel(W4Params p) {
    const int64_t units = p.n * (p.k / 8);
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < units; id += (int64_t)gridDim.x * 256) {
        const int64_t row = units <= UINT32_MAX ? (uint32_t)id / (uint32_t)(p.k / 8) : id / (p.k / 8);
        const int64_t j = (id - row * (p.k / 8)) * 8;
        const int64_t gi = row * p.groups + (uint32_t)j / (uint32_t)p.group;
        const uint32_t c = reinterpret_cast<const uint32_t *>(p.codes)[id];
        const float s = p.scales[gi];
        const int z = p.zps ? p.zps[gi] : 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)((int)((c >> (4 * e)) & 15) - z) * s;
        store_vec<8>(p.out + id * 8, v);
    }
}

#pragma clang fp contract(on)

// ---- Linear -----------------------------------------------------------------------

struct W4LinearParams {
    const void *x;
    const uint8_t *codes;
    const float *scales;
    const uint8_t *zps;
    const void *bias;
    void *y;
    float *part;  // [splits][m][n] where K is split
    int64_t ldx, ldy;
    int m, n, k, group, groups;
    int kper;   // columns per split
    int splits;
    int steps;       // 32-column steps per group (more than there are: one group)
    uint32_t magic;  // 2^32 / steps + 1 (see w4_streams)
};

// Eight codes as f16 pairs (0, 4), (1, 5), (2, 6), (3, 7), z taken off.
struct Zero {
    f16x2 a, b;  // 1024 + z, -(64 + z)
    __device__ __forceinline__ explicit Zero(uint32_t z) {
        z |= z << 16;
        a = __builtin_bit_cast(f16x2, 0x64006400u | z);
        b = __builtin_bit_cast(f16x2, 0xd400d400u | z << 4);
    }
};
__device__ __forceinline__ void unpack8(uint32_t w, const Zero &z, f16x2 (&o)[4]) {
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f16x2 lo = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u);
        const f16x2 hi = __builtin_bit_cast(f16x2, (w & 0x00f000f0u) | 0x64006400u);
        o[2 * i] = lo - z.a;
        o[2 * i + 1] = __builtin_elementwise_fma(hi, sixteenth, z.b);
        w >>= 8;
    }
}

// Where row c of x's quarter h lies among a step's 64 operands in LDS: the 16
// columns of a block row that one instruction writes then fall on all banks (they
// would meet on a quarter of them), and a fragment read stays a permutation.
__device__ __forceinline__ int x_slot(int step, int h, int c) { return h * 16 + (c ^ (4 * ((step & 1) * 2 + (h >> 1)))); }

// 16 bytes from any address that an element may have.
template <typename T>
__device__ __forceinline__ i32x4 load16(const T *p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any {
        i32x4 v;
    };
    return reinterpret_cast<const Any *>(p)->v;
}

// 16 columns of x as fp32.
template <typename T>
__device__ __forceinline__ void load_x(const T *p, float (&v)[16]) {
    constexpr int kPer = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kPer)));
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
        const vec t = __builtin_bit_cast(vec, load16(p + i * kPer));
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[i * kPer + e] = (float)t[e];
    }
}

// M rows of x (up to 4) on the VALU.  A workgroup takes R = 4 rows of W, its waves
// the 1024-column slices in turn: lane l holds 16 columns of x in registers for
// R loads of 8 bytes of codes, so x passes through no LDS and a wave reads 512
// consecutive bytes of a row.  fp32 products of the exact codes and x
// (v_fma_mix); lanes and waves are summed at the end.  Bound by requests for few
// columns and by the VALU for more rows: fp32, 1 x 4096 x 4096 5.7 us (9.0 MB), bf16,
// 1 x 8192 x 28672 31 us (3.9 TB/s), 2 rows of it 46.  (Eight rows of W: 1 x 4096 x
// 4096 6.3 for 5.9, fp32 4 x 4096 x 14336 30 for 26; 2 x 8192 x 28672 44 for 50.)
constexpr int kRowsR = 4;
template <typename T, int M>
__global__ __launch_bounds__(256) void w4_rows_kernel(W4LinearParams p) {
    constexpr int R = kRowsR;
    __shared__ float red[4][M * R];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * R;
    const T *x = static_cast<const T *>(p.x);
    float acc[M][R];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = 0.f;
    u32x2 c[R];
    float s[R];
    uint32_t z[R];
    auto fetch = [&](int j) __attribute__((always_inline)) {
        const int jc = min(j, p.k - 16), g = jc / p.group;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = min(n0 + r, p.n - 1);
            c[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p.codes + (row * p.k + jc) / 2));
            s[r] = p.scales[row * p.groups + g];
            z[r] = p.zps ? p.zps[row * p.groups + g] : 8;
        }
    };
    int j = wave * 1024 + lane * 16;
    if (wave * 1024 < p.k) fetch(j);
    for (; (j & ~1023) < p.k; j += 4096) {
        float xv[M][16];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            if (j < p.k) {
                load_x(x + min(i, p.m - 1) * p.ldx + j, xv[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) xv[i][e] = 0.f;
            }
        }
        u32x2 cc[R];
        float ss[R];
        uint32_t zz[R];
#pragma unroll
        for (int r = 0; r < R; ++r) cc[r] = c[r], ss[r] = s[r], zz[r] = z[r];
        if ((j & ~1023) + 4096 < p.k) fetch(j + 4096);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Zero zero(zz[r]);
            f16x2 o[8];
            f16x2 (&o0)[4] = reinterpret_cast<f16x2 (&)[4]>(o[0]);
            f16x2 (&o1)[4] = reinterpret_cast<f16x2 (&)[4]>(o[4]);
            unpack8(cc[r][0], zero, o0);
            unpack8(cc[r][1], zero, o1);
#pragma unroll
            for (int i = 0; i < M; ++i) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = 8 * (e >> 2) + (e & 3);
                    d = fmaf((float)o[e][0], xv[i][at], d);
                    d = fmaf((float)o[e][1], xv[i][at + 4], d);
                }
                acc[i][r] = fmaf(ss[r], d, acc[i][r]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float t = wave_sum(acc[i][r]);
            if (lane == 0) red[wave][i * R + r] = t;
        }
    __syncthreads();
    if (tid < M * R) {
        const int i = tid / R, n = n0 + tid % R;
        if (i < p.m && n < p.n) {
            float t = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
            if (p.bias) t += (float)static_cast<const T *>(p.bias)[n];
            static_cast<T *>(p.y)[i * p.ldy + n] = (T)t;
        }
    }
}

// More rows on the matrix units: D = x . W^T by 16x16x32 f16.  A workgroup takes
// 128 rows of W and MB blocks of 16 rows of x, a wave RT tiles of 16 rows of W;
// lane (c = l % 16, h = l / 16) unpacks the codes of row c of W straight into its B
// operand and holds the result's column c, so a group's scale is one value per lane.
//
// Slices of 256 columns.  W comes by requests straight to LDS, a ring of kRing
// slices per wave (eight rows of 128 bytes per instruction).  x goes through
// registers into LDS, two buffers for the workgroup and one barrier per slice,
// as f16 in the codes' order (pairs 4 apart): f16 itself; bf16 and fp32 after a
// scaling, per row and slice, by the power of two that brings the largest
// magnitude to [2^14, 2^15), as one piece (bf16: 8 bits, exact above 2^-29 of the
// slice's largest) or three (fp32: 33 bits).  The slice's sums are scaled back as
// they join.  Scales and zero points are looked up per 32 columns, two of a row's
// eight per lane, and go round through LDS.
//
// Bound by waits, which are this tiling's own: a workgroup needs 4 us to its first
// slice and 1.5 us or more for each (LDS reads, then the barrier), so two or more
// blocks of x take eight waves of one tile each rather than four of two (f16, 50 x
// 4096 x 11008: 27.3 us against 32.5 with the join, where its bytes take 5).  K is
// split as far as the workgroups that fit the CUs go.
constexpr int kSlice = 256;
typedef __attribute__((address_space(3))) void *lds_ptr_t;
typedef __attribute__((address_space(1))) void *glb_ptr_t;

template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// PER: 32-column steps per sum (4 where groups are whole 128-column blocks).
template <typename T, int MB, bool ZP, int PER>
__global__ __launch_bounds__(MB == 1 ? 256 : 512, MB == 1 && sizeof(T) == 4 ? 1 : 2) void w4_tiles_kernel(W4LinearParams p) {
    constexpr int NP = std::is_same_v<T, float> ? 3 : 1;
    constexpr int NW = MB == 1 ? 4 : 8, RT = 8 / NW;  // waves, tiles of W each: 128 rows
    constexpr int XB = MB * 4 / NW;                   // x: blocks per thread
    constexpr bool SCALED = !std::is_same_v<T, _Float16>;
    constexpr int kX = NP * MB * kSlice * 16 * 2;  // one buffer of x
    constexpr int kW = RT * 16 * kSlice / 2;       // one slice of a wave's W
    constexpr int kXLoads = sizeof(T);             // per thread and block
    constexpr int kRing = 3;  // slices of W on their way or in use
    // loads of one slice, in their order: x, scales, W
    constexpr int kOps = XB * kXLoads + RT * (ZP ? 4 : 2) + 2 * RT;
    constexpr int kTable = ZP ? 1536 : 512;  // of a tile: scales [16][8], then Zero [16][8]
    __shared__ __attribute__((aligned(1024))) char lds[NW * kRing * kW + 2 * kX + 8 * kTable + 2 * MB * 64];
    char *const xbuf = lds + NW * kRing * kW;
    float *const backs = reinterpret_cast<float *>(xbuf + 2 * kX + 8 * kTable);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    char *const ring = lds + wave * kRing * kW;
    char *const sc = xbuf + 2 * kX + wave * RT * kTable;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
    const int n0 = tile * 128 + wave * 16 * RT, m0 = blockIdx.y * 16 * MB;
    const int k0 = split * p.kper, k1 = min(k0 + p.kper, p.k);
    const int ns = (k1 - k0 + kSlice - 1) / kSlice;
    const T *x = static_cast<const T *>(p.x);

    // W: instruction i of a tile fills rows 8 i .. of it; lane l the chunk (l % 8)
    // ^ (row / 2) of row l / 8, so that a read of 16 rows falls on all banks.  Rows
    // past n are row n - 1, columns past k column 0 (they meet zeros of x).
    const uint8_t *wsrc[RT][2];
    int wcol[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 8 * i + (lane >> 3);
        wcol[i] = 32 * ((lane & 7) ^ (row >> 1));
#pragma unroll
        for (int t = 0; t < RT; ++t) wsrc[t][i] = p.codes + (int64_t)min(n0 + 16 * t + row, p.n - 1) * (p.k / 2);
    }
    auto request_w = [&](int s) __attribute__((always_inline)) {
        const int j = k0 + min(s, ns - 1) * kSlice;  // (past the end: the last slice again, never read)
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int col = j + wcol[i];
                __builtin_amdgcn_global_load_lds((glb_ptr_t)(wsrc[t][i] + (col < p.k ? col : 0) / 2),
                                                 (lds_ptr_t)(ring + (s % kRing) * kW + (t * 2 + i) * 1024), 16, 0, kNtHint);
            }
    };
    // scales of row c, steps 2 h and 2 h + 1 of the next slice to be asked for
    int gi[2], rem[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = k0 + 64 * h + 32 * i;
        gi[i] = col / p.group;
        rem[i] = col - gi[i] * p.group;
    }
    const int gq = kSlice / p.group, gr = kSlice % p.group;
    struct Scales {
        float s[RT][2];
        uint32_t z[RT][2];
    } sa, sb;
    auto fetch_s = [&](Scales &f) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int64_t at = (int64_t)min(n0 + 16 * t + c, p.n - 1) * p.groups;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int g = min(gi[i], p.groups - 1);
                f.s[t][i] = p.scales[at + g];
                if (ZP) f.z[t][i] = p.zps[at + g];
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            gi[i] += gq;
            rem[i] += gr;
            if (rem[i] >= p.group) rem[i] -= p.group, ++gi[i];
        }
    };
    // x: thread (row tid / 16 of a block, 16 columns), as loaded
    i32x4 xa[XB][kXLoads], xb[XB][kXLoads];
    const int xrow = tid >> 4;  // and 4 NW ..
    auto fetch_x = [&](int s, i32x4 (&xr)[XB][kXLoads]) __attribute__((always_inline)) {
        const int col = k0 + s * kSlice + 16 * (tid & 15);
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            const T *at = x + min(m0 + 4 * NW * b + xrow, p.m - 1) * p.ldx + (col < k1 ? col : 0);
#pragma unroll
            for (int i = 0; i < kXLoads; ++i) xr[b][i] = load16(at + i * (16 / sizeof(T)));
        }
    };
    auto stage_x = [&](int s, i32x4 (&xr)[XB][kXLoads]) __attribute__((always_inline)) {
        char *const to = xbuf + (s & 1) * kX;
        if (k0 + (s + 1) * kSlice > k1) {  // (rows past m are copies of the last, never stored)
            const bool ok = k0 + s * kSlice + 16 * (tid & 15) < k1;
#pragma unroll
            for (int b = 0; b < XB; ++b)
#pragma unroll
                for (int i = 0; i < kXLoads; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) xr[b][i][e] = ok ? xr[b][i][e] : 0;
        }
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            float v[16], up = 1.f;
            if constexpr (SCALED) {
                // the exponent of the largest finite magnitude
                float big = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (sizeof(T) == 4) {
                        const int w = xr[b][e / 4][e % 4];
                        v[e] = __int_as_float(w);
                    } else {
                        const uint32_t w = (uint32_t)xr[b][e / 8][e % 8 / 2];
                        v[e] = __uint_as_float(e % 2 ? w & 0xffff0000u : w << 16);
                    }
                    big = fmaxf(big, fabsf(v[e]));
                }
                if (__any(!(big < INFINITY)) || sizeof(T) == 4) {
                    big = 0.f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) big = fmaxf(big, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
                }
                big = fmaxf(big, dpp_mov<0xB1>(big));
                big = fmaxf(big, dpp_mov<0x4E>(big));
                big = fmaxf(big, dpp_mov<0x124>(big));
                big = fmaxf(big, dpp_mov<0x128>(big));
                const int e2 = big > 0.f ? min(15 - __builtin_amdgcn_frexp_expf(big), 126) : 0;
                up = __builtin_ldexpf(1.f, e2);
                if ((tid & 15) == 0) backs[(s & 1) * MB * 16 + 4 * NW * b + xrow] = __builtin_ldexpf(1.f, -e2);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int unit = 2 * (tid & 15) + u;  // of 8 columns
                char *at = to + (((4 * NW * b + xrow) / 16 * 8 + unit / 4) * 64 + x_slot(unit / 4, unit % 4, xrow & 15)) * 16;
                if constexpr (!SCALED) {
                    i32x4 o;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t lo = (uint32_t)xr[b][u][e], hi = (uint32_t)xr[b][u][e + 2];
                        o[2 * e] = (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
                        o[2 * e + 1] = (int)__builtin_amdgcn_perm(hi, lo, 0x07060302u);
                    }
                    *reinterpret_cast<i32x4 *>(at) = o;
                } else {
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        i32x4 o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float &v0 = v[8 * u + e], &v1 = v[8 * u + e + 4];
                            if (q == 0 && NP > 1) v0 *= up, v1 *= up;
                            const f16x2 two = NP > 1 ? f16x2{(_Float16)v0, (_Float16)v1}
                                                     : f16x2{(_Float16)fmaf(v0, up, 0.f), (_Float16)fmaf(v1, up, 0.f)};
                            o[e] = __builtin_bit_cast(int, two);
                            if (q + 1 < NP) {
                                // (nothing is left of what is not finite)
                                const float r0 = v0 - (float)two[0], r1 = v1 - (float)two[1];
                                v0 = fabsf(v0) < INFINITY ? r0 : 0.f;
                                v1 = fabsf(v1) < INFINITY ? r1 : 0.f;
                            }
                        }
                        *reinterpret_cast<i32x4 *>(at + q * MB * kSlice * 32) = o;
                    }
                }
            }
        }
    };
    f32x4 acc[RT][MB], sum[RT][MB], g[RT][MB];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = sum[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    // x and scales two slices ahead, W kRing - 1; every slice makes the same kOps
    // loads in the same order, so the wait for its W is a constant.
    fetch_x(0, xa);
    fetch_x(1, xb);
    fetch_s(sa);
    fetch_s(sb);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s + 1 < kRing; ++s) request_w(s);
    stage_x(0, xa);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
#pragma unroll 1
    for (int s = 0; s < ns; ++s) {
        // this slice's scales into the wave's own table
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            *reinterpret_cast<float2 *>(sc + t * kTable + c * 32 + h * 8) = make_float2(sa.s[t][0], sa.s[t][1]);
            if (ZP) {
                Zero *const z = reinterpret_cast<Zero *>(sc + t * kTable + 512 + c * 64 + h * 16);
                z[0] = Zero(sa.z[t][0]), z[1] = Zero(sa.z[t][1]);
            }
        }
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int i = 0; i < kXLoads; ++i) xa[b][i] = xb[b][i];
        sa = sb;
        __builtin_amdgcn_sched_barrier(0);
        fetch_x(s + 2, xb);
        __builtin_amdgcn_sched_barrier(0);
        fetch_s(sb);
        __builtin_amdgcn_sched_barrier(0);
        request_w(s + kRing - 1);
        __builtin_amdgcn_sched_barrier(0);
        // W of slice s was asked for kRing - 1 slices ago; the first ones in a row
        if (s == 0)
            wait_vm<(kRing - 2) * 2 * RT + kOps>();
        else
            wait_vm<(kRing - 3) * 2 * RT + 2 * kOps>();
        __builtin_amdgcn_sched_barrier(0);
        const char *const wt = ring + (s % kRing) * kW;
        const char *const xt = xbuf + (s & 1) * kX;
        f32x4 sv[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) sv[t][i] = *reinterpret_cast<const f32x4 *>(sc + t * kTable + c * 32 + i * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e % PER == 0) {
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int b = 0; b < MB; ++b) g[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            f16x8 bw[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(wt + t * 2048 + c * 128 + ((e ^ (c >> 1)) << 4) + h * 4);
                f16x2 o[4];
                unpack8(w, ZP ? *reinterpret_cast<const Zero *>(sc + t * kTable + 512 + c * 64 + e * 8) : Zero(8), o);
                bw[t] = __builtin_shufflevector(__builtin_shufflevector(o[0], o[1], 0, 1, 2, 3),
                                                __builtin_shufflevector(o[2], o[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int q = NP - 1; q >= 0; --q) {
                    const f16x8 a = *reinterpret_cast<const f16x8 *>(xt + q * MB * kSlice * 32 +
                                                                     ((b * 8 + e) * 64 + x_slot(e, h, c)) * 16);
#pragma unroll
                    for (int t = 0; t < RT; ++t) g[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bw[t], g[t][b], 0, 0, 0);
                }
            if (e % PER == PER - 1) {
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int b = 0; b < MB; ++b) {
                        f32x4 &to = SCALED ? sum[t][b] : acc[t][b];
#pragma unroll
                        for (int r = 0; r < 4; ++r) to[r] = fmaf(g[t][b][r], sv[t][e / 4][e % 4], to[r]);
                    }
            }
        }
        if (SCALED) {
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                const f32x4 f = *reinterpret_cast<const f32x4 *>(backs + (s & 1) * MB * 16 + 16 * b + 4 * h);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[t][b][r] = fmaf(sum[t][b][r], f[r], acc[t][b][r]);
                    sum[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
        }
        stage_x(s + 1, xa);
        // every wave's x of the next slice is there, and is done with this one's
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm<0>();  // nothing is still on its way into the ring
    // lane (c, h), register r: row 4 h + r of x's block, row c of W's tile
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int n = n0 + 16 * t + c;
        if (n >= p.n) continue;
        const float bias = p.bias && p.splits == 1 ? (float)static_cast<const T *>(p.bias)[n] : 0.f;
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + 16 * b + 4 * h + r;
                if (m >= p.m) continue;
                if (p.splits > 1)
                    p.part[((int64_t)split * p.m + m) * p.n + n] = acc[t][b][r];
                else
                    static_cast<T *>(p.y)[m * p.ldy + n] = (T)(acc[t][b][r] + bias);
            }
    }
}

// ---- up to 16 rows of 16 bits: W as a stream -------------------------------------------

// Eight codes of one row as the B operand of a 16x16x32 product, in their order.
// f16: 0x6400 | c and 0x6400 | c << 4 from one byte, then one packed operation takes
// 1024 + z or 16 (64 + z) off: c - z.  bf16: the byte c is the fp8 (e4m3) number
// c 2^-9 (0 .. 7 the subnormal ones, 8 .. 15 the first binade), so the conversion
// from fp8 gives c itself; z is taken off the sums.
__device__ __forceinline__ f16x8 codes_f16(uint32_t w, f16x2 zero) {
    i32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = __builtin_amdgcn_perm(0, w, 0x0c000c00u | i << 16 | i);
        const f16x2 v = __builtin_bit_cast(f16x2, (two & 0x00f0000fu) | 0x64006400u);
        o[i] = __builtin_bit_cast(int, __builtin_elementwise_fma(v, f16x2{(_Float16)1.f, (_Float16)0.0625f}, zero));
    }
    return __builtin_bit_cast(f16x8, o);
}
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w) {
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
    const uint32_t lo = __builtin_amdgcn_perm(odd, even, 0x05010400u), hi = __builtin_amdgcn_perm(odd, even, 0x07030602u);
    i32x4 o;
    o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, false));
    o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.f, true));
    o[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, false));
    o[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.f, true));
    return __builtin_bit_cast(bf16x8, o);
}
// (c - z as bf16, for x that is not finite)
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w, float z) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (__bf16)((float)((w >> 4 * i) & 15) - z);
    return o;
}

constexpr int kStreamWaves = 8;
constexpr int kStreamTable = 32 << 10;  // bytes of LDS for scales and zero points

// A workgroup takes 16 rows of W, its waves a share of the columns each and no
// barrier between its first and last: K is split inside the workgroup, so there
// are no parts to join and no second launch.  Slices of 128 columns, four on
// their way in registers, asked for two at a time (W's lines hold two):
//   W   lane (c = l % 16, h = l / 16) 16 bytes, columns 32 h .. of row c; four lane
//       swaps transpose (h, dword) so that step j takes columns 32 j + 8 h ..
//   x   four rows of 256 bytes per instruction, through 4 KB of LDS of the wave's
//       own into operands (loaded as operands, 16 rows of 64 bytes, the same
//       bytes take twice the time: 22.4 us against 16.8)
// The 16 rows' scales and zero points go to LDS at once.  bf16: g = sum c x and
// one product with ones, sx = sum x, give s (g - z sx): exact as far as fp32 sums
// are, and 0 for a row of zeros, as g and 8 sx round alike.  Where a sum is not
// finite the wave repeats its share with c - z, so infinities reach what they
// should.
//
// Bound by requests: a CU takes 1 KB of x and W in some 30 cycles, and x, which
// every workgroup reads whole from its L2, is four of five (of 16 rows of W to a
// workgroup; more rows to one would read less of x).  16 x 14336 x 4096: 15.5 us with
// groups of 64 and zero points (34.5 MB, 2.2 TB/s); sixteen waves 15.4 there but 9.6
// against 8.0 at 4096 x 4096 and 30 against 18 at 4096 x 14336.
template <typename T, bool ZP, int PER>
__global__ __launch_bounds__(64 * kStreamWaves, 4) void w4_stream_kernel(W4LinearParams p) {
    constexpr int R = 4, kAt = 2;  // slices on their way or in use, asked for at once
    constexpr int NP = ZP ? 2 : 1;
    constexpr bool BF = !std::is_same_v<T, _Float16>;
    constexpr int kX = 1024;  // floats
    // a slice of x per wave and the table of scales (and zero points); in the end
    // the waves' sums
    __shared__ __attribute__((aligned(16))) float lds[kStreamWaves * kX + kStreamTable / 4];
    float *const table = lds + kStreamWaves * kX;
    const int ld = NP * p.groups | 1;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * 16, rows = min(16, p.n - n0);
    const int all = (p.k + 127) / 128, per = (all + kStreamWaves - 1) / kStreamWaves;
    const int s0 = wave * per, s1 = min(all, s0 + per);
    const char *const xbase = static_cast<const char *>(p.x);
    const uint8_t *const wbase = p.codes + (int64_t)n0 * (p.k / 2);
    char *const xl = reinterpret_cast<char *>(lds + wave * kX);
    // (rows past the last are copies of it, never stored)
    const uint32_t wat = (uint32_t)(min(c, rows - 1) * (p.k / 2) + 16 * h);
    uint32_t xat[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xat[i] = ((uint32_t)min(4 * i + h, p.m - 1) * (uint32_t)p.ldx + 8 * c) * 2;
    struct Stage {
        i32x4 x[4], w;
    } st[R];
    // (past the wave's last slice: one line of the first, never used)
    auto fetch = [&](Stage &f, int s) __attribute__((always_inline)) {
        const uint32_t on = s < s1 ? ~0u : 0u;
        const int col = s < s1 ? s * 128 : 0;
        if (col + 128 <= p.k) {
            f.w = *reinterpret_cast<const i32x4 *>(wbase + col / 2 + (wat & on));
#pragma unroll
            for (int i = 0; i < 4; ++i) f.x[i] = load16(xbase + (int64_t)col * 2 + (xat[i] & on));
        } else {
            f.w = *reinterpret_cast<const i32x4 *>(wbase + col / 2 + (col + 32 * h < p.k ? wat : wat - 16 * h));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                f.x[i] = load16(xbase + (int64_t)col * 2 + (col + 8 * c < p.k ? xat[i] : xat[i] - 16 * c));
        }
    };
    if (s0 < s1) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            fetch(st[i], s0 + i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    for (int row = wave; row < rows; row += kStreamWaves) {
        const float *const from = p.scales + (int64_t)(n0 + row) * p.groups;
        const uint8_t *const zfrom = ZP ? p.zps + (int64_t)(n0 + row) * p.groups : nullptr;
        for (int g = lane; g < p.groups; g += 256) {
            float v[4];
            uint32_t z[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int e = min(g + 64 * y, p.groups - 1);
                v[y] = from[e];
                z[y] = ZP ? zfrom[e] : 0;
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                float *const to = table + row * ld + NP * min(g + 64 * y, p.groups - 1);
                to[0] = v[y];
                // (f16: -(1024 + z), -(64 + z))
                if (ZP) to[1] = BF ? (float)z[y] : __uint_as_float(0xd400e400u + (z[y] | z[y] << 20));
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto use = [&](Stage &f, int s, auto redo) __attribute__((always_inline)) {
        constexpr bool REDO = decltype(redo)::value;
        constexpr bool SX = BF && !REDO;
        if (s * 128 + 128 > p.k && s * 128 + 8 * c >= p.k) {  // no columns there
#pragma unroll
            for (int i = 0; i < 4; ++i) f.x[i] = i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<i32x4 *>(xl + (4 * i + h) * 256 + ((c ^ (4 * i + h)) << 4)) = f.x[i];
        // scales and zero points of the slice's groups
        float sc[4 / PER], zf[4 / PER];
#pragma unroll
        for (int q = 0; q < 4 / PER; ++q) {
            const uint32_t step = 4 * s + PER * q;
            const int g = min((int)(p.steps == 1 ? step : __umulhi(step, p.magic)), p.groups - 1);
            const float *const of = table + min(c, rows - 1) * ld + NP * g;
            sc[q] = of[0];
            zf[q] = ZP ? of[1] : BF ? 8.f : __uint_as_float(0xd480e408u);
        }
        uint32_t d[4] = {(uint32_t)f.w[0], (uint32_t)f.w[1], (uint32_t)f.w[2], (uint32_t)f.w[3]};
        auto swap32 = [&](uint32_t &a, uint32_t &b) {
            const auto v = __builtin_amdgcn_permlane32_swap(a, b, false, false);
            a = v[0], b = v[1];
        };
        auto swap16 = [&](uint32_t &a, uint32_t &b) {
            const auto v = __builtin_amdgcn_permlane16_swap(a, b, false, false);
            a = v[0], b = v[1];
        };
        swap32(d[0], d[2]), swap32(d[1], d[3]);
        swap16(d[0], d[1]), swap16(d[2], d[3]);
#pragma unroll
        for (int q = 0; q < 4 / PER; ++q) {
            f32x4 g = {0.f, 0.f, 0.f, 0.f}, sx = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = PER * q; j < PER * q + PER; ++j) {
                const i32x4 xv = *reinterpret_cast<const i32x4 *>(xl + c * 256 + (((4 * j + h) ^ c) << 4));
                if constexpr (BF) {
                    const bf16x8 a = __builtin_bit_cast(bf16x8, xv);
                    const i32x4 one = {0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};
                    if (SX)
                        sx = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, one), sx, 0, 0, 0);
                    g = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, REDO ? codes_bf16(d[j], zf[q]) : codes_bf16(d[j]), g, 0,
                                                                0, 0);
                } else {
                    g = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, xv),
                                                              codes_f16(d[j], __builtin_bit_cast(f16x2, zf[q])), g, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = fmaf(SX ? fmaf(-zf[q], sx[r], g[r]) : g[r], sc[q], acc[r]);
        }
    };
#pragma unroll 1
    for (int s = s0; s < s1; s += R) {
#pragma unroll
        for (int i = 0; i < R; i += kAt) {
#pragma unroll
            for (int y = i; y < i + kAt; ++y)
                if (s + y < s1) use(st[y], s + y, std::false_type{});
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int y = i; y < i + kAt; ++y) fetch(st[y], s + y + R);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if constexpr (BF) {
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= !(fabsf(acc[r]) < INFINITY);
        if (__any(odd)) {  // (finite sums stay what they are without the others)
            const f32x4 was = acc;
            acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int s = s0; s < s1; ++s) {
                fetch(st[0], s);
                use(st[0], s, std::true_type{});
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = fabsf(was[r]) < INFINITY ? was[r] : acc[r];
        }
    }
    __syncthreads();
    *reinterpret_cast<f32x4 *>(lds + (wave * 64 + lane) * 4) = acc;
    __syncthreads();
    // the waves' sums in their order; lane (c, h), register r: row 4 h + r of x, row
    // c of W
    const int m = threadIdx.x >> 4, n = threadIdx.x & 15;
    if (m >= p.m || n >= rows) return;
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kStreamWaves; ++u) v += lds[(u * 64 + (m >> 2) * 16 + n) * 4 + (m & 3)];
    if (p.bias) v += (float)static_cast<const T *>(p.bias)[n0 + n];
    static_cast<T *>(p.y)[m * p.ldy + n0 + n] = (T)v;
}

// The splits' sums in their order, and the bias.
template <typename T>
__global__ __launch_bounds__(256) void w4_join_kernel(W4LinearParams p) {
    const int n = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
    if (n >= p.n) return;
    const int64_t one = (int64_t)p.m * p.n;
    const float *at = p.part + (int64_t)m * p.n + n;
    float t = 0.f;
    for (int s = 0; s < p.splits; s += 4) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = s + i < p.splits ? at[(s + i) * one] : 0.f;
        t += (v[0] + v[1]) + (v[2] + v[3]);
    }
    if (p.bias) t += (float)static_cast<const T *>(p.bias)[n];
    static_cast<T *>(p.y)[m * p.ldy + n] = (T)t;
}

// Rows of x that the VALU form takes, and whether the stream of W takes a call.
// us of a call's kernels (bf16, groups of 128), VALU / stream / tiles:
//   n x k           m = 1            2             4             16
//   1024 x 4096     3.7 / 7.7        4.4 / 7.5     5.9 / 7.5     - / 7.6 / 12.9
//   4096 x 4096     6.2 / 8.1        7.6 / 8.0     10.5 / 7.8    - / 8.0 / 14.1
//   4096 x 14336    12.2 / 14.8      16.4 / 15.3   23.0 / 15.0   - / 16.0 / 21.6
//   14336 x 4096    11.4 / 17.8      15.8 / 17.9   27.7 / 17.6   - / 18.2 / 20.8
//   28672 x 8192    30.2 / 49.7      43.3 / 49.6   79.0 / 50.4   - / 59.1 / 45.7
// so up to two rows go to the VALU, and where W has 2^27 codes or more, more than
// two to the tiles.  The stream holds a row block's scales and zero points in LDS
// (asked for whether there are zero points or not, and without the strides: the
// size of the workspace is asked for without them).  fp32 x takes three pieces per
// product: four rows go to the VALU.
//
// The stream finds a step's group as the high word of step * magic, where magic =
// 2^32 / steps + 1 (steps per group) is at most `steps` too large after the product
// with steps: the quotient while step * steps < 2^32, so longer groups go elsewhere.
int64_t rows_max(const LinearW4Desc &d) { return d.dtype == GFH_F32 ? 4 : 2; }
bool w4_streams(const LinearW4Desc &d) {
    const int64_t groups = (d.k + d.group - 1) / d.group;
    const bool found = groups == 1 || (d.k / 128 * 4 + 4) * (d.group / 32) < (int64_t)1 << 32;
    return d.dtype != GFH_F32 && d.m > rows_max(d) && d.m <= 16 && d.n * d.k < (int64_t)1 << 27 &&
           16 * (2 * groups + 1) * 4 <= kStreamTable && found;
}

struct W4Plan {
    int mb, splits, kper;
};
W4Plan w4_plan(const LinearW4Desc &d) {
    W4Plan pl{};
    const int64_t blocks = (d.m + 15) / 16;
    pl.mb = (int)std::min<int64_t>(blocks, d.dtype == GFH_F32 ? 2 : 4);
    if (pl.mb == 3) pl.mb = 4;
    const int64_t tiles = (d.n + 127) / 128 * ((d.m + 16 * pl.mb - 1) / (16 * pl.mb));
    const int64_t slices = (d.k + kSlice - 1) / kSlice;
    // K is split as far as the workgroups that fit the CUs at once go
    const int64_t slots = (pl.mb > 1 || d.dtype == GFH_F32 ? 1 : 2) * device_cu_count();
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(slots / tiles, slices / 2));
    const int64_t per = (slices + want - 1) / want;
    pl.kper = (int)(per * kSlice);
    pl.splits = (int)((slices + per - 1) / per);
    return pl;
}

}  // namespace

int launch_quantize_w4(const float *w, int64_t n, int64_t k, int64_t group, uint8_t *codes, float *scales, uint8_t *zps,
                       hipStream_t s) {
    W4Params p{};
    p.w = w, p.codes = codes, p.scales = scales, p.zps = zps;
    p.n = n, p.k = k, p.group = (int)group;
    p.groups = (k + group - 1) / group;
    p.lanes = 4;
    while (p.lanes < 64 && p.lanes * 8 < group) p.lanes *= 2;
    p.lane_bits = __builtin_ctz((unsigned)p.lanes);
    const int64_t blocks = (n * p.groups * p.lanes + 255) / 256;
    if (blocks > (int64_t)1 << 23) return set_error(GFH_INVALID_SHAPE, "quantize_i4_grouped: grid too large");
    hipLaunchKernelGGL(quantize_w4_kernel, dim3((unsigned)blocks), dim3(256), 0, s, p);
    return check_launch("quantize_i4_grouped");
}

int launch_dequantize_w4(const uint8_t *codes, const float *scales, const uint8_t *zps, int64_t n, int64_t k,
                         int64_t group, float *out, hipStream_t s) {
    W4Params p{};
    p.codes = const_cast<uint8_t *>(codes), p.scales = const_cast<float *>(scales), p.zps = const_cast<uint8_t *>(zps);
    p.out = out;
    p.n = n, p.k = k, p.group = (int)group;
    p.groups = (k + group - 1) / group;
    const int64_t blocks = std::min<int64_t>((n * (k / 8) + 255) / 256, (int64_t)1 << 16);
    hipLaunchKernelGGL(dequantize_w4_kernel, dim3((unsigned)blocks), dim3(256), 0, s, p);
    return check_launch("dequantize_i4_grouped");
}

bool linear_w4_fits(const LinearW4Desc &d) {
    if (d.m <= rows_max(d) || w4_streams(d)) return (d.n + kRowsR - 1) / kRowsR <= kMaxBlocks256;
    return (d.n + 127) / 128 * w4_plan(d).splits <= kMaxBlocks256 / 2;  // (of up to 512 threads)
}

size_t linear_w4_workspace_bytes(const LinearW4Desc &d) {
    if (d.m <= rows_max(d) || w4_streams(d)) return 0;
    const W4Plan pl = w4_plan(d);
    return pl.splits > 1 ? (size_t)pl.splits * d.m * d.n * 4 : 0;
}

int launch_linear_w4(const LinearW4Desc &d, void *workspace, hipStream_t s) {
    W4LinearParams p{};
    p.x = d.x, p.codes = d.codes, p.scales = d.scales, p.zps = d.zps, p.bias = d.bias, p.y = d.y;
    p.ldx = d.ldx, p.ldy = d.ldy;
    p.m = (int)d.m, p.n = (int)d.n, p.k = (int)d.k, p.group = (int)d.group;
    p.groups = (int)((d.k + d.group - 1) / d.group);
    p.part = static_cast<float *>(workspace);
    p.splits = 1;
    auto typed = [&](auto &&go) {
        if (d.dtype == GFH_F32)
            go(float{});
        else if (d.dtype == GFH_BF16)
            go(__bf16{});
        else
            go(_Float16{});
    };
    // (its offsets into x have 32 bits; rows further apart go to the VALU below)
    if (w4_streams(d) && d.ldx < (int64_t)1 << 26) {
        p.steps = d.group >= d.k ? 1 << 30 : (int)(d.group / 32);
        p.magic = (uint32_t)(((uint64_t)1 << 32) / p.steps + 1);
        const dim3 grid((unsigned)((d.n + 15) / 16)), block(64 * kStreamWaves);
        auto go = [&](auto t, auto per) {
            using T = decltype(t);
            constexpr int PER = decltype(per)::value;
            if (d.zps)
                hipLaunchKernelGGL((w4_stream_kernel<T, true, PER>), grid, block, 0, s, p);
            else
                hipLaunchKernelGGL((w4_stream_kernel<T, false, PER>), grid, block, 0, s, p);
        };
        auto sized = [&](auto t) {
            if (p.steps % 4 == 0)
                go(t, std::integral_constant<int, 4>{});
            else if (p.steps % 2 == 0)
                go(t, std::integral_constant<int, 2>{});
            else
                go(t, std::integral_constant<int, 1>{});
        };
        if (d.dtype == GFH_BF16)
            sized(__bf16{});
        else
            sized(_Float16{});
        return check_launch("linear_w4");
    }
    if (d.m <= rows_max(d) || w4_streams(d)) {
        typed([&](auto t) {
            using T = decltype(t);
            auto go = [&](auto mc) {
                hipLaunchKernelGGL((w4_rows_kernel<T, decltype(mc)::value>), dim3((unsigned)((d.n + kRowsR - 1) / kRowsR)),
                                   dim3(256), 0, s, p);
            };
            for (int64_t m = 0; m < d.m; m += 4) {
                p.x = static_cast<const T *>(d.x) + m * d.ldx;
                p.y = static_cast<T *>(d.y) + m * d.ldy;
                p.m = (int)std::min<int64_t>(4, d.m - m);
                if (p.m == 1)
                    go(std::integral_constant<int, 1>{});
                else if (p.m == 2)
                    go(std::integral_constant<int, 2>{});
                else
                    go(std::integral_constant<int, 4>{});
            }
        });
        return check_launch("linear_w4");
    }
    const W4Plan pl = w4_plan(d);
    p.splits = pl.splits;
    p.kper = pl.kper;
    const int64_t gx = (d.n + 127) / 128 * pl.splits, gy = (d.m + 16 * pl.mb - 1) / (16 * pl.mb);
    const dim3 grid((unsigned)gx, (unsigned)gy);
    typed([&](auto t) {
        using T = decltype(t);
        auto go = [&](auto mb, auto per) {
            constexpr int MB = decltype(mb)::value, PER = decltype(per)::value;
            if (d.zps)
                hipLaunchKernelGGL((w4_tiles_kernel<T, MB, true, PER>), grid, dim3(MB == 1 ? 256 : 512), 0, s, p);
            else
                hipLaunchKernelGGL((w4_tiles_kernel<T, MB, false, PER>), grid, dim3(MB == 1 ? 256 : 512), 0, s, p);
        };
        auto sized = [&](auto per) {
            if (pl.mb == 1)
                go(std::integral_constant<int, 1>{}, per);
            else if (pl.mb == 2)
                go(std::integral_constant<int, 2>{}, per);
            else if constexpr (!std::is_same_v<T, float>)
                go(std::integral_constant<int, 4>{}, per);
        };
        if (d.group % 128 == 0 || d.group >= d.k)
            sized(std::integral_constant<int, 4>{});
        else
            sized(std::integral_constant<int, 1>{});
    });
    GFH_TRY(check_launch("linear_w4"));
    if (pl.splits > 1) {
        const dim3 jg((unsigned)((d.n + 255) / 256), (unsigned)d.m);
        typed([&](auto t) { hipLaunchKernelGGL(w4_join_kernel<decltype(t)>, jg, dim3(256), 0, s, p); });
        GFH_TRY(check_launch("linear_w4 (join)"));
    }
    return GFH_SUCCESS;
}

}  // namespace gfh
