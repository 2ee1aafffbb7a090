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
// group's finished sum in fp32.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "paged_types.hpp"
#include "quant_math.hpp"

namespace gfh {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

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
    int lanes;  // per group (a power of two up to 64)
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

// A group's 8-column units over `lanes` lanes (several each where the group is
// longer), fp32 in, four code bytes per unit out.  Bound by bytes.
__global__ __launch_bounds__(256) void quantize_w4_kernel(W4Params p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t gi = id / p.lanes;
    const int sub = (int)(id % p.lanes);
    const bool ok = gi < p.n * p.groups;
    const int64_t row = ok ? gi / p.groups : 0, g = ok ? gi % p.groups : 0;
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
    for (int64_t j = j0 + 8 * sub; j < j1; j += 8 * p.lanes) {
        if (!one) load_vec<8>(w + j, v);
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) c |= w4_code(v[e], s, z) << (4 * e);
        *reinterpret_cast<uint32_t *>(p.codes + (row * p.k + j) / 2) = c;
    }
    if (sub == 0) {
        p.scales[gi] = s;
        if (p.zps) p.zps[gi] = (uint8_t)z;
    }
}

__global__ __launch_bounds__(256) void dequantize_w4_kernel(W4Params p) {
    const int64_t units = p.n * (p.k / 8);
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < units; id += (int64_t)gridDim.x * 256) {
        const int64_t row = id / (p.k / 8), j = (id - row * (p.k / 8)) * 8;
        const int64_t gi = row * p.groups + j / p.group;
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
    bool xvec;  // rows of x allow 16-byte loads
    int kper;   // columns per split
    int splits;
};

// Eight codes as f16 pairs (0, 4), (1, 5), (2, 6), (3, 7), z taken off.
struct Zero {
    f16x2 a, b;  // 1024 + z, -(64 + z)
    __device__ __forceinline__ explicit Zero(uint32_t z) {
        a = __builtin_bit_cast(f16x2, 0x64006400u | z | z << 16);
        b = __builtin_bit_cast(f16x2, 0xd400d400u | z << 4 | z << 20);
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

template <int N, typename T>
__device__ __forceinline__ void load_x(const T *p, bool vec, float (&v)[N]) {
    if (vec) {
        load_vec<N>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)p[e];
    }
}

// M rows of x (up to 4) on the VALU.  A workgroup takes R rows of W, its waves
// the 1024-column slices in turn: lane l holds 16 columns of x in registers for
// R loads of 8 bytes of codes, so x passes through no LDS and a wave reads 512
// consecutive bytes of a row.  fp32 products of the exact codes and x
// (v_fma_mix); lanes and waves are summed at the end.
template <typename T, int M, int R>
__global__ __launch_bounds__(256) void w4_rows_kernel(W4LinearParams p) {
    __shared__ float red[4][M * R];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * R;
    const T *x = static_cast<const T *>(p.x);
    float acc[M][R];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = 0.f;
    uint2 c[R];
    float s[R];
    uint32_t z[R];
    auto fetch = [&](int j) __attribute__((always_inline)) {
        const int jc = min(j, p.k - 16), g = jc / p.group;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = min(n0 + r, p.n - 1);
            c[r] = *reinterpret_cast<const uint2 *>(p.codes + (row * p.k + jc) / 2);
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
                load_x<16>(x + min(i, p.m - 1) * p.ldx + j, p.xvec, xv[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) xv[i][e] = 0.f;
            }
        }
        uint2 cc[R];
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
            unpack8(cc[r].x, zero, o0);
            unpack8(cc[r].y, zero, o1);
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

// More rows on the matrix units: D = x . W^T by 16x16x32 f16.  A wave takes RT
// tiles of 16 rows of W and MB blocks of 16 rows of x; lane (c = l % 16, h = l /
// 16) unpacks the codes of row c of W straight into its B operand and holds the
// result's column c, so a group's scale is one value per lane.
//
// x goes through LDS as f16 in the codes' order (pairs 4 apart): f16 itself;
// bf16 and fp32 after a scaling, per row and 256-column slice, by the power of
// two that brings the largest magnitude to [2^14, 2^15), as one piece (bf16: 8
// bits, exact above 2^-29 of the slice's largest) or three (fp32: 33 bits).  The
// slice's sums are scaled back as they join.
//
// Loads of 16 bytes give lane (c, h) columns 32 h .. of a 128-column block.
// Where groups are whole blocks the products take them so (step t: columns 32 h
// + 8 t of every h); else (T32) a 4 x 4 transposition over the four lanes of a row
// makes step t the columns 32 t + 8 h, all of one group.
constexpr int kSlice = 256;

template <typename T, int MB, int RT, bool T32>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void w4_tiles_kernel(W4LinearParams p) {
    constexpr int NP = std::is_same_v<T, float> ? 3 : 1;
    constexpr bool SCALED = !std::is_same_v<T, _Float16>;
    constexpr int NG = T32 ? 8 : 2;  // scales per slice
    constexpr int kBuf = NP * MB * kSlice * 16 * 2;
    __shared__ __attribute__((aligned(16))) char lds[2 * kBuf];
    __shared__ __attribute__((aligned(16))) float back[2][MB * 16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
    const int n0 = tile * 64 * RT + wave * 16 * RT, m0 = blockIdx.y * 16 * MB;
    const int k0 = split * p.kper, k1 = min(k0 + p.kper, p.k);
    const T *x = static_cast<const T *>(p.x);

    struct Set {
        i32x4 w[RT][2];
        float s[RT][NG];
        uint32_t z[RT][NG];
    };
    auto fetch = [&](int j, Set &f) __attribute__((always_inline)) {
        j = min(j, k1 - 1) & ~(kSlice - 1);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int64_t row = min(n0 + 16 * t + c, p.n - 1);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int col = j + 128 * b + 32 * h;
                f.w[t][b] = *reinterpret_cast<const i32x4 *>(p.codes + (row * p.k + (col < p.k ? col : 0)) / 2);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int64_t at = row * p.groups + min((j + (kSlice / NG) * g) / p.group, p.groups - 1);
                f.s[t][g] = p.scales[at];
                f.z[t][g] = p.zps ? p.zps[at] : 8;
            }
        }
    };
    // x: thread (row tid / 16 of a block, 16 columns)
    float xr[MB][16];
    auto fetch_x = [&](int j) __attribute__((always_inline)) {
        const int col = j + 16 * (tid & 15);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int row = m0 + 16 * b + (tid >> 4);
            if (row < p.m && col < k1) {
                load_x<16>(x + row * p.ldx + col, p.xvec, xr[b]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) xr[b][e] = 0.f;
            }
        }
    };
    auto stage_x = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            if constexpr (SCALED) {
                // the largest finite magnitude's power of two
                float big = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float a = fabsf(xr[b][e]);
                    big = fmaxf(big, a < INFINITY ? a : 0.f);
                }
                big = fmaxf(big, dpp_mov<0xB1>(big));
                big = fmaxf(big, dpp_mov<0x4E>(big));
                big = fmaxf(big, dpp_mov<0x124>(big));
                big = fmaxf(big, dpp_mov<0x128>(big));
                const int e2 = big > 0.f ? min(14 - ilogbf(big), 126) : 0;
                const float up = ldexpf(1.f, e2);
#pragma unroll
                for (int e = 0; e < 16; ++e) xr[b][e] *= up;
                if ((tid & 15) == 0) back[buf][16 * b + (tid >> 4)] = ldexpf(1.f, -e2);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int unit = 2 * (tid & 15) + u;  // of 8 columns
                const int step = T32 ? unit / 4 : 4 * (unit / 16) + unit % 4, hh = T32 ? unit % 4 : (unit % 16) / 4;
                char *at = lds + buf * kBuf + ((b * 8 + step) * 64 + hh * 16 + (tid >> 4)) * 16;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = xr[b][8 * u + (e >> 1) + 4 * (e & 1)];
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    f16x8 o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] = (_Float16)v[e];
                        // (nothing is left of what is not finite)
                        const float r = v[e] - (float)o[e];
                        v[e] = fabsf(v[e]) < INFINITY ? r : 0.f;
                    }
                    *reinterpret_cast<f16x8 *>(at + q * MB * kSlice * 32) = o;
                }
            }
        }
    };
    f32x4 acc[RT][MB], sum[RT][MB];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int buf, Set &f) __attribute__((always_inline)) {
        if (SCALED) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int b = 0; b < MB; ++b) sum[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t w[RT][4];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[t][e] = (uint32_t)f.w[t][k][e];
                if (T32) {
                    // register e of quarter h <-> register h of quarter e
                    const auto a = __builtin_amdgcn_permlane32_swap(w[t][0], w[t][2], false, false);
                    const auto d = __builtin_amdgcn_permlane32_swap(w[t][1], w[t][3], false, false);
                    const auto u = __builtin_amdgcn_permlane16_swap(a[0], d[0], false, false);
                    const auto v = __builtin_amdgcn_permlane16_swap(a[1], d[1], false, false);
                    w[t][0] = u[0], w[t][1] = u[1], w[t][2] = v[0], w[t][3] = v[1];
                }
            }
            f32x4 g[RT][MB];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (T32 || e == 0) {
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int b = 0; b < MB; ++b) g[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                const int gi = T32 ? 4 * k + e : k;
                f16x8 bw[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    f16x2 o[4];
                    unpack8(w[t][e], Zero(f.z[t][gi]), o);
                    bw[t] = __builtin_shufflevector(__builtin_shufflevector(o[0], o[1], 0, 1, 2, 3),
                                                    __builtin_shufflevector(o[2], o[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int q = NP - 1; q >= 0; --q) {
                        const f16x8 a = *reinterpret_cast<const f16x8 *>(
                            lds + buf * kBuf + q * MB * kSlice * 32 + ((b * 8 + 4 * k + e) * 64 + lane) * 16);
#pragma unroll
                        for (int t = 0; t < RT; ++t) g[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bw[t], g[t][b], 0, 0, 0);
                    }
                if (T32 || e == 3) {
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int b = 0; b < MB; ++b) {
                            f32x4 &to = SCALED ? sum[t][b] : acc[t][b];
#pragma unroll
                            for (int r = 0; r < 4; ++r) to[r] = fmaf(g[t][b][r], f.s[t][gi], to[r]);
                        }
                }
            }
        }
        if (SCALED) {
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                const f32x4 s = *reinterpret_cast<const f32x4 *>(&back[buf][16 * b + 4 * h]);
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[t][b][r] = fmaf(sum[t][b][r], s[r], acc[t][b][r]);
            }
        }
    };
    const int ns = (k1 - k0 + kSlice - 1) / kSlice;
    Set f[2];
    fetch_x(k0);
    fetch(k0, f[0]);
    fetch(k0 + kSlice, f[1]);
    stage_x(0);
    __syncthreads();
    for (int i = 0; i < ns; i += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (i + u < ns) {
                const int j = k0 + (i + u) * kSlice;
                if (i + u + 1 < ns) fetch_x(j + kSlice);
                compute(u, f[u]);
                fetch(j + 2 * kSlice, f[u]);
                if (i + u + 1 < ns) stage_x(u ^ 1);
                __syncthreads();
            }
        }
    }
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

constexpr int kRowsMax = 4;  // rows of x that the VALU form takes

struct W4Plan {
    int mb, rt, splits, kper;
};
W4Plan w4_plan(const LinearW4Desc &d) {
    W4Plan pl{};
    const int64_t blocks = (d.m + 15) / 16;
    pl.mb = (int)std::min<int64_t>(blocks, d.dtype == GFH_F32 ? 2 : 4);
    if (pl.mb == 3) pl.mb = 4;
    pl.rt = pl.mb == 1 ? 1 : 2;
    const int64_t tiles = (d.n + 64 * pl.rt - 1) / (64 * pl.rt) * ((d.m + 16 * pl.mb - 1) / (16 * pl.mb));
    const int64_t slices = (d.k + kSlice - 1) / kSlice;
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(2 * device_cu_count() / tiles, slices / 2));
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

size_t linear_w4_workspace_bytes(const LinearW4Desc &d) {
    if (d.m <= kRowsMax) return 0;
    const W4Plan pl = w4_plan(d);
    return pl.splits > 1 ? (size_t)pl.splits * d.m * d.n * 4 : 0;
}

int launch_linear_w4(const LinearW4Desc &d, void *workspace, hipStream_t s) {
    W4LinearParams p{};
    p.x = d.x, p.codes = d.codes, p.scales = d.scales, p.zps = d.zps, p.bias = d.bias, p.y = d.y;
    p.ldx = d.ldx, p.ldy = d.ldy;
    p.m = (int)d.m, p.n = (int)d.n, p.k = (int)d.k, p.group = (int)d.group;
    p.groups = (int)((d.k + d.group - 1) / d.group);
    p.xvec = aligned16(d.x) && d.ldx % (d.dtype == GFH_F32 ? 4 : 8) == 0;
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
    if (d.m <= kRowsMax) {
        // eight rows of W per workgroup where that leaves two for every CU
        const bool eight = d.n >= 8 * 2 * device_cu_count();
        typed([&](auto t) {
            using T = decltype(t);
            auto go = [&](auto mc) {
                constexpr int M = decltype(mc)::value;
                if (eight)
                    hipLaunchKernelGGL((w4_rows_kernel<T, M, 8>), dim3((unsigned)((d.n + 7) / 8)), dim3(256), 0, s, p);
                else
                    hipLaunchKernelGGL((w4_rows_kernel<T, M, 4>), dim3((unsigned)((d.n + 3) / 4)), dim3(256), 0, s, p);
            };
            if (d.m == 1)
                go(std::integral_constant<int, 1>{});
            else if (d.m == 2)
                go(std::integral_constant<int, 2>{});
            else
                go(std::integral_constant<int, 4>{});
        });
        return check_launch("linear_w4");
    }
    const W4Plan pl = w4_plan(d);
    p.splits = pl.splits;
    p.kper = pl.kper;
    const int64_t gx = (d.n + 64 * pl.rt - 1) / (64 * pl.rt) * pl.splits, gy = (d.m + 16 * pl.mb - 1) / (16 * pl.mb);
    if (gx > (1 << 23) || gy > 65535) return set_error(GFH_INVALID_SHAPE, "linear_w4: grid too large");
    const dim3 grid((unsigned)gx, (unsigned)gy);
    typed([&](auto t) {
        using T = decltype(t);
        auto go = [&](auto mb, auto rt) {
            constexpr int MB = decltype(mb)::value, RT = decltype(rt)::value;
            if (d.group % 128 == 0)
                hipLaunchKernelGGL((w4_tiles_kernel<T, MB, RT, false>), grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((w4_tiles_kernel<T, MB, RT, true>), grid, dim3(256), 0, s, p);
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        using Four = std::integral_constant<int, 4>;
        if (pl.mb == 1)
            go(One{}, One{});
        else if (pl.mb == 2)
            go(Two{}, Two{});
        else if constexpr (!std::is_same_v<T, float>)
            go(Four{}, Two{});
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
