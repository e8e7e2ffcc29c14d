// Grouped products of few rows with 4-bit weights (gg_gemm_w4 in include/gg_moe_layer.h):
// out[m, n] = sum_k x[m, k] s (q[n, k] - z), s and z of each `group` consecutive k.
//
// What bounds it: the packed weights of the groups that have rows, read once. A wave takes 16 weight rows
// (NT such tiles) and every W-th tile of 128 k; a tile is one 16-byte load per lane, 1 KB in a row, and
// the operand of four 16x16x32 matrix instructions. A nibble becomes a 16-bit float by three bit
// operations on a word, two nibbles at a time: rotated to the top of the mantissa of 16.0 it is 16 + q,
// exact in bf16 and fp16. The products therefore sum x (16 + q); the scale's share of the sum,
// s (sum x (16 + q) - (16 + z) sum x), takes sum x from one more matrix instruction whose weights are
// ones. Nothing is rounded before the float32 sums. The W partial sums are added through LDS.
#include <algorithm>

#include "gg_layer.h"

namespace gg {
namespace layer {
namespace {

typedef __bf16   bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct W4Args {
    const int64_t *lens, *offs;
    const void    *x, *packed, *scales;
    const uint8_t *zeros;
    void          *out;
    int64_t        total_m;
    int            group_num, n, k, n_tiles, k_tiles, groups; // groups: scales along k
};

template <typename T> struct W4Type;
template <> struct W4Type<BF16> {
    static constexpr unsigned mask = 0x00780078u, sixteen = 0x41804180u, one = 0x3f803f80u;
    static constexpr int      shift = 3; // of q's lowest bit in the half word
    static __device__ __forceinline__ f32x4 mma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct W4Type<F16> {
    static constexpr unsigned mask = 0x03c003c0u, sixteen = 0x4c004c00u, one = 0x3c003c00u;
    static constexpr int      shift = 6;
    static __device__ __forceinline__ f32x4 mma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Eight nibbles of a word as 16 + q: element 2 i from nibble i, 2 i + 1 from nibble i + 4.
template <typename T> __device__ __forceinline__ u32x4 expand(unsigned w) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned turned = __builtin_amdgcn_alignbit(w, w, (4 * i - W4Type<T>::shift) & 31);
        r[i]                  = (turned & W4Type<T>::mask) | W4Type<T>::sixteen;
    }
    return r;
}

// The `want`-th group with rows: its number, or -1, its first row and its rows. A bad length counts as no
// rows, a group that does not lie inside [0, total_m) has no work.
struct Found {
    int     group;
    int64_t row0;
    int     rows;
};
__device__ __forceinline__ Found find_group(const W4Args &a, int want, int lane) {
    int64_t base = 0; // rows of the groups before this window of 64
    for (int g0 = 0; g0 < a.group_num; g0 += 64) {
        const int g   = g0 + lane;
        int64_t   len = g < a.group_num ? a.lens[g] : 0;
        if (len < 0 || len > INT32_MAX)
            len = 0;
        int64_t incl = len;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(incl, d);
            incl += lane >= d ? o : 0;
        }
        const int64_t  row0 = a.offs != nullptr ? (g < a.group_num ? a.offs[g] : 0) : base + incl - len;
        const bool     ok   = len > 0 && row0 >= 0 && row0 <= a.total_m && len <= a.total_m - row0;
        const uint64_t have = __ballot(ok);
        const int      n    = __builtin_popcountll(have);
        if (want < n) {
            uint64_t m = have;
            for (int i = 0; i < want; ++i)
                m &= m - 1;
            const int src = __builtin_ctzll(m);
            Found     f;
            f.group = g0 + src;
            f.row0  = __shfl(row0, src);
            f.rows  = static_cast<int>(__shfl(len, src));
            return f;
        }
        want -= n;
        base += __shfl(incl, 63);
    }
    return {-1, 0, 0};
}

// Grid: workgroup (tile block of 16 NT columns, one of the groups with rows). MT row tiles of 16 at a time.
// G: k of one scale.
template <typename T, int MT, int NT, int W, int G> __global__ void __launch_bounds__(W * 64) w4_kernel(const W4Args a) {
    using X = W4Type<T>;
    __shared__ f32x4 part[W][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int blocks = (a.n_tiles + NT - 1) / NT;
    const int nb     = static_cast<int>(blockIdx.x) % blocks;
    const int slots  = static_cast<int>(gridDim.x) / blocks;
    for (int want = static_cast<int>(blockIdx.x) / blocks;; want += slots) {
        const Found f = find_group(a, want, lane);
        if (f.group < 0)
            return;
        const int   tile0 = nb * NT;
        const char *wp[NT], *sp[NT], *zp[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int64_t tile = static_cast<int64_t>(f.group) * a.n_tiles + min(tile0 + i, a.n_tiles - 1); // past N: the last again
            wp[i] = static_cast<const char *>(a.packed) + tile * a.k_tiles * 1024 + lane * 16;
            sp[i] = static_cast<const char *>(a.scales) + tile * a.groups * 32 + quad * 8;
            zp[i] = reinterpret_cast<const char *>(a.zeros) + tile * a.groups * 16 + quad * 4;
        }
        for (int m0 = 0; m0 < f.rows; m0 += 16 * MT) {
            const uint16_t *xp[MT];
            bool            has[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int m = m0 + 16 * i + col;
                has[i]      = m < f.rows;
                xp[i]       = static_cast<const uint16_t *>(a.x) + (f.row0 + (has[i] ? m : 0)) * a.k + quad * 8;
            }
            f32x4 acc[MT][NT];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int c = wave; c < a.k_tiles; c += W) {
                u32x4 wv[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    wv[j] = *reinterpret_cast<const u32x4 *>(wp[j] + static_cast<int64_t>(c) * 1024);
                constexpr int kSteps = G / 32; // matrix instructions of one scale
#pragma unroll
                for (int q = 0; q < 4 / kSteps; ++q) { // scales of this tile
                    const int sg = c * (128 / G) + q;
                    if (sg >= a.groups) // past K
                        break;
                    f32x4 sum[MT][NT], ones[MT];
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        ones[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) {
                        const int step = q * kSteps + st;
                        u32x4     xv[MT];
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            xv[i] = u32x4{0, 0, 0, 0};
                            if (has[i])
                                xv[i] = *reinterpret_cast<const u32x4 *>(xp[i] + static_cast<int64_t>(c) * 128 + step * 32);
                        }
                        const u32x4 one{X::one, X::one, X::one, X::one};
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            ones[i] = X::mma(one, xv[i], ones[i]);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const u32x4 wf = expand<T>(wv[j][step]);
#pragma unroll
                            for (int i = 0; i < MT; ++i)
                                sum[i][j] = X::mma(wf, xv[i], sum[i][j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float       s[4], z[4];
                        const u32x2 sw = *reinterpret_cast<const u32x2 *>(sp[j] + static_cast<int64_t>(sg) * 32);
                        T::pair(sw[0], s[0], s[1]);
                        T::pair(sw[1], s[2], s[3]);
                        if (a.zeros != nullptr) {
                            const unsigned zw = *reinterpret_cast<const unsigned *>(zp[j] + static_cast<int64_t>(sg) * 16);
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                z[r] = static_cast<float>((zw >> (8 * r)) & 255u) + 16.f;
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                z[r] = 24.f;
                        }
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                acc[i][j][r] = fmaf(s[r], fmaf(-z[r], ones[i][r], sum[i][j][r]), acc[i][j][r]);
                    }
                }
            }
            // the waves' sums, in their order; each wave stores every W-th of the MT x NT tiles
            __syncthreads(); // the tiles before are read
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    part[wave][i * NT + j][lane] = acc[i][j];
            __syncthreads();
            for (int u = wave; u < MT * NT; u += W) {
                f32x4 v = part[0][u][lane];
#pragma unroll
                for (int w = 1; w < W; ++w)
                    v += part[w][u][lane];
                const int m = m0 + 16 * (u / NT) + col, n = (tile0 + u % NT) * 16 + quad * 4;
                if (m < f.rows && n < a.n) // n % 8 == 0: four columns are all there or none
                    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + (f.row0 + m) * a.n + n) =
                        u32x2{T::word(v[0], v[1]), T::word(v[2], v[3])};
            }
        }
    }
}

template <typename T, int MT, int NT, int W> int launch_w4(const W4Args &a, int group, hipStream_t s) {
    const int64_t blocks = (a.n_tiles + NT - 1) / NT;
    // at most total_m groups have rows (device offsets that overlap may give more: slots are walked in strides);
    // HIP refuses grids of 2^32 threads
    const int64_t slots = std::clamp<int64_t>(std::min<int64_t>(a.group_num, a.total_m), 1, (int64_t(1) << 31) / (W * 64) / blocks);
    const int64_t grid  = blocks * slots;
    return launch("gemm_w4", group == 128 ? w4_kernel<T, MT, NT, W, 128> : group == 64 ? w4_kernel<T, MT, NT, W, 64> : w4_kernel<T, MT, NT, W, 32>,
                  grid, W * 64, s, a);
}

template <typename T> int run_w4(const W4Args &a, int group, hipStream_t s) { return launch_w4<T, 1, 1, 8>(a, group, s); }

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" int gg_gemm_w4(int dtype, int group_num, int64_t total_m, int64_t n, int64_t k, int group,
                          const int64_t *group_lens, const int64_t *group_offs, const void *x, const void *packed,
                          const void *scales, const uint8_t *zeros, void *out, void *stream) {
    g_error[0] = 0;
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (group_num < 0 || total_m < 0 || n < 0 || k < 1)
        return fail(GG_ERR_INVALID, "group_num, total_m and n must be >= 0 and k >= 1");
    if (group != 32 && group != 64 && group != 128)
        return fail(GG_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
    if (n % 8 != 0 || k % group != 0)
        return fail(GG_ERR_UNSUPPORTED, "N must be a multiple of 8 and K of group");
    if (n > (1 << 21) || k > (1 << 21) || group_num > 8192)
        return fail(GG_ERR_UNSUPPORTED, "N and K must be at most 2097152 and groups at most 8192");
    if (group_num == 0 || total_m == 0 || n == 0)
        return GG_OK;
    if (group_lens == nullptr || x == nullptr || packed == nullptr || scales == nullptr || out == nullptr)
        return fail(GG_ERR_INVALID, "group_lens, x, packed, scales and out must be device pointers");
    if (!aligned(x, 16) || !aligned(packed, 16) || !aligned(scales, 16) || !aligned(out, 16) || !aligned(zeros, 4))
        return fail(GG_ERR_UNSUPPORTED, "x, packed, scales and out must be 16-byte aligned, zeros 4-byte");
    W4Args a{};
    a.lens      = group_lens;
    a.offs      = group_offs;
    a.x         = x;
    a.packed    = packed;
    a.scales    = scales;
    a.zeros     = zeros;
    a.out       = out;
    a.total_m   = total_m;
    a.group_num = group_num;
    a.n         = static_cast<int>(n);
    a.k         = static_cast<int>(k);
    a.n_tiles   = static_cast<int>((n + 15) / 16);
    a.k_tiles   = static_cast<int>((k + 127) / 128);
    a.groups    = static_cast<int>(k / group);
    return dtype == GG_DTYPE_BF16 ? run_w4<BF16>(a, group, static_cast<hipStream_t>(stream))
                                  : run_w4<F16>(a, group, static_cast<hipStream_t>(stream));
}
