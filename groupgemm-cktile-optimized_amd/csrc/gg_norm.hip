// RMS norm with the residual's addition, 16-bit or fp8 output, and its gradients (gg_rms_norm,
// gg_rms_norm_backward in include/gg_moe_layer.h).
//
// Forward: h = round(x + r), rstd = (mean h^2 + eps)^-1/2, y = h rstd w. A row stays in the registers
// of the waves that work on it (one wave up to 1024 values, four up to 16384, of few rows up to 2048, else sixteen), so
// x and r are read once and h and y written once: bound by HBM. The tensor scale needs the largest |y|
// of all rows before the first value is rounded: a first pass writes h, rstd and one maximum per
// workgroup, a second reads h again and rounds.
//
// The norm is taken of the rounded h, the value that later layers and the backward pass read, so the
// passes agree whatever the scale.
//
// Measured: 32768 rows of 7168, bf16 with residual to fp8 with a tensor scale, 377 us: 245 for the first pass (x and r
// read, h written: 5.8 TB/s) and 133 for the second (h read, y written: 5.3); 5 rows to bf16 3.8, the latency of a launch,
// a row's loads and a barrier. Backward 16640 x 2880 with a gradient past the norm: 75 us, 5.1 TB/s (69 row by row, 6 for
// the weight's gradient).
#include "gg_layer.h"

#include <algorithm>

namespace gg {
namespace layer {

thread_local char g_error[256] = "";

namespace {

constexpr int kMaxParts = GG_NORM_WORKSPACE / 4; // workgroups of a tensor scale's first pass

struct NormArgs {
    const void *x, *residual, *weight;
    void       *h, *y;
    float      *rstd, *scale, *parts;
    int64_t     rows, x_stride, r_stride, h_stride;
    int         hidden, mode, n_parts;
    float       eps;
    bool        w32, e5m2;
};

// Eight weights from element i on, as float32.
template <typename T> __device__ __forceinline__ void load_w(const void *w, bool w32, int i, float (&v)[8]) {
    if (w32) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(w) + i);
        const f32x4  a = p[0], b = p[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j]     = a[j];
            v[4 + j] = b[j];
        }
    } else {
        unpack8<T>(*reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(w) + i), v);
    }
}

// Saturates (the conversion would give NaN past the largest value); a NaN stays one.
__device__ __forceinline__ float saturate(float v, float top) { return v != v ? v : fminf(fmaxf(v, -top), top); }

// Division by a scale, rounded as a float32 division is: the product with the rounded reciprocal, corrected once by its
// remainder, which a fused multiply-add gives exactly (Markstein 1990). By the product alone one in sixty of the values
// within two float32 units of a tie of the format went to the neighbouring code. The product is clamped first, far past
// either format's range, so that the remainder stays finite; a NaN comes back with the remainder. Outside 2^-64 .. 2^64
// the remainder could be subnormal, and `exact` divides.
struct Divisor {
    float s, inv;
    bool  exact;
    __device__ __forceinline__ explicit Divisor(float scale)
        : s(scale), inv(1.f / scale), exact(!(fabsf(scale) >= 0x1p-64f && fabsf(scale) <= 0x1p64f)) {}
    __device__ __forceinline__ float quotient(float v) const {
        const float q = __builtin_amdgcn_fmed3f(v * inv, -131072.f, 131072.f);
        return fmaf(-fmaf(q, s, -v), inv, q); // (in this order of signs a zero keeps its own)
    }
};

// Eight values divided by the scale, as fp8.
__device__ __forceinline__ u32x2 pack_fp8(const float (&v)[8], const Divisor &d, bool e5m2) {
    u32x2 w;
    const float top = e5m2 ? 57344.f : 448.f;
    float s[8];
    if (d.exact) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s[i] = saturate(v[i] / d.s, top);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            s[i] = saturate(d.quotient(v[i]), top);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int q = 0;
        if (e5m2) {
            q = __builtin_amdgcn_cvt_pk_bf8_f32(s[4 * i], s[4 * i + 1], q, false);
            q = __builtin_amdgcn_cvt_pk_bf8_f32(s[4 * i + 2], s[4 * i + 3], q, true);
        } else {
            q = __builtin_amdgcn_cvt_pk_fp8_f32(s[4 * i], s[4 * i + 1], q, false);
            q = __builtin_amdgcn_cvt_pk_fp8_f32(s[4 * i + 2], s[4 * i + 3], q, true);
        }
        w[i] = static_cast<unsigned>(q);
    }
    return w;
}

// Scale of the largest |y| (bits of a float >= 0 or NaN): 1 where the quotient is zero or subnormal, which a division
// by it could turn into NaN or a value of few bits.
__device__ __forceinline__ float scale_of(unsigned top_bits, bool e5m2) {
    const float s = __uint_as_float(top_bits) / (e5m2 ? 57344.f : 448.f);
    return s < 1.17549435e-38f ? 1.f : s;
}

// Reductions over the WPR waves of a row; `turn` alternates so that one barrier per call is enough.
template <int WPR> struct RowReduce {
    float    sums[2][WPR];
    unsigned tops[2][WPR];
};
template <int WPR> __device__ __forceinline__ float row_sum(RowReduce<WPR> &m, int turn, float v, int wave, int lane) {
    v = wave_sum(v);
    if constexpr (WPR == 1)
        return v;
    if (lane == 0)
        m.sums[turn][wave] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i)
        s += m.sums[turn][i];
    return s;
}
template <int WPR> __device__ __forceinline__ unsigned row_max(RowReduce<WPR> &m, int turn, unsigned v, int wave, int lane) {
    v = wave_max(v);
    if constexpr (WPR == 1)
        return v;
    if (lane == 0)
        m.tops[turn][wave] = v;
    __syncthreads();
    unsigned s = 0;
#pragma unroll
    for (int i = 0; i < WPR; ++i)
        s = max(s, m.tops[turn][i]);
    return s;
}

constexpr int block_threads(int wpr) { return wpr == 1 ? 256 : 64 * wpr; }
constexpr int rows_per_block(int wpr) { return wpr == 1 ? 4 : 1; }

// One pass over the rows. FIRST: the first pass of a tensor scale (no y; the workgroup's largest |y|).
template <typename T, int WPR, int U, bool FIRST>
__global__ void __launch_bounds__(block_threads(WPR)) norm_kernel(const NormArgs a) {
    __shared__ RowReduce<WPR> m;
    __shared__ unsigned       block_top[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t    = WPR == 1 ? lane : static_cast<int>(threadIdx.x); // thread of the row
    unsigned  top  = 0;
    int       turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * rows_per_block(WPR);
    // every wave of a block that shares a row makes the same trips, so the barriers match
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_block(WPR) + (WPR == 1 ? wave : 0); row < a.rows;
         row += step, turn ^= 1) {
        float v[U][8];
        float sq = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[u][j] = 0.f;
            if (i < a.hidden) {
                const u32x4 xw = load_once(static_cast<const uint16_t *>(a.x) + row * a.x_stride + i);
                unpack8<T>(xw, v[u]);
                if (a.residual != nullptr) {
                    float r[8];
                    unpack8<T>(load_once(static_cast<const uint16_t *>(a.residual) + row * a.r_stride + i), r);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[u][j] += r[j];
                    const u32x4 hw = pack8<T>(v[u]);
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.h) + row * a.h_stride + i) = hw;
                    unpack8<T>(hw, v[u]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    sq = fmaf(v[u][j], v[u][j], sq);
            }
        }
        sq = row_sum<WPR>(m, turn, sq, wave, lane);
        const float rstd = 1.f / sqrtf(sq / static_cast<float>(a.hidden) + a.eps);
        if (t == 0 && a.rstd != nullptr)
            a.rstd[row] = rstd;
        unsigned row_top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.hidden) {
                float w[8];
                load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[u][j] = v[u][j] * rstd * w[j];
                    row_top = max(row_top, __float_as_uint(fabsf(v[u][j])));
                }
            }
        }
        if constexpr (FIRST) {
            top = max(top, row_top);
        } else {
            float s = 1.f;
            if (a.mode == GG_NORM_SCALE_ROW) {
                s = scale_of(row_max<WPR>(m, turn, row_top, wave, lane), a.e5m2);
                if (t == 0)
                    a.scale[row] = s;
            } else if (a.mode == GG_NORM_SCALE_GIVEN) {
                s = a.scale[0];
            }
            const Divisor by(s);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = (u * 64 * WPR + t) * 8;
                if (i < a.hidden) {
                    if (a.mode == GG_NORM_PLAIN) {
                        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.y) + row * a.hidden + i) = pack8<T>(v[u]);
                    } else {
                        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + row * a.hidden + i) = pack_fp8(v[u], by, a.e5m2);
                    }
                }
            }
        }
    }
    if constexpr (FIRST) {
        top = wave_max(top);
        constexpr int waves = block_threads(WPR) / 64;
        static_assert(waves <= 16, "");
        if constexpr (WPR == 1) {
            if (lane == 0)
                block_top[wave] = top;
        } else {
            __syncthreads(); // the last row's tops are read
            if (lane == 0)
                m.tops[0][wave] = top;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned s = 0;
            for (int i = 0; i < waves; ++i)
                s = max(s, WPR == 1 ? block_top[i & 3] : m.tops[0][i % WPR]);
            reinterpret_cast<unsigned *>(a.parts)[blockIdx.x] = s;
        }
    }
}

// The tensor scale's second pass: the largest of the first pass's maxima, then y from h and rstd.
template <typename T, int THREADS> __global__ void __launch_bounds__(THREADS) quantize_kernel(const NormArgs a) {
    __shared__ unsigned tops[THREADS / 64];
    unsigned            top = 0;
    for (int i = threadIdx.x; i < a.n_parts; i += THREADS)
        top = max(top, reinterpret_cast<const unsigned *>(a.parts)[i]);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0)
        tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i)
        top = max(top, tops[i]);
    const float   s = scale_of(top, a.e5m2);
    const Divisor by(s);
    if (blockIdx.x == 0 && threadIdx.x == 0)
        a.scale[0] = s;
    // from the last row backwards: the rows written last are still in the Infinity Cache
    for (int64_t row = a.rows - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
        const float rstd = a.rstd[row];
        for (int i = threadIdx.x * 8; i < a.hidden; i += THREADS * 8) {
            float v[8], w[8];
            unpack8<T>(load_once(static_cast<const uint16_t *>(a.h) + row * a.h_stride + i), v);
            load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = v[j] * rstd * w[j];
            *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + row * a.hidden + i) = pack_fp8(v, by, a.e5m2);
        }
    }
}

struct BackArgs {
    const void  *g, *h, *weight, *gh;
    const float *rstd;
    void        *gx;
    float       *parts; // [workgroups][hidden] partial sums of grad_weight
    int64_t      rows, g_stride, h_stride, gh_stride;
    int          hidden;
    bool         w32;
};

// grad_x row by row; grad_weight's partial sums stay in registers over the rows of a workgroup and are
// written once.
template <typename T, int WPR, int U, bool SUMS>
__global__ void __launch_bounds__(block_threads(WPR)) norm_back_kernel(const BackArgs a) {
    __shared__ RowReduce<WPR> m;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t    = WPR == 1 ? lane : static_cast<int>(threadIdx.x);
    float     dw[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            dw[u][j] = 0.f;
    int           turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * rows_per_block(WPR);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_block(WPR) + (WPR == 1 ? wave : 0); row < a.rows;
         row += step, turn ^= 1) {
        u32x4 gw[U], hw[U], rw[U];
        float dot = 0.f;
        const float rstd = a.rstd[row];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.hidden) {
                gw[u] = load_once(static_cast<const uint16_t *>(a.g) + row * a.g_stride + i);
                hw[u] = load_once(static_cast<const uint16_t *>(a.h) + row * a.h_stride + i);
                if (a.gh != nullptr)
                    rw[u] = load_once(static_cast<const uint16_t *>(a.gh) + row * a.gh_stride + i);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.hidden) {
                float g[8], h[8], w[8];
                unpack8<T>(gw[u], g);
                unpack8<T>(hw[u], h);
                load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    dot      = fmaf(g[j] * w[j], h[j], dot);
                    if constexpr (SUMS)
                        dw[u][j] = fmaf(g[j] * h[j], rstd, dw[u][j]);
                }
            }
        }
        dot = row_sum<WPR>(m, turn, dot, wave, lane);
        const float c = rstd * (rstd * (rstd * (dot / static_cast<float>(a.hidden)))); // (rstd^3 alone may be past float32)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.hidden) {
                float g[8], h[8], w[8], r[8];
                unpack8<T>(gw[u], g);
                unpack8<T>(hw[u], h);
                load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    g[j] = rstd * (g[j] * w[j]) - h[j] * c;
                if (a.gh != nullptr) {
                    unpack8<T>(rw[u], r);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        g[j] += r[j];
                }
                *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.gx) + row * a.hidden + i) = pack8<T>(g);
            }
        }
    }
    if constexpr (!SUMS)
        return;
    // a workgroup whose waves had rows of their own adds them up first, in their order
    if constexpr (WPR == 1) {
        __shared__ f32x4 mine[3][U][2][64];
        if (wave > 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    mine[wave - 1][u][q][lane] = f32x4{dw[u][4 * q], dw[u][4 * q + 1], dw[u][4 * q + 2], dw[u][4 * q + 3]};
        __syncthreads();
        if (wave > 0)
            return;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int o = 0; o < 3; ++o)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        dw[u][4 * q + j] += mine[o][u][q][lane][j];
    }
    float *part = a.parts + static_cast<int64_t>(blockIdx.x) * a.hidden;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 * WPR + t) * 8;
        if (i < a.hidden) {
            f32x4 *p = reinterpret_cast<f32x4 *>(part + i);
            p[0]     = f32x4{dw[u][0], dw[u][1], dw[u][2], dw[u][3]};
            p[1]     = f32x4{dw[u][4], dw[u][5], dw[u][6], dw[u][7]};
        }
    }
}

// grad_weight from g and h themselves: 64 columns (a line of 128 bytes a row) by 128 slices of the rows a workgroup.
template <typename T> __global__ void __launch_bounds__(1024) weight_strip_kernel(const BackArgs a, void *out) {
    __shared__ f32x4 sums[2][128][8];
    const int c8 = threadIdx.x & 7, slice = threadIdx.x >> 3, col = blockIdx.x * 64 + c8 * 8; // hidden % 8 == 0
    f32x4     s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    if (col < a.hidden) {
        const uint16_t *g = static_cast<const uint16_t *>(a.g) + col, *h = static_cast<const uint16_t *>(a.h) + col;
#pragma unroll 4
        for (int64_t row = slice; row < a.rows; row += 128) {
            float gv[8], hv[8];
            unpack8<T>(*reinterpret_cast<const u32x4 *>(g + row * a.g_stride), gv);
            unpack8<T>(*reinterpret_cast<const u32x4 *>(h + row * a.h_stride), hv);
            const float rstd = a.rstd[row];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s[j / 4][j % 4] = fmaf(gv[j] * hv[j], rstd, s[j / 4][j % 4]);
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
        sums[q][slice][c8] = s[q];
    __syncthreads();
#pragma unroll
    for (int half = 64; half > 0; half >>= 1) {
        if (slice < half)
#pragma unroll
            for (int q = 0; q < 2; ++q)
                sums[q][slice][c8] = s[q] += sums[q][slice + half][c8];
        __syncthreads();
    }
    if (slice == 0 && col < a.hidden) {
        if (a.w32) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
                reinterpret_cast<f32x4 *>(static_cast<float *>(out) + col)[q] = s[q];
        } else {
            const float v[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]};
            *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(out) + col) = pack8<T>(v);
        }
    }
}

// grad_weight: the sum of the partial sums of each column, in a fixed order; 32 columns by 128 slices of the parts a
// workgroup.
template <typename T>
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float *parts, int n_parts, int hidden, void *out, bool w32) {
    __shared__ f32x4 sums[128][8];
    const int c4 = threadIdx.x & 7, slice = threadIdx.x >> 3, col = blockIdx.x * 32 + c4 * 4; // hidden % 8 == 0
    f32x4     s{0.f, 0.f, 0.f, 0.f};
    if (col < hidden)
#pragma unroll 8
        for (int p = slice; p < n_parts; p += 128)
            s += *reinterpret_cast<const f32x4 *>(parts + static_cast<int64_t>(p) * hidden + col);
    sums[slice][c4] = s;
    __syncthreads();
#pragma unroll
    for (int half = 64; half > 0; half >>= 1) {
        if (slice < half)
            sums[slice][c4] = s += sums[slice + half][c4];
        __syncthreads();
    }
    if (slice == 0 && col < hidden) {
        if (w32)
            *reinterpret_cast<f32x4 *>(static_cast<float *>(out) + col) = s;
        else
            *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + col) = u32x2{T::word(s[0], s[1]), T::word(s[2], s[3])};
    }
}

// Few rows: a row's latency counts, and not how many are in flight. Then (WIDE) sixteen waves take a row of more than 2048
// values, and grad_weight is summed from g and h again, which are in the caches, instead of from partial sums, which would be
// as many bytes as the rows. us, sixteen waves and four: norm of 5 rows of 7168 3.9, 5.1, of 256 5.5, 7.3, 512 8.4, 10.8, 1024
// 14.5, 14.8; of 512 rows of 4096 5.7, 5.6, 1024 10.8, 9.5; 256 of 14336 8.5, 14.0. Backward, with the sums and without:
// 64 of 7168 7.1, 9.1, 481 of 13456 22.2, 34.3, 512 of 7168 16.6, 18.1, 512 of 4096 13.9, 12.4, 1024 of 8192 27.6, 27.4.
bool few(int64_t rows, int64_t hidden) { return hidden > 1024 && rows <= (hidden > 5120 ? 512 : 256); }

template <bool WIDE> int waves_per_row(int64_t hidden) {
    return hidden <= 1024 ? 1 : hidden <= (WIDE ? 2048 : 16384) ? 4 : 16;
}

int64_t row_blocks(int64_t rows, int64_t hidden) { return hidden <= 1024 ? (rows + 3) / 4 : rows; }

// f(WPR, U) of the instance for `hidden` values a row: U pieces of 8 per lane.
template <bool WIDE, typename F> int with_shape(int64_t hidden, F f) {
    using std::integral_constant;
    const int wpr = waves_per_row<WIDE>(hidden), u = static_cast<int>((hidden + 512 * wpr - 1) / (512 * wpr));
#define GG_SHAPE(W, N)                                                                                                 \
    if (wpr == W && u <= N)                                                                                            \
        return f(integral_constant<int, W>{}, integral_constant<int, N>{});
    GG_SHAPE(1, 1) GG_SHAPE(1, 2) GG_SHAPE(4, 1)
    if constexpr (WIDE) {
        GG_SHAPE(16, 1) GG_SHAPE(16, 2)
    } else {
        GG_SHAPE(4, 2) GG_SHAPE(4, 3) GG_SHAPE(4, 4) GG_SHAPE(4, 6) GG_SHAPE(4, 8)
    }
#undef GG_SHAPE
    return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
}

constexpr int64_t kMaxBlocks = int64_t(1) << 20;

template <typename T, bool WIDE> int run_norm(const NormArgs &a, hipStream_t s) {
    const int64_t blocks = row_blocks(a.rows, a.hidden);
    if (a.mode != GG_NORM_SCALE_TENSOR)
        return with_shape<WIDE>(a.hidden, [&](auto wpr, auto u) {
            return launch("rms_norm", norm_kernel<T, wpr.value, u.value, false>, std::min(blocks, kMaxBlocks),
                          block_threads(wpr.value), s, a);
        });
    // The first pass: as many workgroups as fit at once, each with its share of the rows (32768 rows of 7168: 1792
    // workgroups fit, 377 us for both passes; 1536 377, 1280 389, 1024 421, 2048, 1.1 rounds of them, 453).
    NormArgs b = a;
    if (b.residual == nullptr) { // h is x
        b.h        = const_cast<void *>(b.x);
        b.h_stride = b.x_stride;
    }
    const int st = with_shape<WIDE>(a.hidden, [&](auto wpr, auto u) {
        constexpr auto kernel = norm_kernel<T, wpr.value, u.value, true>;
        // (asked for each call, as devices differ; few workgroups fit in any case)
        b.n_parts = static_cast<int>(blocks <= 256 ? blocks : std::min<int64_t>(blocks, std::min(resident_blocks(kernel, block_threads(wpr.value)), kMaxParts)));
        return launch("rms_norm", kernel, b.n_parts, block_threads(wpr.value), s, b);
    });
    constexpr int kThreads = WIDE ? 1024 : 256;
    return st ? st : launch("rms_norm", quantize_kernel<T, kThreads>, std::min<int64_t>(b.rows, 8192), kThreads, s, b);
}

// Workgroups of the backward pass: at most those that 256 CUs hold at once (by the instances' registers, 68 to 224: numbers
// that a test holds to the compiler's report, as the size of the workspace is asked for without a device or a type; 1024
// to two pieces and one wave a row, where 1280 fit), fewer where each would have less than four rows and their partial sums would cost more than they save. us at 1, 2
// and 4 rows each, of 7168: 512 rows 19.9, 18.6, 21.6; 2048 46.8, 37.9, 34.2. At once against 1024:
// 16640 rows of 2880 73.7 (1536) and 77.6, 4096 of 14336 108.5 (512) and 118.6.
int64_t back_blocks(int64_t rows, int64_t hidden) {
    const int     wpr = waves_per_row<false>(hidden), u = static_cast<int>((hidden + 512 * wpr - 1) / (512 * wpr));
    const int64_t fit = wpr == 16 ? 256 : u == 1 ? 1792 : u > 4 ? 512 : u == 2 && wpr == 4 ? 1536 : 1024;
    const int64_t b   = row_blocks(rows, hidden);
    return std::min(fit, std::max(b / 4, b <= 256 ? b : std::min<int64_t>(b / 2, 512)));
}

template <typename T> int run_back(const BackArgs &a, void *grad_weight, hipStream_t s) {
    if (few(a.rows, a.hidden)) { // (grad_weight first: grad_x may take the place of an input)
        const int st = launch("rms_norm_backward", weight_strip_kernel<T>, (a.hidden + 63) / 64, 1024, s, a, grad_weight);
        return st ? st : with_shape<true>(a.hidden, [&](auto wpr, auto u) {
            return launch("rms_norm_backward", norm_back_kernel<T, wpr.value, u.value, false>, row_blocks(a.rows, a.hidden),
                          block_threads(wpr.value), s, a);
        });
    }
    const int st = with_shape<false>(a.hidden, [&](auto wpr, auto u) {
        return launch("rms_norm_backward", norm_back_kernel<T, wpr.value, u.value, true>, back_blocks(a.rows, a.hidden),
                      block_threads(wpr.value), s, a);
    });
    return st ? st : launch("rms_norm_backward", weight_sum_kernel<T>, (a.hidden + 31) / 32, 1024, s, a.parts,
                            static_cast<int>(back_blocks(a.rows, a.hidden)), a.hidden, grad_weight, a.w32);
}

// Rules shared by both passes.
int check_norm(int dtype, int weight_dtype, int64_t rows, int64_t hidden) {
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (weight_dtype != dtype && weight_dtype != GG_DTYPE_FP32)
        return fail(GG_ERR_INVALID, "weight_dtype must be dtype or GG_DTYPE_FP32");
    if (rows < 0 || hidden < 1)
        return fail(GG_ERR_INVALID, "rows must be >= 0 and hidden >= 1");
    if (hidden % 8 != 0 || hidden > 32768)
        return fail(GG_ERR_UNSUPPORTED, "hidden must be a multiple of 8 and at most 32768");
    return GG_OK;
}
// A matrix operand: rows at least hidden apart, 16-byte pieces.
int check_rows(const char *name, const void *p, int64_t stride, int64_t rows) {
    if (rows > 0 && p == nullptr)
        return fail(GG_ERR_INVALID, "%s is null", name);
    if (rows > 1 && stride < 0)
        return fail(GG_ERR_INVALID, "%s has a negative row stride", name);
    if (!aligned(p, 16) || (rows > 1 && stride % 8 != 0))
        return fail(GG_ERR_UNSUPPORTED, "%s must be 16-byte aligned with row strides of multiples of 8", name);
    return GG_OK;
}

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

const char *gg_layer_last_error(void) { return g_error; }

int gg_rms_norm(int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden, float eps,
                const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                void *h, int64_t h_stride, void *y, float *rstd, float *scale, void *workspace, void *stream) {
    g_error[0] = 0;
    if (const int st = check_norm(dtype, weight_dtype, rows, hidden))
        return st;
    if (scale_mode < GG_NORM_PLAIN || scale_mode > GG_NORM_SCALE_GIVEN)
        return fail(GG_ERR_INVALID, "scale_mode must be a gg_norm_scale");
    if (scale_mode == GG_NORM_PLAIN ? out_dtype != dtype : !is8(out_dtype))
        return fail(GG_ERR_INVALID, "out_dtype must be dtype, or an fp8 type with a scale");
    if (scale_mode != GG_NORM_PLAIN && scale == nullptr && (rows > 0 || scale_mode != GG_NORM_SCALE_ROW)) // (a row scale of no rows)
        return fail(GG_ERR_INVALID, "scale is null");
    if (rows == 0 && scale_mode != GG_NORM_SCALE_TENSOR)
        return GG_OK;
    if (weight == nullptr || (rows > 0 && y == nullptr))
        return fail(GG_ERR_INVALID, "weight and y must be device pointers");
    if (scale_mode == GG_NORM_SCALE_TENSOR && (workspace == nullptr || (rows > 0 && rstd == nullptr)))
        return fail(GG_ERR_INVALID, "a tensor scale needs workspace and rstd");
    if (const int st = check_rows("x", x, x_stride, rows))
        return st;
    if (residual != nullptr) {
        if (const int st = check_rows("residual", residual, residual_stride, rows))
            return st;
        if (const int st = check_rows("h", h, h_stride, rows))
            return st;
        if (rows > 1 && h_stride < hidden)
            return fail(GG_ERR_INVALID, "rows of h overlap");
    }
    if (!aligned(weight, 16) || !aligned(y, scale_mode == GG_NORM_PLAIN ? 16 : 8) || !aligned(workspace, 4))
        return fail(GG_ERR_UNSUPPORTED, "weight and y must be 16-byte aligned (fp8 y: 8)");
    NormArgs a{};
    a.x        = x;
    a.residual = residual;
    a.weight   = weight;
    a.h        = h;
    a.y        = y;
    a.rstd     = rstd;
    a.scale    = scale;
    a.parts    = static_cast<float *>(workspace);
    a.rows     = rows;
    a.x_stride = x_stride;
    a.r_stride = residual_stride;
    a.h_stride = h_stride;
    a.hidden   = static_cast<int>(hidden);
    a.mode     = scale_mode;
    a.eps      = eps;
    a.w32      = weight_dtype == GG_DTYPE_FP32;
    a.e5m2     = out_dtype == GG_DTYPE_FP8_E5M2;
    if (rows == 0) { // no maximum: the scale alone
        return launch("rms_norm", quantize_kernel<BF16, 256>, 1, 256, static_cast<hipStream_t>(stream), a);
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool        wide = few(rows, hidden);
    if (dtype == GG_DTYPE_BF16)
        return wide ? run_norm<BF16, true>(a, st) : run_norm<BF16, false>(a, st);
    return wide ? run_norm<F16, true>(a, st) : run_norm<F16, false>(a, st);
}

size_t gg_rms_norm_backward_workspace(int64_t rows, int64_t hidden) {
    if (rows < 1 || hidden < 1 || hidden > 32768 || few(rows, hidden))
        return 0;
    return static_cast<size_t>(back_blocks(rows, hidden)) * static_cast<size_t>(hidden) * 4;
}

int gg_rms_norm_backward(int dtype, int weight_dtype, int64_t rows, int64_t hidden, const void *grad_y,
                         int64_t grad_y_stride, const void *h, int64_t h_stride, const void *weight, const float *rstd,
                         const void *grad_h, int64_t grad_h_stride, void *grad_x, void *grad_weight, void *workspace,
                         size_t workspace_bytes, void *stream) {
    g_error[0] = 0;
    if (const int st = check_norm(dtype, weight_dtype, rows, hidden))
        return st;
    if (weight == nullptr || grad_weight == nullptr || (rows > 0 && (grad_x == nullptr || rstd == nullptr)))
        return fail(GG_ERR_INVALID, "weight, rstd, grad_x and grad_weight must be device pointers");
    if (const int st = check_rows("grad_y", grad_y, grad_y_stride, rows))
        return st;
    if (const int st = check_rows("h", h, h_stride, rows))
        return st;
    if (grad_h != nullptr)
        if (const int st = check_rows("grad_h", grad_h, grad_h_stride, rows))
            return st;
    if (!aligned(weight, 16) || !aligned(grad_x, 16) || !aligned(grad_weight, 16))
        return fail(GG_ERR_UNSUPPORTED, "weight, grad_x and grad_weight must be 16-byte aligned");
    const size_t need = gg_rms_norm_backward_workspace(rows, hidden);
    if (workspace_bytes < need || (need > 0 && (workspace == nullptr || !aligned(workspace, 16))))
        return fail(GG_ERR_WORKSPACE, "workspace must be 16-byte aligned and of gg_rms_norm_backward_workspace(rows, hidden) bytes");
    BackArgs a{};
    a.g         = grad_y;
    a.h         = h;
    a.weight    = weight;
    a.gh        = grad_h;
    a.rstd      = rstd;
    a.gx        = grad_x;
    a.parts     = static_cast<float *>(workspace);
    a.rows      = rows;
    a.g_stride  = grad_y_stride;
    a.h_stride  = h_stride;
    a.gh_stride = grad_h_stride;
    a.hidden    = static_cast<int>(hidden);
    a.w32       = weight_dtype == GG_DTYPE_FP32;
    if (rows == 0) { // the sums of no rows
        return launch("rms_norm_backward", weight_sum_kernel<BF16>, (a.hidden + 31) / 32, 1024,
                      static_cast<hipStream_t>(stream), nullptr, 0, a.hidden, grad_weight, a.w32);
    }
    return dtype == GG_DTYPE_BF16 ? run_back<BF16>(a, grad_weight, static_cast<hipStream_t>(stream))
                                  : run_back<F16>(a, grad_weight, static_cast<hipStream_t>(stream));
}

} // extern "C"
