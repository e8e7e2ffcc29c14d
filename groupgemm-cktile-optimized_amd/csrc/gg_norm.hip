// RMS norm and layer norm with the residual's addition, 16-bit, fp8 or int8 output, and their gradients (gg_rms_norm,
// gg_layer_norm, .. in include/gg_moe_layer.h).
//
// Forward: h = round(x + r), rstd = (mean h^2 + eps)^-1/2, y = h rstd w; layer norm (CENTER) takes h less its mean, in
// the mean square too, and adds a bias. A row stays in the registers
// of the waves that work on it (the RMS norm's: one wave up to 1024 values, four up to 16384, of few rows up to 2048, else
// sixteen, with_shape; the layer norm's: with_center_forward, and center_shape for its gradients), so x and r are read once
// and h and y written once: bound by HBM. The tensor scale needs the largest |y|
// of all rows before the first value is rounded: a first pass writes h, rstd and one maximum per
// workgroup, a second reads h again and rounds.
//
// The norm is taken of the rounded h, the value that later layers and the backward pass read, so the
// passes agree whatever the scale.
//
// Measured: 32768 rows of 7168, bf16 with residual to fp8 with a tensor scale, 377 us: 245 for the first pass (x and r
// read, h written: 5.8 TB/s) and 133 for the second (h read, y written: 5.3); 5 rows to bf16 3.8, the latency of a launch,
// a row's loads and a barrier. Backward 16640 x 2880 with a gradient past the norm: 75 us, 5.1 TB/s (69 row by row, 6 for
// the weight's gradient). 8192 of 7168 with residual to int8 73 (5.6). Layer norm: 32768 rows of 4096 bf16 87.5 us (6.2 TB/s),
// 8192 of 7168 with residual to int8 75 (5.5), to fp8 with a scale a row 85 (4.8), for the tensor 62 + 36; 6 of 7168 4.7;
// backward 16640 x 2880 with a gradient past the norm 76 + 5 for the two sums (5.2 TB/s), 1024 x 8192 26.
#include "gg_row.h"

#include <algorithm>

namespace gg {
namespace layer {

thread_local char g_error[256] = "";

namespace {

constexpr int kMaxParts = GG_NORM_WORKSPACE / 4; // workgroups of a tensor scale's first pass

struct NormArgs {
    const void *x, *residual, *weight, *bias; // bias (layer norm only) may be null
    void       *h, *y;
    float      *mean, *rstd, *scale, *parts; // mean: layer norm only
    int64_t     rows, x_stride, r_stride, h_stride;
    int         hidden, mode, n_parts;
    float       eps;
    bool        w32, e5m2;
};

// The largest |y| of a workgroup's rows, for a tensor scale's second pass.
template <int WPR>
__device__ __forceinline__ void store_top(const NormArgs &a, unsigned top, unsigned (&block_top)[4], RowReduce<WPR> &m, int wave, int lane) {
    top                 = wave_max(top);
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

// One pass over the rows: the whole norm in 16 bits or fp8, in int8 with a scale for each row (instances of its own: the
// rounding's registers would cost the others a wave per SIMD), or the first pass of a tensor scale (no y; the workgroup's
// largest |y|).
enum Pass : int { kWhole = 0, kInt8 = 1, kFirst = 2 };
template <typename T, int WPR, int U, int PASS>
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
        if constexpr (PASS == kFirst) {
            top = max(top, row_top);
        } else {
            float s = 1.f;
            if (PASS == kInt8 || a.mode == GG_NORM_SCALE_ROW) {
                s = scale_of(row_max<WPR>(m, turn, row_top, wave, lane), PASS == kInt8 ? kTopI8 : a.e5m2 ? kTopE5M2 : kTopE4M3);
                if constexpr (PASS == kInt8)
                    s = uniform(s);
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
                    if constexpr (PASS == kInt8) {
                        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + row * a.hidden + i) = pack_i8(v[u], by);
                    } else if (a.mode == GG_NORM_PLAIN) {
                        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.y) + row * a.hidden + i) = pack8<T>(v[u]);
                    } else {
                        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + row * a.hidden + i) = pack_fp8(v[u], by, a.e5m2);
                    }
                }
            }
        }
    }
    if constexpr (PASS == kFirst)
        store_top<WPR>(a, top, block_top, m, wave, lane);
}

// ---- layer norm ----

// The two sums of a row over its waves, with one barrier.
template <int WPR> struct PairReduce {
    float sums[2][2][WPR];
};
template <int WPR>
__device__ __forceinline__ void row_sums(PairReduce<WPR> &m, int turn, float &p, float &q, int wave, int lane) {
    p = wave_sum(p);
    q = wave_sum(q);
    if constexpr (WPR > 1) {
        if (lane == 0) {
            m.sums[turn][0][wave] = p;
            m.sums[turn][1][wave] = q;
        }
        __syncthreads();
        p = q = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            p += m.sums[turn][0][i];
            q += m.sums[turn][1][i];
        }
    }
}

// Mean and sum of squares about it of a row, with one barrier. A wave finds the mean m_w of its own n_w values, the sum of
// their squares about that, and what rounding left of their sum, e = sum (x - m_w); the waves' are put together exactly,
// sum (x - m)^2 = sum (x - m_w)^2 + 2 (m_w - m) e + n_w (m_w - m)^2, each by a lane of every wave. So nothing cancels but
// what a second pass over the row would lose, too. The means are quotients, not products with rounded reciprocals: equal
// 16-bit values have exact sums, and a row of them has to have that value for its mean, as a unit of float32 off is
// eps^-1/2 times as much in y (mean_of).
template <int WPR> struct Moments {
    f32x4 of_wave[2][WPR]; // m_w n_w, m_w, squares, e
};
// sum / n by 1 / n, corrected once by the remainder, which a fused multiply-add gives exactly: a quotient that is a float32
// comes out as that (32768 rows of 4096 93.3 -> 94.0 us, with divisions 96.4). An infinite sum has no remainder and stays.
__device__ __forceinline__ float mean_of(float sum, float n, float inv) {
    const float q = sum * inv, c = fmaf(fmaf(-n, q, sum), inv, q);
    return c == c ? c : q;
}
template <int WPR, int U> struct RowMoments {
    float own, inv_own, n; // values of this wave, and of wave lane % WPR
    float all, inv_hidden;
    __device__ __forceinline__ RowMoments(int hidden, int wave, int lane) {
        // in each of the U rounds the waves take 512 values one after the other
        const auto count = [&](int w) {
            int c = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
                c += min(max(hidden - (u * WPR + w) * 512, 0), 512);
            return static_cast<float>(c);
        };
        own        = count(WPR == 1 ? 0 : wave);
        inv_own    = own > 0.f ? 1.f / own : 0.f;
        n          = count(lane & (WPR - 1));
        all        = static_cast<float>(hidden);
        inv_hidden = 1.f / all;
    }
    // v holds zeros past the row's end; mine: the lane's pieces of 8 that are not.
    __device__ __forceinline__ void operator()(Moments<WPR> &m, int turn, const float (&v)[U][8], const bool (&mine)[U], int wave,
                                               int lane, float &mean, float &square) const {
        float s[2] = {0.f, 0.f}, q[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s[j & 1] += v[u][j];
        const float sum = wave_sum(s[0] + s[1]), mw = mean_of(sum, own, inv_own);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (mine[u])
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = v[u][j] - mw;
                    q[j & 1] = fmaf(d, d, q[j & 1]);
                }
        const float sq = wave_sum(q[0] + q[1]);
        if constexpr (WPR == 1) {
            mean   = mw;
            square = sq;
        } else {
            if (lane == 0)
                m.of_wave[turn][wave] = f32x4{sum, mw, sq, fmaf(-own, mw, sum)};
            __syncthreads();
            const f32x4 w = m.of_wave[turn][lane & (WPR - 1)];
            mean          = mean_of(group_sum<WPR>(w[0]), all, inv_hidden);
            const float d = w[1] - mean;
            square        = group_sum<WPR>(n > 0.f ? fmaf(d, fmaf(n, d, 2.f * w[3]), w[2]) : 0.f);
        }
    }
};

// As norm_kernel. A workgroup takes one row after the other and, where a lane has at most four pieces of one, has the next
// one's values under way while it works on a row and keeps weight and bias (as many bytes as a row each, or in float32
// twice as many) in registers.
template <typename T, int WPR, int U, int PASS>
__global__ void __launch_bounds__(block_threads(WPR)) center_norm_kernel(const NormArgs a) {
    __shared__ Moments<WPR>  mom;
    __shared__ RowReduce<WPR> m;
    __shared__ unsigned       block_top[4];
    constexpr bool kHold = U <= 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t    = WPR == 1 ? lane : static_cast<int>(threadIdx.x); // thread of the row
    unsigned  top  = 0;
    int       turn = 0;
    bool      mine[U];
    u32x4     xw[U], rw[U];
    const RowMoments<WPR, U> moments(a.hidden, wave, lane);
    const int64_t step = static_cast<int64_t>(gridDim.x) * rows_per_block(WPR);
    int64_t       row  = static_cast<int64_t>(blockIdx.x) * rows_per_block(WPR) + (WPR == 1 ? wave : 0);
    const auto fetch = [&](int64_t r) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (mine[u]) {
                const int i = (u * 64 * WPR + t) * 8;
                xw[u]       = load_once(static_cast<const uint16_t *>(a.x) + r * a.x_stride + i);
                if (a.residual != nullptr)
                    rw[u] = load_once(static_cast<const uint16_t *>(a.residual) + r * a.r_stride + i);
            }
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
        mine[u] = (u * 64 * WPR + t) * 8 < a.hidden;
    if (kHold && row < a.rows)
        fetch(row);
    float w[kHold ? U : 1][8], b[kHold ? U : 1][8];
    if constexpr (kHold) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[u][j] = b[u][j] = 0.f;
            if (mine[u]) {
                load_w<T>(a.weight, a.w32, (u * 64 * WPR + t) * 8, w[u]);
                if (a.bias != nullptr)
                    load_w<T>(a.bias, a.w32, (u * 64 * WPR + t) * 8, b[u]);
            }
        }
    }
    // every wave of a block that shares a row makes the same trips, so the barriers match
    for (; row < a.rows; row += step, turn ^= 1) {
        float v[U][8];
        if constexpr (!kHold)
            fetch(row);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[u][j] = 0.f;
            if (mine[u]) {
                unpack8<T>(xw[u], v[u]);
                if (a.residual != nullptr) {
                    float r[8];
                    unpack8<T>(rw[u], r);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[u][j] += r[j];
                    const u32x4 hw = pack8<T>(v[u]);
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.h) + row * a.h_stride + (u * 64 * WPR + t) * 8) = hw;
                    unpack8<T>(hw, v[u]);
                }
            }
        }
        if (kHold && row + step < a.rows)
            fetch(row + step);
        float mean, square;
        moments(mom, turn, v, mine, wave, lane, mean, square);
        const float rstd = 1.f / sqrtf(square * moments.inv_hidden + a.eps);
        if (t == 0) {
            if (a.mean != nullptr)
                a.mean[row] = mean;
            if (a.rstd != nullptr)
                a.rstd[row] = rstd;
        }
        unsigned row_top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (mine[u]) {
                if constexpr (!kHold) {
                    load_w<T>(a.weight, a.w32, (u * 64 * WPR + t) * 8, w[0]);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        b[0][j] = 0.f;
                    if (a.bias != nullptr)
                        load_w<T>(a.bias, a.w32, (u * 64 * WPR + t) * 8, b[0]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[u][j] = fmaf((v[u][j] - mean) * rstd, w[kHold ? u : 0][j], b[kHold ? u : 0][j]);
                    if (PASS != kWhole || a.mode == GG_NORM_SCALE_ROW)
                        row_top = max(row_top, __float_as_uint(fabsf(v[u][j])));
                }
            }
        if constexpr (PASS == kFirst) {
            top = max(top, row_top);
        } else {
            float s = 1.f;
            if (PASS == kInt8 || a.mode == GG_NORM_SCALE_ROW) {
                s = uniform(scale_of(row_max<WPR>(m, turn, row_top, wave, lane), PASS == kInt8 ? kTopI8 : a.e5m2 ? kTopE5M2 : kTopE4M3));
                if (t == 0)
                    a.scale[row] = s;
            } else if (a.mode == GG_NORM_SCALE_GIVEN) {
                s = a.scale[0];
            }
            const Divisor by(s);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (mine[u]) {
                    const int64_t at = row * a.hidden + (u * 64 * WPR + t) * 8;
                    if constexpr (PASS == kInt8)
                        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + at) = pack_i8(v[u], by);
                    else if (a.mode == GG_NORM_PLAIN)
                        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.y) + at) = pack8<T>(v[u]);
                    else
                        *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + at) = pack_fp8(v[u], by, a.e5m2);
                }
        }
    }
    if constexpr (PASS == kFirst)
        store_top<WPR>(a, top, block_top, m, wave, lane);
}

// The tensor scale's second pass: the largest of the first pass's maxima, then y from h and rstd.
template <typename T, bool CENTER, int THREADS> __global__ void __launch_bounds__(THREADS) quantize_kernel(const NormArgs a) {
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
    const float   s = scale_of(top, a.e5m2 ? kTopE5M2 : kTopE4M3);
    const Divisor by(s);
    if (blockIdx.x == 0 && threadIdx.x == 0)
        a.scale[0] = s;
    // from the last row backwards: the rows written last are still in the Infinity Cache
    for (int64_t row = a.rows - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
        const float rstd = a.rstd[row], mean = CENTER ? a.mean[row] : 0.f;
        for (int i = threadIdx.x * 8; i < a.hidden; i += THREADS * 8) {
            float v[8], w[8];
            unpack8<T>(load_once(static_cast<const uint16_t *>(a.h) + row * a.h_stride + i), v);
            load_w<T>(a.weight, a.w32, i, w);
            if constexpr (CENTER) {
                float b[8] = {};
                if (a.bias != nullptr)
                    load_w<T>(a.bias, a.w32, i, b);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = fmaf((v[j] - mean) * rstd, w[j], b[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = v[j] * rstd * w[j];
            }
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

// grad_weight, and grad_bias where parts hold `width` = 2 * hidden columns: the sum of the partial sums of each column, in
// a fixed order; 32 columns by 128 slices of the parts a workgroup.
template <typename T>
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float *parts, int n_parts, int width, int hidden, void *grad_weight,
                                                          void *grad_bias, bool w32) {
    __shared__ f32x4 sums[128][8];
    const int c4 = threadIdx.x & 7, slice = threadIdx.x >> 3, col = blockIdx.x * 32 + c4 * 4; // hidden % 8 == 0
    f32x4     s{0.f, 0.f, 0.f, 0.f};
    if (col < width)
#pragma unroll 8
        for (int p = slice; p < n_parts; p += 128)
            s += *reinterpret_cast<const f32x4 *>(parts + static_cast<int64_t>(p) * width + col);
    sums[slice][c4] = s;
    __syncthreads();
#pragma unroll
    for (int half = 64; half > 0; half >>= 1) {
        if (slice < half)
            sums[slice][c4] = s += sums[slice + half][c4];
        __syncthreads();
    }
    if (slice == 0 && col < width) {
        void     *out = col < hidden ? grad_weight : grad_bias;
        const int at  = col < hidden ? col : col - hidden;
        if (w32)
            *reinterpret_cast<f32x4 *>(static_cast<float *>(out) + at) = s;
        else
            *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + at) = u32x2{T::word(s[0], s[1]), T::word(s[2], s[3])};
    }
}

// ---- layer norm's gradients ----

struct CenterArgs {
    BackArgs     b; // parts: [workgroups][2][hidden], grad_weight's and grad_bias's
    const float *mean;
};

// With d = h - mean: grad_x = grad_h + rstd (w g - mean(w g) - d rstd^2 mean(w g d)), row by row; the partial sums of
// g d rstd and of g stay in registers over the rows of a workgroup, which has R at a time, and are written once. Two sums a
// column are twice the registers of the RMS norm's one, so rows past 8192 values take eight waves, and with more than four pieces a lane (past
// 16384) load the inputs again, from the caches, instead of keeping them.
template <typename T, int WPR, int U, bool SUMS, int R>
__global__ void __launch_bounds__(64 * WPR * R) center_back_kernel(const CenterArgs c) {
    __shared__ PairReduce<WPR> m[R];
    const BackArgs &a    = c.b;
    constexpr bool  kKeep = U <= 4;
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % WPR, own = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
    const int t    = static_cast<int>(threadIdx.x) % (64 * WPR);
    float     dw[U][8], db[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            dw[u][j] = db[u][j] = 0.f;
    int           turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * R;
    // every wave of the workgroup makes the same trips, so the barriers match; past the last row they have no values
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * R; first < a.rows; first += step, turn ^= 1) {
        const int64_t   row  = R == 1 ? first : std::min(first + own, a.rows - 1);
        const int       here = R == 1 || first + own < a.rows ? a.hidden : 0;
        const uint16_t *gp = static_cast<const uint16_t *>(a.g) + row * a.g_stride;
        const uint16_t *hp = static_cast<const uint16_t *>(a.h) + row * a.h_stride;
        const uint16_t *rp = a.gh == nullptr ? nullptr : static_cast<const uint16_t *>(a.gh) + row * a.gh_stride;
        u32x4       gw[U], hw[U], rw[U];
        float       sum = 0.f, dot = 0.f;
        const float rstd = a.rstd[row], mean = c.mean[row];
        if constexpr (kKeep) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = (u * 64 * WPR + t) * 8;
                if (i < here) {
                    gw[u] = load_once(gp + i);
                    hw[u] = load_once(hp + i);
                    if (rp != nullptr)
                        rw[u] = load_once(rp + i);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < here) {
                float g[8], h[8], w[8];
                unpack8<T>(kKeep ? gw[u] : *reinterpret_cast<const u32x4 *>(gp + i), g);
                unpack8<T>(kKeep ? hw[u] : *reinterpret_cast<const u32x4 *>(hp + i), h);
                load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = h[j] - mean, wg = g[j] * w[j];
                    sum += wg;
                    dot = fmaf(wg, d, dot);
                    if constexpr (SUMS) {
                        dw[u][j] = fmaf(g[j] * d, rstd, dw[u][j]);
                        db[u][j] += g[j];
                    }
                }
            }
        }
        row_sums<WPR>(m[own], turn, sum, dot, wave, lane);
        // vmcnt 0: the row's loads are back. Said once here, or the compiler, which sees lanes past the row's end that wait for
        // none, has each of the next row's loads wait for the one before it (4096 x 14336 105 instead of 101 us).
        __builtin_amdgcn_s_waitcnt(0x0f70);
        const float n  = static_cast<float>(a.hidden);
        const float c1 = sum / n, c2 = rstd * (rstd * (dot / n)); // of w g and of d in grad_x / rstd (rstd^2 alone may be past float32)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < here) {
                float g[8], h[8], w[8], r[8];
                unpack8<T>(kKeep ? gw[u] : load_once(gp + i), g);
                unpack8<T>(kKeep ? hw[u] : load_once(hp + i), h);
                load_w<T>(a.weight, a.w32, i, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) // h - mean first: c2 h - c2 mean would cancel where the mean is large
                    g[j] = fmaf(-c2, h[j] - mean, fmaf(g[j], w[j], -c1));
                if (rp != nullptr) {
                    unpack8<T>(kKeep ? rw[u] : load_once(rp + i), r);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        g[j] = fmaf(rstd, g[j], r[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        g[j] *= rstd;
                }
                *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.gx) + row * a.hidden + i) = pack8<T>(g);
            }
        }
    }
    if constexpr (!SUMS)
        return;
    // the sums of a workgroup's R rows are added up first, in their order
    if constexpr (R > 1) {
        __shared__ f32x4 mine[R - 1][U][4][64 * WPR];
        if (own > 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    mine[own - 1][u][q][t]     = f32x4{dw[u][4 * q], dw[u][4 * q + 1], dw[u][4 * q + 2], dw[u][4 * q + 3]};
                    mine[own - 1][u][2 + q][t] = f32x4{db[u][4 * q], db[u][4 * q + 1], db[u][4 * q + 2], db[u][4 * q + 3]};
                }
        __syncthreads();
        if (own > 0)
            return;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int o = 0; o < R - 1; ++o)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dw[u][4 * q + j] += mine[o][u][q][t][j];
                        db[u][4 * q + j] += mine[o][u][2 + q][t][j];
                    }
    }
    float *part = a.parts + static_cast<int64_t>(blockIdx.x) * 2 * a.hidden;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * 64 * WPR + t) * 8;
        if (i < a.hidden) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                *reinterpret_cast<f32x4 *>(part + i + 4 * q) = f32x4{dw[u][4 * q], dw[u][4 * q + 1], dw[u][4 * q + 2], dw[u][4 * q + 3]};
                *reinterpret_cast<f32x4 *>(part + a.hidden + i + 4 * q) =
                    f32x4{db[u][4 * q], db[u][4 * q + 1], db[u][4 * q + 2], db[u][4 * q + 3]};
            }
        }
    }
}

// grad_weight and grad_bias from g and h themselves: 64 columns (a line of 128 bytes a row) by 128 slices of the rows a workgroup.
template <typename T> __global__ void __launch_bounds__(1024) center_strip_kernel(const CenterArgs c, void *grad_weight, void *grad_bias) {
    __shared__ f32x4 sums[4][128][8];
    const BackArgs &a = c.b;
    const int c8 = threadIdx.x & 7, slice = threadIdx.x >> 3, col = blockIdx.x * 64 + c8 * 8; // hidden % 8 == 0
    f32x4     s[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
        s[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (col < a.hidden) {
        const uint16_t *g = static_cast<const uint16_t *>(a.g) + col, *h = static_cast<const uint16_t *>(a.h) + col;
#pragma unroll 4
        for (int64_t row = slice; row < a.rows; row += 128) {
            float gv[8], hv[8];
            unpack8<T>(*reinterpret_cast<const u32x4 *>(g + row * a.g_stride), gv);
            unpack8<T>(*reinterpret_cast<const u32x4 *>(h + row * a.h_stride), hv);
            const float rstd = a.rstd[row], mean = c.mean[row];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[j / 4][j % 4] = fmaf(gv[j] * (hv[j] - mean), rstd, s[j / 4][j % 4]);
                s[2 + j / 4][j % 4] += gv[j];
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        sums[q][slice][c8] = s[q];
    __syncthreads();
#pragma unroll
    for (int half = 64; half > 0; half >>= 1) {
        if (slice < half)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                sums[q][slice][c8] = s[q] += sums[q][slice + half][c8];
        __syncthreads();
    }
    if (slice == 0 && col < a.hidden) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            void *out = o == 0 ? grad_weight : grad_bias;
            if (a.w32) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    reinterpret_cast<f32x4 *>(static_cast<float *>(out) + col)[q] = s[2 * o + q];
            } else {
                const f32x4 l = s[2 * o], r = s[2 * o + 1];
                const float v[8] = {l[0], l[1], l[2], l[3], r[0], r[1], r[2], r[3]};
                *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(out) + col) = pack8<T>(v);
            }
        }
    }
}

constexpr int64_t kMaxBlocks = int64_t(1) << 20;

// The layer norm's shapes: eight waves for a row of 6145 to 8192 values and sixteen for up to 16384, which keep weight and
// bias in registers and have a next row's values under way, where four would have to choose; eight from 2049 on in few
// rows. us at four, eight and sixteen waves: 8192 rows of 7168 to int8 81.6, 71.9, 90.7, to bf16 82.3, 74.6, 79.3; 4096 of
// 5120 31.3, 33.3, 33.2; at four and sixteen: 8000 of 12288 97.6, 74.5; at eight and sixteen, with residual to int8, 64 of
// 7168 5.0, 5.8, 512 9.2, 11.6; at four and eight 64 of 4096 4.3, 4.0, 256 4.8, 4.6, 600 7.1, 8.4.
template <typename F> int with_center_forward(int64_t rows, int64_t hidden, F f) {
    using std::integral_constant;
    const int wpr = hidden <= 1024                                      ? 1
                    : hidden <= 2048 || (hidden <= 6144 && rows > 256) ? 4
                    : hidden <= 8192 || hidden > 16384                  ? 8
                                                                        : 16;
    const int u   = static_cast<int>((hidden + 512 * wpr - 1) / (512 * wpr));
#define GG_SHAPE(W, N)                                                                                                 \
    if (wpr == W && u <= N)                                                                                            \
        return f(integral_constant<int, W>{}, integral_constant<int, N>{});
    GG_SHAPE(1, 1) GG_SHAPE(1, 2) GG_SHAPE(4, 1) GG_SHAPE(4, 2) GG_SHAPE(4, 3) GG_SHAPE(8, 1) GG_SHAPE(8, 2) GG_SHAPE(16, 2)
#undef GG_SHAPE
    return f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
}
// The shape of either norm's forward pass.
template <bool CENTER, bool WIDE, typename F> int with_norm_shape(int64_t rows, int64_t hidden, F f) {
    if constexpr (CENTER)
        return with_center_forward(rows, hidden, f);
    else
        return with_shape<WIDE>(hidden, f);
}

// The kernel of either norm for one pass.
template <typename T, bool CENTER, int WPR, int U, int PASS> constexpr auto norm_pass() {
    if constexpr (CENTER)
        return center_norm_kernel<T, WPR, U, PASS>;
    else
        return norm_kernel<T, WPR, U, PASS>;
}

template <typename T, bool CENTER, bool WIDE> int run_norm(const NormArgs &a, bool i8, hipStream_t s) {
    constexpr const char *kWhat = CENTER ? "layer_norm" : "rms_norm";
    const int64_t blocks = row_blocks(a.rows, a.hidden);
    if (a.mode != GG_NORM_SCALE_TENSOR)
        return with_norm_shape<CENTER, WIDE>(a.rows, a.hidden, [&](auto wpr, auto u) {
            const auto kernel = i8 ? norm_pass<T, CENTER, wpr.value, u.value, kInt8>() : norm_pass<T, CENTER, wpr.value, u.value, kWhole>();
            // the layer norm's workgroups go from row to row: as many as fit at once
            const int64_t grid = !CENTER || blocks <= 256 ? blocks : std::min<int64_t>(blocks, resident_blocks(kernel, block_threads(wpr.value)));
            return launch(kWhat, kernel, std::min(grid, kMaxBlocks), block_threads(wpr.value), s, a);
        });
    // The first pass: as many workgroups as fit at once, each with its share of the rows (32768 rows of 7168: 1792
    // workgroups fit, 377 us for both passes; 1536 377, 1280 389, 1024 421, 2048, 1.1 rounds of them, 453).
    NormArgs b = a;
    if (b.residual == nullptr) { // h is x
        b.h        = const_cast<void *>(b.x);
        b.h_stride = b.x_stride;
    }
    const int st = with_norm_shape<CENTER, WIDE>(a.rows, a.hidden, [&](auto wpr, auto u) {
        constexpr auto kernel = norm_pass<T, CENTER, wpr.value, u.value, kFirst>();
        // (asked for each call, as devices differ; few workgroups fit in any case)
        b.n_parts = static_cast<int>(blocks <= 256 ? blocks : std::min<int64_t>(blocks, std::min(resident_blocks(kernel, block_threads(wpr.value)), kMaxParts)));
        return launch(kWhat, kernel, b.n_parts, block_threads(wpr.value), s, b);
    });
    constexpr int kThreads = WIDE ? 1024 : 256;
    return st ? st : launch(kWhat, quantize_kernel<T, CENTER, kThreads>, std::min<int64_t>(b.rows, 8192), kThreads, s, b);
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
                            static_cast<int>(back_blocks(a.rows, a.hidden)), a.hidden, a.hidden, grad_weight, nullptr, a.w32);
}

// Layer norm's backward pass: waves of a row, pieces of a lane and rows of a workgroup (see center_back_kernel). Rows that
// share a workgroup share its partial sums, but wait for each other at the barriers. us at one, two and three rows:
// 1000 x 2880 17.6, 14.8, 14.5; 1500 x 4096 24.8, 22.9, 20.3; 16640 x 2048 61.3, 63.6, 56.6; of 6144 163, 170, 160; but 8192 x
// 4096 61.8, 59.3, 60.9; 16640 x 2880 82.1, 81.4, 87.2; at one and two (three are short of registers) 2500 x 7168 48.8, 43.9,
// 8192 x 7168 104, 110. So two rows past 2048 with two pieces, with four two up to 4096 and then one.
struct CenterShape {
    int waves, pieces, rows;
};
CenterShape center_shape(int64_t rows, int64_t hidden) {
    const int wpr = hidden <= 1024 ? 1 : hidden <= 8192 ? 4 : 8, u = static_cast<int>((hidden + 512 * wpr - 1) / (512 * wpr));
    return {wpr, wpr == 8 ? (u <= 3 ? 3 : u == 4 ? 4 : 8) : u,
            wpr == 1 ? 4 : wpr == 8 ? 1 : u == 2 ? (rows <= 2048 ? 3 : 2) : u == 4 ? (rows <= 4096 ? 2 : 1) : 3};
}
template <typename F> int with_center_shape(int64_t rows, int64_t hidden, F f) {
    using std::integral_constant;
    const CenterShape c = center_shape(rows, hidden);
#define GG_SHAPE(W, N, R)                                                                                              \
    if (c.waves == W && c.pieces == N && c.rows == R)                                                                  \
        return f(integral_constant<int, W>{}, integral_constant<int, N>{}, integral_constant<int, R>{});
    GG_SHAPE(1, 1, 4) GG_SHAPE(1, 2, 4) GG_SHAPE(4, 1, 3) GG_SHAPE(4, 2, 2) GG_SHAPE(4, 2, 3) GG_SHAPE(4, 3, 3) GG_SHAPE(4, 4, 1)
    GG_SHAPE(4, 4, 2) GG_SHAPE(8, 3, 1) GG_SHAPE(8, 4, 1)
#undef GG_SHAPE
    return f(integral_constant<int, 8>{}, integral_constant<int, 8>{}, integral_constant<int, 1>{});
}
// Its workgroups: at most those that 256 CUs hold at once by the instances' registers (a test holds the numbers to the
// compiler's report). Of up to eight turns each has as many as the others (3200 x 6144 46.1 -> 44.0; of many, what the
// last turn leaves idle is less than what fewer workgroups lose, 16640 x 2880 81.4, 83.5), and past 256 two turns at least,
// which halves the partial sums (1500 x 1536 13.0 -> 11.5). (The next row's values under way while a row is worked on cost registers, and so workgroups:
// 16640 x 2880 102 us instead of 79; forcing five waves a SIMD where the registers give four spilled: 90.)
int64_t center_blocks(int64_t rows, int64_t hidden) {
    const CenterShape c     = center_shape(rows, hidden);
    const int64_t     fit   = c.waves == 8 ? 256 : c.waves == 1 ? (c.pieces == 1 ? 1280 : 768) : c.rows == 1 ? 768 : c.pieces == 1 || (c.pieces == 2 && c.rows == 2) ? 512 : 256;
    const int64_t     b     = (rows + c.rows - 1) / c.rows;
    const int64_t     turns = std::max<int64_t>((b + fit - 1) / fit, b <= 256 ? 1 : 2);
    return turns > 8 ? fit : (b + turns - 1) / turns;
}

template <typename T> int run_center_back(const CenterArgs &a, void *grad_weight, void *grad_bias, hipStream_t s) {
    const int64_t rows = a.b.rows, hidden = a.b.hidden;
    if (few(rows, hidden)) { // (the sums first: grad_x may take the place of an input)
        const int st = launch("layer_norm_backward", center_strip_kernel<T>, (hidden + 63) / 64, 1024, s, a, grad_weight, grad_bias);
        return st ? st : with_shape<true>(hidden, [&](auto wpr, auto u) {
            constexpr int r = rows_per_block(wpr.value);
            return launch("layer_norm_backward", center_back_kernel<T, wpr.value, u.value, false, r>, row_blocks(rows, hidden),
                          64 * wpr.value * r, s, a);
        });
    }
    const int blocks = static_cast<int>(center_blocks(rows, hidden));
    const int st     = with_center_shape(rows, hidden, [&](auto wpr, auto u, auto r) {
        return launch("layer_norm_backward", center_back_kernel<T, wpr.value, u.value, true, r.value>, blocks, 64 * wpr.value * r.value, s, a);
    });
    return st ? st : launch("layer_norm_backward", weight_sum_kernel<T>, (2 * hidden + 31) / 32, 1024, s, a.b.parts, blocks,
                            2 * a.b.hidden, a.b.hidden, grad_weight, grad_bias, a.b.w32);
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
} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

const char *gg_layer_last_error(void) { return g_error; }

// Both norms' forward pass (center: layer norm).
static int norm_forward(bool center, int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden,
                        float eps, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                        const void *weight, const void *bias, void *h, int64_t h_stride, void *y, float *mean, float *rstd,
                        float *scale, void *workspace, void *stream) {
    g_error[0] = 0;
    if (const int st = check_norm(dtype, weight_dtype, rows, hidden))
        return st;
    if (scale_mode < GG_NORM_PLAIN || scale_mode > GG_NORM_SCALE_GIVEN)
        return fail(GG_ERR_INVALID, "scale_mode must be a gg_norm_scale");
    if (scale_mode == GG_NORM_PLAIN ? out_dtype != dtype
                                    : !is8(out_dtype) && !(out_dtype == GG_DTYPE_INT8 && scale_mode == GG_NORM_SCALE_ROW))
        return fail(GG_ERR_INVALID, "out_dtype must be dtype, an fp8 type with a scale, or int8 with a scale for each row");
    if (scale_mode != GG_NORM_PLAIN && scale == nullptr && (rows > 0 || scale_mode != GG_NORM_SCALE_ROW)) // (a row scale of no rows)
        return fail(GG_ERR_INVALID, "scale is null");
    if (rows == 0 && scale_mode != GG_NORM_SCALE_TENSOR)
        return GG_OK;
    if (weight == nullptr || (rows > 0 && y == nullptr))
        return fail(GG_ERR_INVALID, "weight and y must be device pointers");
    if (scale_mode == GG_NORM_SCALE_TENSOR && (workspace == nullptr || (rows > 0 && (rstd == nullptr || (center && mean == nullptr)))))
        return fail(GG_ERR_INVALID, center ? "a tensor scale needs workspace, mean and rstd" : "a tensor scale needs workspace and rstd");
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
    if (!aligned(weight, 16) || !aligned(bias, 16) || !aligned(y, scale_mode == GG_NORM_PLAIN ? 16 : 8) || !aligned(workspace, 4))
        return fail(GG_ERR_UNSUPPORTED, "weight%s and y must be 16-byte aligned (8-bit y: 8)", center ? ", bias" : "");
    NormArgs a{};
    a.x        = x;
    a.residual = residual;
    a.weight   = weight;
    a.bias     = bias;
    a.h        = h;
    a.y        = y;
    a.mean     = mean;
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
    const bool        i8 = out_dtype == GG_DTYPE_INT8;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (rows == 0) // no maximum: the scale alone
        return launch(center ? "layer_norm" : "rms_norm", quantize_kernel<BF16, false, 256>, 1, 256, st, a);
    const bool wide = few(rows, hidden);
    const auto run  = [&](auto type, auto centered) {
        using T = decltype(type);
        return wide ? run_norm<T, centered.value, true>(a, i8, st) : run_norm<T, centered.value, false>(a, i8, st);
    };
    if (dtype == GG_DTYPE_BF16)
        return center ? run(BF16{}, std::true_type{}) : run(BF16{}, std::false_type{});
    return center ? run(F16{}, std::true_type{}) : run(F16{}, std::false_type{});
}

int gg_rms_norm(int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden, float eps,
                const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                void *h, int64_t h_stride, void *y, float *rstd, float *scale, void *workspace, void *stream) {
    return norm_forward(false, dtype, weight_dtype, out_dtype, scale_mode, rows, hidden, eps, x, x_stride, residual,
                        residual_stride, weight, nullptr, h, h_stride, y, nullptr, rstd, scale, workspace, stream);
}

int gg_layer_norm(int dtype, int weight_dtype, int out_dtype, int scale_mode, int64_t rows, int64_t hidden, float eps,
                  const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight,
                  const void *bias, void *h, int64_t h_stride, void *y, float *mean, float *rstd, float *scale,
                  void *workspace, void *stream) {
    return norm_forward(true, dtype, weight_dtype, out_dtype, scale_mode, rows, hidden, eps, x, x_stride, residual,
                        residual_stride, weight, bias, h, h_stride, y, mean, rstd, scale, workspace, stream);
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
                      static_cast<hipStream_t>(stream), nullptr, 0, a.hidden, a.hidden, grad_weight, nullptr, a.w32);
    }
    return dtype == GG_DTYPE_BF16 ? run_back<BF16>(a, grad_weight, static_cast<hipStream_t>(stream))
                                  : run_back<F16>(a, grad_weight, static_cast<hipStream_t>(stream));
}

size_t gg_layer_norm_backward_workspace(int64_t rows, int64_t hidden) {
    if (rows < 1 || hidden < 1 || hidden > 32768 || few(rows, hidden))
        return 0;
    return static_cast<size_t>(center_blocks(rows, hidden)) * static_cast<size_t>(hidden) * 8;
}

int gg_layer_norm_backward(int dtype, int weight_dtype, int64_t rows, int64_t hidden, const void *grad_y,
                           int64_t grad_y_stride, const void *h, int64_t h_stride, const void *weight, const float *mean,
                           const float *rstd, const void *grad_h, int64_t grad_h_stride, void *grad_x, void *grad_weight,
                           void *grad_bias, void *workspace, size_t workspace_bytes, void *stream) {
    g_error[0] = 0;
    if (const int st = check_norm(dtype, weight_dtype, rows, hidden))
        return st;
    if (weight == nullptr || grad_weight == nullptr || grad_bias == nullptr ||
        (rows > 0 && (grad_x == nullptr || mean == nullptr || rstd == nullptr)))
        return fail(GG_ERR_INVALID, "weight, mean, rstd, grad_x, grad_weight and grad_bias must be device pointers");
    if (const int st = check_rows("grad_y", grad_y, grad_y_stride, rows))
        return st;
    if (const int st = check_rows("h", h, h_stride, rows))
        return st;
    if (grad_h != nullptr)
        if (const int st = check_rows("grad_h", grad_h, grad_h_stride, rows))
            return st;
    if (!aligned(weight, 16) || !aligned(grad_x, 16) || !aligned(grad_weight, 16) || !aligned(grad_bias, 16))
        return fail(GG_ERR_UNSUPPORTED, "weight, grad_x, grad_weight and grad_bias must be 16-byte aligned");
    const size_t need = gg_layer_norm_backward_workspace(rows, hidden);
    if (workspace_bytes < need || (need > 0 && (workspace == nullptr || !aligned(workspace, 16))))
        return fail(GG_ERR_WORKSPACE, "workspace must be 16-byte aligned and of gg_layer_norm_backward_workspace(rows, hidden) bytes");
    CenterArgs a{};
    a.b.g         = grad_y;
    a.b.h         = h;
    a.b.weight    = weight;
    a.b.gh        = grad_h;
    a.b.rstd      = rstd;
    a.b.gx        = grad_x;
    a.b.parts     = static_cast<float *>(workspace);
    a.b.rows      = rows;
    a.b.g_stride  = grad_y_stride;
    a.b.h_stride  = h_stride;
    a.b.gh_stride = grad_h_stride;
    a.b.hidden    = static_cast<int>(hidden);
    a.b.w32       = weight_dtype == GG_DTYPE_FP32;
    a.mean        = mean;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (rows == 0) // the sums of no rows
        return launch("layer_norm_backward", weight_sum_kernel<BF16>, (2 * a.b.hidden + 31) / 32, 1024, st, nullptr, 0,
                      2 * a.b.hidden, a.b.hidden, grad_weight, grad_bias, a.b.w32);
    return dtype == GG_DTYPE_BF16 ? run_center_back<BF16>(a, grad_weight, grad_bias, st)
                                  : run_center_back<F16>(a, grad_weight, grad_bias, st);
}

} // extern "C"
