// The gated activation between an expert's two products and its gradient, and the rounding of rows to int8
// (gg_silu_product, gg_silu_product_backward, gg_quantize_rows in include/gg_moe_layer.h).
//
// y = gate s(gate) up with s(v) = 1 / (1 + exp(-v)); a row holds its gates, then its ups. With p = s(gate):
// grad_gate = g up p (1 + gate (1 - p)), grad_up = g gate p. Everything in float32 from the 16-bit inputs, rounded once.
// A sigmoid below 2^-126, that of gates below -87.3, may come out as 0: then y and the gradients lose less than that part of
// gate up, of g up (1 - gate) and of g gate.
// Bound by HBM: every value is read once and written once. 16-bit outputs need nothing of the rest of their row, so the
// pieces of 8 values are dealt to the lanes one after the other. An int8 row's scale needs its largest |y| before the
// first value is rounded: the row's values stay in registers, as in the norms.
//
// Measured (us): 32768 rows of 2048 bf16 60 (6.7 TB/s), to int8 57 (5.9), backward 97 (6.9); 16640 of 2880 fp16 to int8 40.6
// (5.9); 33 of 2048 to int8 3.3, a launch and a row's latency. Rounding alone, 4160 of 2048: 8.
#include <algorithm>

#include "gg_row.h"

namespace gg {
namespace layer {
namespace {

struct ActArgs {
    const void *x, *grad; // gates and ups (or the rows to round), the gradient of y
    void       *y;        // y, or the gradient of x
    float      *scale;
    int64_t     rows, stride, grad_stride;
    int         inner; // values of a row of y
};

// By the reciprocal instruction, which is off by a unit in the last place, as the exponential's is (a division rounded as
// IEEE asks takes ten instructions, and the int8 rows' kernel is held up by what it computes as much as by what it reads).
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// y of the eight values from element i of a row on.
template <typename T, bool GATED> __device__ __forceinline__ void load_y(const ActArgs &a, const uint16_t *x, int i, float (&v)[8]) {
    unpack8<T>(load_once(x + i), v);
    if constexpr (GATED) {
        float u[8];
        unpack8<T>(load_once(x + a.inner + i), u);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = v[j] * sigmoid(v[j]) * u[j];
    }
}

// int8 rows.
template <typename T, bool GATED, int WPR, int U>
__global__ void __launch_bounds__(block_threads(WPR)) round_rows_kernel(const ActArgs a) {
    __shared__ RowReduce<WPR> m;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t    = WPR == 1 ? lane : static_cast<int>(threadIdx.x); // thread of the row
    int       turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * rows_per_block(WPR);
    // every wave of a block that shares a row makes the same trips, so the barriers match
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_block(WPR) + (WPR == 1 ? wave : 0); row < a.rows;
         row += step, turn ^= 1) {
        const uint16_t *x   = static_cast<const uint16_t *>(a.x) + row * a.stride;
        float           v[U][8];
        unsigned        top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.inner) {
                load_y<T, GATED>(a, x, i, v[u]);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    top = max(top, __float_as_uint(fabsf(v[u][j])));
            }
        }
        const float s = uniform(scale_of(row_max<WPR>(m, turn, top, wave, lane), kTopI8));
        if (t == 0)
            a.scale[row] = s;
        const Divisor by(s);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * 64 * WPR + t) * 8;
            if (i < a.inner)
                *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.y) + row * a.inner + i) = pack_i8(v[u], by);
        }
    }
}

// 16-bit outputs: y of a piece of 8 values, or (BACK) the gradients of its gates and ups.
template <typename T, bool BACK> __global__ void __launch_bounds__(256) silu_kernel(const ActArgs a) {
    const int64_t pieces = a.inner / 8, all = a.rows * pieces;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; p < all; p += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t   row = p / pieces;
        const int       i   = static_cast<int>(p - row * pieces) * 8;
        const uint16_t *x   = static_cast<const uint16_t *>(a.x) + row * a.stride;
        float           v[8];
        if constexpr (!BACK) {
            load_y<T, true>(a, x, i, v);
            *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.y) + row * a.inner + i) = pack8<T>(v);
        } else {
            float u[8], g[8], d[8];
            unpack8<T>(load_once(x + i), v);
            unpack8<T>(load_once(x + a.inner + i), u);
            unpack8<T>(load_once(static_cast<const uint16_t *>(a.grad) + row * a.grad_stride + i), g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // (grad_y last: its product with a large gate or up may be past float32; half of the slope, which is up to
                // 1.1, and twice the result: up times it may be, too)
                const float s = sigmoid(v[j]);
                d[j]          = (0.5f * s) * (1.f + v[j] * (1.f - s)) * u[j] * g[j] * 2.f;
                g[j]          = v[j] * s * g[j];
            }
            uint16_t *o = static_cast<uint16_t *>(a.y) + row * 2 * a.inner + i;
            *reinterpret_cast<u32x4 *>(o)           = pack8<T>(d);
            *reinterpret_cast<u32x4 *>(o + a.inner) = pack8<T>(g);
        }
    }
}

constexpr int64_t kMaxBlocks = int64_t(1) << 20;

// f(waves of a row, pieces of a lane). Of many rows, one wave takes a row of up to 2048 values, whose four pieces it has
// under way together and which needs no barrier: at four waves the kernel waited (us, four waves and one: 32768 rows of
// 2048 69.4, 56.8, rounding alone 50.6, 35.7; 3000 9.9, 8.3; but 1000 5.1, 5.6, 400 3.7, 5.5). Up to 8192 values four waves
// take one, past it sixteen where there are few (512 of 12288 11.9, 8.3; 1400 18.7, 18.0; 3000 36, 33; rounding alone 23, 24).
template <typename F> int with_round_shape(int64_t rows, int64_t n, F f) {
    using std::integral_constant;
    if (n > 8192 && rows <= 1024)
        return with_shape<true>(n, f);
    if (n > 2048 || (n > 1024 && rows <= 1280))
        return with_shape<false>(n, f);
    return n <= 512    ? f(integral_constant<int, 1>{}, integral_constant<int, 1>{})
           : n <= 1024 ? f(integral_constant<int, 1>{}, integral_constant<int, 2>{})
           : n <= 1536 ? f(integral_constant<int, 1>{}, integral_constant<int, 3>{})
                       : f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
}
template <typename T, bool GATED> int run_round(const char *what, const ActArgs &a, hipStream_t s) {
    return with_round_shape(a.rows, a.inner, [&](auto wpr, auto u) {
        const int64_t blocks = wpr.value == 1 ? (a.rows + 3) / 4 : a.rows;
        return launch(what, round_rows_kernel<T, GATED, wpr.value, u.value>, std::min(blocks, kMaxBlocks), block_threads(wpr.value), s, a);
    });
}
template <bool GATED> int run_round(const char *what, int dtype, const ActArgs &a, hipStream_t s) {
    return dtype == GG_DTYPE_BF16 ? run_round<BF16, GATED>(what, a, s) : run_round<F16, GATED>(what, a, s);
}

template <bool BACK> int run_silu(const char *what, int dtype, const ActArgs &a, hipStream_t s) {
    const int64_t blocks = std::min((a.rows * (a.inner / 8) + 255) / 256, kMaxBlocks);
    return dtype == GG_DTYPE_BF16 ? launch(what, silu_kernel<BF16, BACK>, blocks, 256, s, a)
                                  : launch(what, silu_kernel<F16, BACK>, blocks, 256, s, a);
}

int check_act(int dtype, int64_t rows, int64_t n, const char *name) {
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (rows < 0 || n < 1)
        return fail(GG_ERR_INVALID, "rows must be >= 0 and %s >= 1", name);
    if (n % 8 != 0 || n > 32768)
        return fail(GG_ERR_UNSUPPORTED, "%s must be a multiple of 8 and at most 32768", name);
    return GG_OK;
}

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

int gg_silu_product(int dtype, int out_dtype, int64_t rows, int64_t inner, const void *gu, int64_t gu_stride, void *y,
                    float *scale, void *stream) {
    g_error[0] = 0;
    if (const int st = check_act(dtype, rows, inner, "inner"))
        return st;
    const bool i8 = out_dtype == GG_DTYPE_INT8;
    if (!i8 && out_dtype != dtype)
        return fail(GG_ERR_INVALID, "out_dtype must be dtype or GG_DTYPE_INT8");
    if (rows == 0)
        return GG_OK;
    if (y == nullptr || (i8 && scale == nullptr))
        return fail(GG_ERR_INVALID, i8 ? "y and scale must be device pointers" : "y must be a device pointer");
    if (const int st = check_rows("gu", gu, gu_stride, rows))
        return st;
    if (!aligned(y, i8 ? 8 : 16))
        return fail(GG_ERR_UNSUPPORTED, "y must be 16-byte aligned (int8: 8)");
    const ActArgs a{gu, nullptr, y, scale, rows, gu_stride, 0, static_cast<int>(inner)};
    return i8 ? run_round<true>("silu_product", dtype, a, static_cast<hipStream_t>(stream))
              : run_silu<false>("silu_product", dtype, a, static_cast<hipStream_t>(stream));
}

int gg_silu_product_backward(int dtype, int64_t rows, int64_t inner, const void *grad_y, int64_t grad_y_stride,
                             const void *gu, int64_t gu_stride, void *grad_gu, void *stream) {
    g_error[0] = 0;
    if (const int st = check_act(dtype, rows, inner, "inner"))
        return st;
    if (rows == 0)
        return GG_OK;
    if (grad_gu == nullptr)
        return fail(GG_ERR_INVALID, "grad_gu must be a device pointer");
    if (const int st = check_rows("grad_y", grad_y, grad_y_stride, rows))
        return st;
    if (const int st = check_rows("gu", gu, gu_stride, rows))
        return st;
    if (!aligned(grad_gu, 16))
        return fail(GG_ERR_UNSUPPORTED, "grad_gu must be 16-byte aligned");
    const ActArgs a{gu, grad_y, grad_gu, nullptr, rows, gu_stride, grad_y_stride, static_cast<int>(inner)};
    return run_silu<true>("silu_product_backward", dtype, a, static_cast<hipStream_t>(stream));
}

int gg_quantize_rows(int dtype, int64_t rows, int64_t n, const void *x, int64_t x_stride, int8_t *y, float *scale, void *stream) {
    g_error[0] = 0;
    if (const int st = check_act(dtype, rows, n, "n"))
        return st;
    if (rows == 0)
        return GG_OK;
    if (y == nullptr || scale == nullptr)
        return fail(GG_ERR_INVALID, "y and scale must be device pointers");
    if (const int st = check_rows("x", x, x_stride, rows))
        return st;
    if (!aligned(y, 8))
        return fail(GG_ERR_UNSUPPORTED, "y must be 8-byte aligned");
    const ActArgs a{x, nullptr, y, scale, rows, x_stride, 0, static_cast<int>(n)};
    return run_round<false>("quantize_rows", dtype, a, static_cast<hipStream_t>(stream));
}

} // extern "C"
