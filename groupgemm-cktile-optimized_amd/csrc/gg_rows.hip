// Rows of the experts: dispatch, combine and their gradients (gg_dispatch, gg_combine, .. in
// include/gg_moe_layer.h).
//
// Every kernel moves rows of hidden values in 16-byte pieces between a token's row and the top_k rows
// that its slots have in expert order. Bound by HBM: the tokens' rows are read or written once, the
// experts' rows once. Measured, 4096 tokens of 7168 to 8 experts each: dispatch of fp8 46 us (5.7 TB/s), of int8
// with scales 48 (5.5), combine of bf16 108
// (4.9); 4160 tokens of 2880 to 4: combine_backward 34 (6.3 TB/s: part of y comes from the Infinity Cache).
#include <algorithm>

#include "gg_layer.h"

namespace gg {
namespace layer {
namespace {

struct RowArgs {
    const void    *in, *grad; // rows read: tokens' (scattering kernels) or experts'; combine_backward: y
    void          *out;
    const int     *rows;
    const float   *weights;
    float         *grad_weights;
    const int64_t *offs;
    const float   *scale;     // dispatch with scales: of each token's row,
    float         *out_scale; // and of each row that is written
    int64_t        tokens, stride; // stride of the tokens' rows that are read, in bytes
    int            top_k, experts, pieces; // 16-byte pieces of a row
};

// Whether a slot has a row: not -1, and whatever a caller put there, inside the experts' rows.
__device__ __forceinline__ bool has_row(const RowArgs &a, int64_t row) {
    return static_cast<uint64_t>(row) < static_cast<uint64_t>(a.tokens * a.top_k);
}

template <bool PAST> __device__ __forceinline__ void store(u32x4 *p, const u32x4 &v) {
    if constexpr (PAST)
        __builtin_nontemporal_store(v, p);
    else
        *p = v;
}

// Rows past the last expert's: one in `grid` of them for each workgroup.
__device__ __forceinline__ void zero_tail(const RowArgs &a) {
    const int64_t pairs = a.tokens * a.top_k;
    for (int64_t row = max(a.offs[a.experts], int64_t(0)) + blockIdx.x; row < pairs; row += gridDim.x)
        for (int i = threadIdx.x; i < a.pieces; i += blockDim.x)
            static_cast<u32x4 *>(a.out)[row * a.pieces + i] = u32x4{0, 0, 0, 0};
}

// A token's row to the rows of its slots: read once, written top_k times. PAST: the stores go past the caches. SCALED: the
// row's scale goes with it (top_k <= 32, and a workgroup has 64 threads at least).
template <bool PAST, bool SCALED> __global__ void __launch_bounds__(1024) dispatch_kernel(const RowArgs a) {
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const u32x4 *x    = reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.in) + t * a.stride);
        const int   *rows = a.rows + t * a.top_k;
        if constexpr (SCALED) {
            if (static_cast<int>(threadIdx.x) < a.top_k) {
                const int64_t row = rows[threadIdx.x];
                if (has_row(a, row))
                    a.out_scale[row] = a.scale[t];
            }
        }
        for (int i = threadIdx.x; i < a.pieces; i += blockDim.x) {
            const u32x4 v = x[i];
            for (int s = 0; s < a.top_k; ++s) {
                const int64_t row = rows[s];
                if (has_row(a, row))
                    store<PAST>(static_cast<u32x4 *>(a.out) + row * a.pieces + i, v);
            }
        }
    }
    zero_tail(a);
    if constexpr (SCALED) {
        const int64_t pairs = a.tokens * a.top_k;
        for (int64_t row = max(a.offs[a.experts], int64_t(0)) + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; row < pairs;
             row += static_cast<int64_t>(gridDim.x) * blockDim.x)
            a.out_scale[row] = 0.f;
    }
}

// out[t] = sum of the rows of its slots (WEIGHTED: times their weights), in the order of the slots, four of whose
// pieces are asked for at a time (32768 x 2 rows of 2048: 76.6 us, eight 94.9).
template <typename T, bool WEIGHTED> __global__ void __launch_bounds__(1024) combine_kernel(const RowArgs a) {
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int   *rows = a.rows + t * a.top_k;
        const float *w    = WEIGHTED ? a.weights + t * a.top_k : nullptr;
        for (int i = threadIdx.x; i < a.pieces; i += blockDim.x) {
            float sum[8] = {};
            for (int s0 = 0; s0 < a.top_k; s0 += 4) {
                u32x4 in[4];
                float c[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int64_t row = s0 + s < a.top_k ? rows[s0 + s] : -1;
                    in[s]             = u32x4{0, 0, 0, 0}; // (a zero adds nothing, whatever the weight of a missing slot)
                    c[s]              = 0.f;
                    if (has_row(a, row)) {
                        in[s] = static_cast<const u32x4 *>(a.in)[row * a.pieces + i];
                        c[s]  = WEIGHTED ? w[s0 + s] : 1.f;
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    float v[8];
                    unpack8<T>(in[s], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        sum[j] = WEIGHTED ? fmaf(c[s], v[j], sum[j]) : sum[j] + v[j];
                }
            }
            static_cast<u32x4 *>(a.out)[t * a.pieces + i] = pack8<T>(sum);
        }
    }
}

// One wave for each (token, slot) pair: grad_y's row is the weight times the token's gradient, the weight's
// gradient the product of that gradient with y's row.
template <typename T, bool PAST> __global__ void __launch_bounds__(256) combine_back_kernel(const RowArgs a) {
    const int     lane = threadIdx.x & 63;
    const int64_t pairs = a.tokens * a.top_k;
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); p < pairs; p += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t row = a.rows[p];
        float         dot = 0.f;
        if (has_row(a, row)) {
            const u32x4 *g = reinterpret_cast<const u32x4 *>(static_cast<const char *>(a.grad) + p / a.top_k * a.stride);
            const u32x4 *y = static_cast<const u32x4 *>(a.in) + row * a.pieces;
            u32x4       *o = static_cast<u32x4 *>(a.out) + row * a.pieces;
            const float  w = a.weights[p];
            for (int i = lane; i < a.pieces; i += 64) {
                float gv[8], yv[8];
                unpack8<T>(g[i], gv);
                unpack8<T>(load_once(y + i), yv);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    dot = fmaf(gv[j], yv[j], dot);
                    gv[j] *= w;
                }
                store<PAST>(o + i, pack8<T>(gv));
            }
        }
        dot = wave_sum(dot);
        if (lane == 0)
            a.grad_weights[p] = dot;
    }
    zero_tail(a);
}

constexpr int64_t kMaxGrid = int64_t(1) << 20;

// Threads of a workgroup that takes one row: all of its pieces at once up to 1024, else in equal parts (64 tokens of
// 8 x 7168 combine in 4.7 us with 1024 threads, 9.0 with 256; 4096 in 108 and 113).
int row_threads(int pieces) {
    const int passes = (pieces + 1023) / 1024;
    return ((pieces + passes - 1) / passes + 63) / 64 * 64;
}

// Whether rows written by a scatter go past the caches: where they are more than the 256 MB Infinity Cache keeps for
// who reads them next. Measured (us, stores past the caches and plain): dispatch of 235 MB 47 and 56, of 268 MB
// 61 and 76; 96 MB 20 and 20; combine_backward of 470 MB 184 and 198, of 67 MB 33 and 29.
bool past_caches(const RowArgs &a) { return a.tokens * a.top_k * a.pieces * 16 > int64_t(192) << 20; }

int check_rows(int es, int64_t tokens, int top_k, int64_t hidden) {
    if (tokens < 0 || top_k < 1 || hidden < 1)
        return fail(GG_ERR_INVALID, "tokens must be >= 0, top_k and hidden >= 1");
    if (top_k > 32 || tokens > INT32_MAX / top_k)
        return fail(GG_ERR_UNSUPPORTED, "top_k must be at most 32 and tokens * top_k below 2^31");
    if (hidden > (128 << 10) / es || hidden * es % 16 != 0)
        return fail(GG_ERR_UNSUPPORTED, "a row must be a multiple of 16 bytes and at most 128 KB");
    return GG_OK;
}

bool pieces(const void *p) { return p != nullptr && aligned(p, 16); }

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

// Both forms of dispatch (scaled: scale and xs_scale).
static int dispatch_rows(bool scaled, int elem_size, int64_t tokens, int top_k, int64_t hidden, int experts, const void *x,
                         int64_t stride, const float *scale, const int *rows, const int64_t *offs, void *xs, float *xs_scale,
                         void *stream) {
    g_error[0] = 0;
    if (elem_size != 1 && elem_size != 2 && elem_size != 4)
        return fail(GG_ERR_INVALID, "elem_size must be 1, 2 or 4");
    if (const int st = check_rows(elem_size, tokens, top_k, hidden))
        return st;
    if (tokens == 0)
        return GG_OK;
    if (experts < 0 || rows == nullptr || offs == nullptr)
        return fail(GG_ERR_INVALID, "rows and offs must be device pointers");
    if (tokens > 1 && stride < 0)
        return fail(GG_ERR_INVALID, "x has a negative row stride");
    if (scaled && (scale == nullptr || xs_scale == nullptr))
        return fail(GG_ERR_INVALID, "scale and xs_scale must be device pointers");
    if (!pieces(x) || !pieces(xs) || (tokens > 1 && stride * elem_size % 16 != 0))
        return fail(GG_ERR_UNSUPPORTED, "x and xs must be 16-byte aligned, strides multiples of 16 bytes");
    RowArgs a{};
    a.in      = x;
    a.out     = xs;
    a.rows    = rows;
    a.offs    = offs;
    a.tokens  = tokens;
    a.stride  = stride * elem_size;
    a.top_k   = top_k;
    a.experts = experts;
    a.pieces  = static_cast<int>(hidden * elem_size / 16);
    const bool past = past_caches(a);
    const auto plain = past ? dispatch_kernel<true, false> : dispatch_kernel<false, false>;
    if (!scaled)
        return launch("dispatch", plain, std::min(tokens, kMaxGrid), row_threads(a.pieces), static_cast<hipStream_t>(stream), a);
    a.scale     = scale;
    a.out_scale = xs_scale;
    return launch("dispatch_scaled", past ? dispatch_kernel<true, true> : dispatch_kernel<false, true>, std::min(tokens, kMaxGrid),
                  row_threads(a.pieces), static_cast<hipStream_t>(stream), a);
}

int gg_dispatch(int elem_size, int64_t tokens, int top_k, int64_t hidden, int experts, const void *x, int64_t stride,
                const int *rows, const int64_t *offs, void *xs, void *stream) {
    return dispatch_rows(false, elem_size, tokens, top_k, hidden, experts, x, stride, nullptr, rows, offs, xs, nullptr, stream);
}

int gg_dispatch_scaled(int elem_size, int64_t tokens, int top_k, int64_t hidden, int experts, const void *x, int64_t stride,
                       const float *scale, const int *rows, const int64_t *offs, void *xs, float *xs_scale, void *stream) {
    return dispatch_rows(true, elem_size, tokens, top_k, hidden, experts, x, stride, scale, rows, offs, xs, xs_scale, stream);
}

static int sum_rows(const char *what, bool weighted, int dtype, int64_t tokens, int top_k, int64_t hidden, const void *y,
                    const int *rows, const float *weights, void *out, void *stream) {
    g_error[0] = 0;
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (const int st = check_rows(2, tokens, top_k, hidden))
        return st;
    if (tokens == 0)
        return GG_OK;
    if (rows == nullptr || (weighted && weights == nullptr))
        return fail(GG_ERR_INVALID, "rows and weights must be device pointers");
    if (!pieces(y) || !pieces(out))
        return fail(GG_ERR_UNSUPPORTED, "inputs and outputs must be 16-byte aligned device pointers");
    RowArgs a{};
    a.in      = y;
    a.out     = out;
    a.rows    = rows;
    a.weights = weights;
    a.tokens  = tokens;
    a.top_k   = top_k;
    a.pieces  = static_cast<int>(hidden / 8);
    const hipStream_t s       = static_cast<hipStream_t>(stream);
    const int64_t     grid    = std::min(tokens, kMaxGrid);
    const int         threads = row_threads(a.pieces);
    if (dtype == GG_DTYPE_BF16)
        return launch(what, weighted ? combine_kernel<BF16, true> : combine_kernel<BF16, false>, grid, threads, s, a);
    return launch(what, weighted ? combine_kernel<F16, true> : combine_kernel<F16, false>, grid, threads, s, a);
}

int gg_dispatch_backward(int dtype, int64_t tokens, int top_k, int64_t hidden, const void *grad_xs, const int *rows,
                         void *grad_x, void *stream) {
    return sum_rows("dispatch_backward", false, dtype, tokens, top_k, hidden, grad_xs, rows, nullptr, grad_x, stream);
}

int gg_combine(int dtype, int64_t tokens, int top_k, int64_t hidden, const void *y, const int *rows,
               const float *weights, void *out, void *stream) {
    return sum_rows("combine", true, dtype, tokens, top_k, hidden, y, rows, weights, out, stream);
}

int gg_combine_backward(int dtype, int64_t tokens, int top_k, int64_t hidden, int experts, const void *grad_out,
                        int64_t stride, const void *y, const int *rows, const int64_t *offs, const float *weights,
                        void *grad_y, float *grad_weights, void *stream) {
    g_error[0] = 0;
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (const int st = check_rows(2, tokens, top_k, hidden))
        return st;
    if (tokens == 0)
        return GG_OK;
    if (experts < 0 || rows == nullptr || offs == nullptr || weights == nullptr || grad_weights == nullptr)
        return fail(GG_ERR_INVALID, "rows, offs, weights and grad_weights must be device pointers");
    if (tokens > 1 && stride < 0)
        return fail(GG_ERR_INVALID, "grad_out has a negative row stride");
    if (!pieces(grad_out) || !pieces(y) || !pieces(grad_y) || (tokens > 1 && stride % 8 != 0))
        return fail(GG_ERR_UNSUPPORTED, "grad_out, y and grad_y must be 16-byte aligned, strides multiples of 8");
    RowArgs a{};
    a.in           = y;
    a.grad         = grad_out;
    a.out          = grad_y;
    a.rows         = rows;
    a.weights      = weights;
    a.grad_weights = grad_weights;
    a.offs         = offs;
    a.tokens       = tokens;
    a.stride       = stride * 2;
    a.top_k        = top_k;
    a.experts      = experts;
    a.pieces       = static_cast<int>(hidden / 8);
    const int64_t grid = std::min((tokens * top_k + 3) / 4, kMaxGrid);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (past_caches(a))
        return launch("combine_backward", dtype == GG_DTYPE_BF16 ? combine_back_kernel<BF16, true> : combine_back_kernel<F16, true>,
                      grid, 256, s, a);
    return launch("combine_backward", dtype == GG_DTYPE_BF16 ? combine_back_kernel<BF16, false> : combine_back_kernel<F16, false>,
                  grid, 256, s, a);
}

} // extern "C"
