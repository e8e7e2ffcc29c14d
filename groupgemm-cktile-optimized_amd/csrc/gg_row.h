// Rows that stay in the registers of the waves that work on them (gg_norm.hip, gg_act.hip): which waves take a row,
// reductions over them, and the 8-bit formats that an output is rounded to.
#pragma once

#include "gg_layer.h"

namespace gg {
namespace layer {

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

constexpr float kTopE4M3 = 448.f, kTopE5M2 = 57344.f, kTopI8 = 127.f; // largest values

// Eight values divided by the scale, as fp8.
__device__ __forceinline__ u32x2 pack_fp8(const float (&v)[8], const Divisor &d, bool e5m2) {
    u32x2 w;
    const float top = e5m2 ? kTopE5M2 : kTopE4M3;
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

// Eight values of a row divided by the row's scale, as int8: quotients as float32 division rounds them (Divisor), to the
// nearest whole number, halves to even. With a finite scale no value of the row is more than 127 scales (and a float32's
// rounding), so nothing needs to be clamped, and in a row without one, which has a NaN or an infinity, all are 0: four
// operations a value where clamps and checks for each would be twelve. Next to 1.5 * 2^23 a float32 steps by one: the sum
// is rounded to it, and its low byte is the number.
__device__ __forceinline__ u32x2 pack_i8(const float (&v)[8], const Divisor &d) {
    u32x2 w{0, 0};
    if (!(d.s < __builtin_inff()))
        return w;
    float y[8];
    if (d.exact) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = v[i] / d.s;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = v[i] * d.inv;
            y[i] = fmaf(-fmaf(y[i], d.s, -v[i]), d.inv, y[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        unsigned q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            q[j] = __float_as_uint(y[4 * i + j] + 12582912.f);
        w[i] = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
    }
    return w;
}

// Scale of the largest |y| (bits of a float >= 0 or NaN): 1 where the quotient is zero or subnormal, which a division
// by it could turn into NaN or a value of few bits.
__device__ __forceinline__ float scale_of(unsigned top_bits, float format_top) {
    const float s = __uint_as_float(top_bits) / format_top;
    return s < 1.17549435e-38f ? 1.f : s;
}
// A value that every lane of the wave has, as a scalar (what depends on it branches for the wave).
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(__float_as_uint(v)))));
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

// Few rows: a row's latency counts, and not how many are in flight. Then (WIDE) sixteen waves take a row of more than 2048
// values, and grad_weight is summed from g and h again, which are in the caches, instead of from partial sums, which would be
// as many bytes as the rows. us, sixteen waves and four: norm of 5 rows of 7168 3.9, 5.1, of 256 5.5, 7.3, 512 8.4, 10.8, 1024
// 14.5, 14.8; of 512 rows of 4096 5.7, 5.6, 1024 10.8, 9.5; 256 of 14336 8.5, 14.0. Backward, with the sums and without:
// 64 of 7168 7.1, 9.1, 481 of 13456 22.2, 34.3, 512 of 7168 16.6, 18.1, 512 of 4096 13.9, 12.4, 1024 of 8192 27.6, 27.4.
inline bool few(int64_t rows, int64_t hidden) { return hidden > 1024 && rows <= (hidden > 5120 ? 512 : 256); }

template <bool WIDE> inline int waves_per_row(int64_t hidden) {
    return hidden <= 1024 ? 1 : hidden <= (WIDE ? 2048 : 16384) ? 4 : 16;
}

inline int64_t row_blocks(int64_t rows, int64_t hidden) { return hidden <= 1024 ? (rows + 3) / 4 : rows; }

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

// A matrix operand: rows at least hidden apart, 16-byte pieces.
inline int check_rows(const char *name, const void *p, int64_t stride, int64_t rows) {
    if (rows > 0 && p == nullptr)
        return fail(GG_ERR_INVALID, "%s is null", name);
    if (rows > 1 && stride < 0)
        return fail(GG_ERR_INVALID, "%s has a negative row stride", name);
    if (!aligned(p, 16) || (rows > 1 && stride % 8 != 0))
        return fail(GG_ERR_UNSUPPORTED, "%s must be 16-byte aligned with row strides of multiples of 8", name);
    return GG_OK;
}

} // namespace layer
} // namespace gg
