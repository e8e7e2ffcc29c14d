// Shared pieces of the layer operators (gg_norm.hip, gg_route.hip, gg_rows.hip, gg_w4.hip): the
// message of the last failed call, argument checks, 16-byte vectors of 16-bit values as float32 and
// reductions over the lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "gg_moe_layer.h"

namespace gg {
namespace layer {

// A fixed buffer, so that no entry point can throw. Defined in gg_norm.hip.
extern thread_local char g_error[256];

inline int fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return status;
}

// One launch on `stream`; its own status, not one that an earlier call of the process left behind.
template <typename... P>
int launch(const char *what, void (*kernel)(P...), int64_t grid, int threads, hipStream_t stream,
           std::type_identity_t<P>... args) {
    void            *ptrs[] = {&args...};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(static_cast<unsigned>(grid)),
                                         dim3(static_cast<unsigned>(threads)), ptrs, 0, stream);
    return e == hipSuccess ? static_cast<int>(GG_OK) : fail(GG_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// Workgroups of a kernel that the GPU holds at once.
template <typename... P> int resident_blocks(void (*kernel)(P...), int threads) {
    int dev = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, reinterpret_cast<const void *>(kernel), threads, 0) != hipSuccess ||
        cus < 1 || per_cu < 1)
        return 1024;
    return cus * per_cu;
}

inline bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline bool is16(int dtype) { return dtype == GG_DTYPE_BF16 || dtype == GG_DTYPE_FP16; }
inline bool is8(int dtype) { return dtype == GG_DTYPE_FP8_E4M3 || dtype == GG_DTYPE_FP8_E5M2; }

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16   bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 16-bit element types. pair: two of them from the halves of a word; word: the reverse, rounded to nearest even.
struct BF16 {
    static __device__ __forceinline__ void pair(unsigned w, float &lo, float &hi) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ unsigned word(float lo, float hi) {
        return __builtin_bit_cast(unsigned, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
    }
};
struct F16 {
    static __device__ __forceinline__ void pair(unsigned w, float &lo, float &hi) {
        const f16x2 v = __builtin_bit_cast(f16x2, w);
        lo            = static_cast<float>(v[0]);
        hi            = static_cast<float>(v[1]);
    }
    static __device__ __forceinline__ unsigned word(float lo, float hi) {
        return __builtin_bit_cast(unsigned, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
    }
};

// Sixteen bytes that nothing reads again soon: they go past the caches, which keep what comes after.
__device__ __forceinline__ u32x4 load_once(const void *p) { return __builtin_nontemporal_load(static_cast<const u32x4 *>(p)); }

// Eight values of 16 bytes.
template <typename T> __device__ __forceinline__ void unpack8(const u32x4 &w, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        T::pair(w[i], v[2 * i], v[2 * i + 1]);
}
template <typename T> __device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = T::word(v[2 * i], v[2 * i + 1]);
    return w;
}

// Between LDS accesses of one wave's lanes to each other's values (the hardware keeps a wave's own order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// op over groups of L consecutive lanes, in every lane of the group, in the same order in every run. Within a row of
// 16 lanes by register moves between lanes (pairs, quads, halves and rows mirrored), then by swaps of rows and halves:
// a step costs an instruction or two, where a shuffle goes through the LDS unit.
template <int CTRL> __device__ __forceinline__ unsigned lane_move(unsigned v) {
    return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
template <int L, typename F> __device__ __forceinline__ unsigned group_reduce(unsigned v, F op) {
    if constexpr (L >= 2)
        v = op(v, lane_move<0xb1>(v)); // quad_perm 1 0 3 2
    if constexpr (L >= 4)
        v = op(v, lane_move<0x4e>(v)); // quad_perm 2 3 0 1
    if constexpr (L >= 8)
        v = op(v, lane_move<0x141>(v)); // row_half_mirror
    if constexpr (L >= 16)
        v = op(v, lane_move<0x140>(v)); // row_mirror
    if constexpr (L >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v            = op(r[0], r[1]);
    }
    if constexpr (L >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v            = op(r[0], r[1]);
    }
    return v;
}
template <int L> __device__ __forceinline__ unsigned group_max(unsigned v) {
    return group_reduce<L>(v, [](unsigned x, unsigned y) { return max(x, y); });
}
template <int L> __device__ __forceinline__ float group_sum(float v) {
    return __uint_as_float(group_reduce<L>(__float_as_uint(v), [](unsigned x, unsigned y) {
        return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
    }));
}
// Sum over the lanes of the same number in the wave's groups of L >= 16 lanes.
template <int L> __device__ __forceinline__ float rows_sum(float v) {
    if constexpr (L < 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v            = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (L < 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v            = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
__device__ __forceinline__ float    wave_sum(float v) { return group_sum<64>(v); }
__device__ __forceinline__ unsigned wave_max(unsigned v) { return group_max<64>(v); }

} // namespace layer
} // namespace gg
