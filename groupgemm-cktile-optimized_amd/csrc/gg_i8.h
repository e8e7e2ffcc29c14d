// Between the int8 products' entry point (gg_i8.hip) and the plans of the grouped GEMM (gg_capi.hip). Host-only.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gg {

// Device memory of a call: the group table and its header.
size_t i8_workspace(int group_num);

// Enqueues out = x @ w[g]^T, int8, times the scales, on the persistent or the few-row kernel; a gg_status, with the reason
// of a failure in why. The arguments have been checked (gg_gemm_i8).
int run_i8(int out_dtype, int group_num, int64_t total_m, int64_t n, int64_t k, const int64_t *group_lens,
           const int64_t *group_offs, const void *x, const void *w, const float *x_scale, const float *w_scale, void *out,
           void *workspace, hipStream_t stream, char *why, size_t why_size);

} // namespace gg
