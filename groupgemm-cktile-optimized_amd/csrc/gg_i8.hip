// Grouped products in 8-bit integers with a scale for each row and each output channel (gg_gemm_i8 in
// include/gg_moe_layer.h): out[m, n] = sx[m] sw[g, n] sum_k qx[m, k] qw[g, n, k].
//
// The sums are exact in int32; each is made a float32 once, takes both scales and is rounded to 16 bits. They run on the
// grouped GEMM's own kernels: many rows on the persistent 256 x 256 one (gg_kernel_impl.h, mode kInI8), few on the
// few-row one (gg_few.hip), chosen by the launch-time model of the device-size plans (choose_few_rows).
// What bounds it: few rows, the reading of w (8 of 32 groups with a row each, 4096 x 7168: 41 us, 5.7 TB/s); many, the
// matrix pipes (8 groups of 32768 rows in all, 4096 x 7168: 690 us, 2.8 POP/s).
#include "gg_i8.h"

#include "gg_layer.h"
#include "gg_schedule.h"

using namespace gg::layer;

extern "C" {

size_t gg_gemm_i8_workspace(int group_num) { return group_num < 1 ? 0 : gg::i8_workspace(group_num); }

int gg_gemm_i8(int out_dtype, int group_num, int64_t total_m, int64_t n, int64_t k, const int64_t *group_lens,
               const int64_t *group_offs, const int8_t *x, const int8_t *w, const float *x_scale, const float *w_scale,
               void *out, void *workspace, size_t workspace_bytes, void *stream) {
    g_error[0] = 0;
    if (!is16(out_dtype))
        return fail(GG_ERR_INVALID, "out_dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (group_num < 0 || total_m < 0 || n < 0 || k < 1)
        return fail(GG_ERR_INVALID, "group_num, total_m and n must be >= 0 and k >= 1");
    if (n % 8 != 0 || k % 16 != 0)
        return fail(GG_ERR_UNSUPPORTED, "N must be a multiple of 8 and K of 16");
    if (n > (1 << 21) || k >= (1 << 17) || group_num > 8192 || total_m > (1 << 27))
        return fail(GG_ERR_UNSUPPORTED, "N must be at most 2097152, K below 131072, groups at most 8192 and rows at most 134217728");
    if ((gg::cdiv(total_m, gg::kTileM) + group_num) * gg::cdiv(n, gg::kTileN) > gg::kMaxLoopTiles)
        return fail(GG_ERR_UNSUPPORTED, "too many output tiles for 32-bit indices");
    if (group_num == 0 || total_m == 0 || n == 0)
        return GG_OK;
    if (group_lens == nullptr || x == nullptr || w == nullptr || x_scale == nullptr || w_scale == nullptr || out == nullptr)
        return fail(GG_ERR_INVALID, "group_lens, x, w, x_scale, w_scale and out must be device pointers");
    if (!aligned(x, 16) || !aligned(w, 16) || !aligned(out, 16) || !aligned(w_scale, 16) || !aligned(x_scale, 4))
        return fail(GG_ERR_UNSUPPORTED, "x, w, w_scale and out must be 16-byte aligned, x_scale 4-byte");
    if (workspace_bytes < gg::i8_workspace(group_num) || workspace == nullptr || !aligned(workspace, 16))
        return fail(GG_ERR_WORKSPACE, "workspace must be 16-byte aligned and of gg_gemm_i8_workspace(group_num) bytes");
    return gg::run_i8(out_dtype, group_num, total_m, n, k, group_lens, group_offs, x, w, x_scale, w_scale, out, workspace,
                      static_cast<hipStream_t>(stream), g_error, sizeof(g_error));
}

} // extern "C"
