// Stand-ins for the launches behind cubecl_amd/csrc/linear_ops.cpp (test infrastructure, like the rest of this folder): they count themselves and
// remember what they were given, so that the argument checks of the operators around a linear layer run on a box without a device.
// mi355_gemm_fused is the product's epilogue check without the product.
#include "../../cubecl_amd/csrc/linear_ops.hpp"

namespace {
struct seen {
    uint64_t norm, norm_grad, fold, epilogue, fused_grad, sums, scale, finish, chunks, partials;
} log_;
}  // namespace

namespace mi355 {

void launch_rms_norm(hipStream_t, int32_t, int, const norm_args &) { ++log_.norm; }
void launch_rms_norm_grad(hipStream_t, int32_t, const norm_grad_args &) { ++log_.norm_grad; }
void launch_fold_columns(hipStream_t, const float *, int64_t, int64_t, int64_t, void *, int32_t) { ++log_.fold; }
void launch_fused_grad(hipStream_t, int32_t, int32_t, const fused_grad_args &) { ++log_.fused_grad; }
void launch_square_sums(hipStream_t, const flat_table &t, uint32_t grid, double *) { ++log_.sums; log_.chunks += t.chunks; log_.partials += grid; }
void launch_square_sums(hipStream_t, const rows_table &t, uint32_t grid, double *) { ++log_.sums; log_.chunks += t.chunks; log_.partials += grid; }
void launch_scale(hipStream_t, const flat_table &, uint32_t, const double *, uint32_t, float, float *) { ++log_.scale; }
void launch_scale(hipStream_t, const rows_table &, uint32_t, const double *, uint32_t, float, float *) { ++log_.scale; }
void launch_finish_norm(hipStream_t, const double *, uint32_t, float *) { ++log_.finish; }

}  // namespace mi355

MI355_API int32_t mi355_gemm_fused(mi355_ctx *ctx, mi355_stream, const mi355_gemm_desc *desc, const mi355_gemm_epilogue *epilogue, const void *a, const void *b, void *c)
{
    MI355_REQUIRE_CTX(ctx);
    if (!epilogue) return mi355::fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: the epilogue is NULL");
    const int32_t rc = mi355::validate_epilogue(ctx, *desc, *epilogue, a, b, c);
    if (rc == MI355_OK) ++log_.epilogue;
    return rc;
}

extern "C" __attribute__((visibility("default"))) void lineartest_log(uint64_t *out, int32_t clear)
{
    memcpy(out, &log_, sizeof log_);
    if (clear) log_ = seen{};
}
