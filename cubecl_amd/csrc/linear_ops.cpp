// linear_ops.cpp -- host side of the operators around a linear layer: mi355_rms_norm and its gradient, the gradient of mi355_gemm_fused's
// epilogue, mi355_global_norm and mi355_clip_by_global_norm.  What a call may not ask for is refused here, before anything is launched.
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <vector>

#include "linear_ops.hpp"
#include "row_span.hpp"

using namespace mi355;

namespace {

// every pointer of a call against the size of what it points to
struct operand { const void *p; int64_t esz; };
bool aligned(std::initializer_list<operand> ops)
{
    return std::all_of(ops.begin(), ops.end(), [](const operand &o) { return (reinterpret_cast<uintptr_t>(o.p) & (uintptr_t)(o.esz - 1)) == 0; });
}

bool float_type(int32_t t) { return t == MI355_DTYPE_F32 || t == MI355_DTYPE_BF16 || t == MI355_DTYPE_F16; }

// ---- the epilogue and its gradient -------------------------------------------------------------------------------------------------------
// rows of a slab: enough workgroups to fill the chip (512 columns wide each), no more than 256 partial rows a batch entry to fold, no less than
// four rows (one a wave).  bf16, us, at most 64 slabs and 1024 workgroups / 256 and 4096 / 1024 and 16384: 512 x 1024 7.6 / 6.5 / 6.5, 8192 x 1024
// 43.7 / 18.9 / 19.4, 4096 x 4096 31.3 / 27.3 / 28.9, 16384 x 8192 161 / 168 / 159.
int64_t slab_rows(const mi355_gemm_fused_grad_desc &d)
{
    const int64_t wide = (d.n + 511) / 512 * d.batch;
    const int64_t slabs = std::max<int64_t>(1, std::min<int64_t>({256, (d.m + 3) / 4, (4096 + wide - 1) / wide}));
    return (d.m + slabs - 1) / slabs;
}
int64_t slab_count(const mi355_gemm_fused_grad_desc &d)
{
    const int64_t r = slab_rows(d);
    return (d.m + r - 1) / r;
}

// (a launch holds fewer than 2^32 threads: 8 columns each, 256 to a workgroup; the fold cuts its columns by itself)
bool grad_desc_sane(const mi355_gemm_fused_grad_desc &d)
{
    return d.m >= 0 && d.n >= 0 && d.batch >= 0 && d.batch <= 65535 && d.n <= (1ll << 31) / std::max<int64_t>(d.batch, 1);
}
uint64_t grad_bytes(const mi355_gemm_fused_grad_desc &d)
{
    return d.m && d.n && d.batch ? (uint64_t)(d.batch * slab_count(d)) * (uint64_t)d.n * sizeof(float) : 0;
}

}  // namespace

namespace mi355 {

int32_t validate_epilogue(mi355_ctx *ctx, const mi355_gemm_desc &d, const mi355_gemm_epilogue &ep, const void *a, const void *b, const void *c)
{
    if (ep.activation < MI355_ACT_NONE || ep.activation > MI355_ACT_SILU)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_fused: unknown activation %d", ep.activation);
    if (ep.bias && ep.dtype_bias != MI355_DTYPE_F32 && ep.dtype_bias != d.dtype_c)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_fused: the bias must be f32 or the output's type (got %d)", ep.dtype_bias);
    if ((ep.residual && ep.ld_residual < d.n) || (ep.pre && ep.ld_pre < d.n))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm_fused: a leading dimension is smaller than the row (residual %lld, pre %lld)",
                    (long long)ep.ld_residual, (long long)ep.ld_pre);
    if (ep.stride_bias < 0 || ep.inc_row_scale < 0 || ep.stride_row_scale < 0 || ep.inc_col_scale < 0 || ep.stride_col_scale < 0 ||
        (ep.residual && ep.stride_residual < 0))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm_fused: negative stride");
    if (ep.pre && !entries_apart(d.batch, d.m, d.n, ep.ld_pre, ep.stride_pre))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm_fused: batch entries of the pre-activation overlap");
    const int64_t ec = (int64_t)dtype_size(d.dtype_c), ea = (int64_t)dtype_size(d.dtype_ab), eb = ep.bias ? (int64_t)dtype_size(ep.dtype_bias) : 1;
    if ((reinterpret_cast<uintptr_t>(ep.residual) | reinterpret_cast<uintptr_t>(ep.pre)) & (uintptr_t)(ec - 1) ||
        (reinterpret_cast<uintptr_t>(ep.bias) & (uintptr_t)(eb - 1)) ||
        ((reinterpret_cast<uintptr_t>(ep.row_scale) | reinterpret_cast<uintptr_t>(ep.col_scale)) & 3u))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: an operand of the epilogue is not aligned to its element");
    const row_span out = span_of(c, d.m, d.n, d.ldc, ec, d.batch, d.stride_c), pre = span_of(ep.pre, d.m, d.n, ep.ld_pre, ec, d.batch, ep.stride_pre);
    const row_span res = span_of(ep.residual, d.m, d.n, ep.ld_residual, ec, d.batch, ep.stride_residual);
    auto vec = [&](const void *p, int64_t count, int64_t inc, int64_t stride) {
        return inc == 1 ? span_of(p, 1, count, 0, 4, d.batch, stride) : span_of(p, count, 1, inc, 4, d.batch, stride);
    };
    const row_span reads[] = {
        d.k ? span_of(a, d.trans_a ? d.k : d.m, d.trans_a ? d.m : d.k, d.lda, ea, d.batch, d.stride_a) : NO_SPAN,
        d.k ? span_of(b, d.trans_b ? d.n : d.k, d.trans_b ? d.k : d.n, d.ldb, ea, d.batch, d.stride_b) : NO_SPAN,
        span_of(ep.bias, 1, d.n, 0, eb, d.batch, ep.stride_bias), vec(ep.row_scale, d.m, ep.inc_row_scale, ep.stride_row_scale),
        vec(ep.col_scale, d.n, ep.inc_col_scale, ep.stride_col_scale)};
    for (const row_span &r : reads)
        if (spans_relation(out, r) != SPANS_APART || spans_relation(pre, r) != SPANS_APART)
            return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: an output overlaps an operand");
    const int at = spans_relation(out, res);
    if (at == SPANS_OVERLAP || (at == SPANS_SAME && d.batch > 1 && ep.stride_residual != d.stride_c))      // (the same bytes, entries and rows exchanged)
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: the residual overlaps the output without being it");
    if (spans_relation(pre, res) != SPANS_APART || spans_relation(pre, out) != SPANS_APART)
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: the pre-activation overlaps the output or the residual");
    return MI355_OK;
}

}  // namespace mi355

MI355_API int32_t mi355_gemm_fused_grad_workspace_bytes(const mi355_gemm_fused_grad_desc *desc, uint64_t *out_bytes)
{
    if (!desc || !out_bytes || !grad_desc_sane(*desc)) return MI355_E_INVALID_ARGUMENT;
    *out_bytes = grad_bytes(*desc);
    return MI355_OK;
}

MI355_API int32_t mi355_gemm_fused_grad(mi355_ctx *ctx, mi355_stream stream, const mi355_gemm_fused_grad_desc *desc, const void *grad_out,
                                        const void *pre, void *grad_pre, void *grad_bias, void *workspace, uint64_t workspace_bytes)
{
    MI355_REQUIRE_CTX(ctx);
    if (!desc) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: descriptor is NULL");
    const mi355_gemm_fused_grad_desc &d = *desc;
    if (!grad_desc_sane(d)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: a size is negative, or more than 65535 batch entries or 2^31 columns over the batch");
    if (d.dtype != MI355_DTYPE_F32 && d.dtype != MI355_DTYPE_BF16 && d.dtype != MI355_DTYPE_F16)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_fused_grad: unsupported dtype %d", d.dtype);
    if (d.activation < MI355_ACT_NONE || d.activation > MI355_ACT_SILU)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_fused_grad: unknown activation %d", d.activation);
    if (grad_bias && d.dtype_bias != MI355_DTYPE_F32 && d.dtype_bias != d.dtype)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_fused_grad: the bias gradient must be f32 or of the operands' type (got %d)", d.dtype_bias);
    if (d.n == 0) return MI355_OK;
    if (!aligned({{grad_bias, (int64_t)dtype_size(d.dtype_bias)}})) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: grad_bias is not aligned to its element");
    hipStream_t s = stream_of(ctx, stream);
    if (d.m == 0 || d.batch == 0) {                                   // sums over no rows: zeros
        if (grad_bias && (d.batch || !d.batch_bias)) launch_fold_columns(s, nullptr, 0, d.n, d.batch_bias ? d.batch : 1, grad_bias, d.dtype_bias);
        check_launch(ctx, "mi355_gemm_fused_grad");
        return MI355_OK;
    }
    if (!grad_out || (!pre && d.activation != MI355_ACT_NONE)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: NULL operand");
    if (!grad_pre && !grad_bias) return MI355_OK;
    const bool reads_pre = d.activation != MI355_ACT_NONE;
    if (d.ld_out < d.n || (reads_pre && d.ld_pre < d.n) || (grad_pre && d.ld_grad < d.n))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm_fused_grad: a leading dimension is smaller than the row");
    if (d.batch > 1 && (d.stride_out < 0 || (reads_pre && d.stride_pre < 0) || (grad_pre && !entries_apart(d.batch, d.m, d.n, d.ld_grad, d.stride_grad))))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm_fused_grad: a batch stride is negative, or entries of grad_pre overlap");
    {
        const int64_t es = (int64_t)dtype_size(d.dtype);
        if (!aligned({{grad_out, es}, {reads_pre ? pre : nullptr, es}, {grad_pre, es}}))
            return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: an operand is not aligned to its element");
    }
    const uint64_t need = grad_bias ? grad_bytes(d) : 0;
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: the workspace has %llu of %llu bytes", (unsigned long long)workspace_bytes, (unsigned long long)need);
    {
        const int64_t es = (int64_t)dtype_size(d.dtype);
        const int64_t bias_len = d.n * (d.batch_bias ? d.batch : 1);
        const row_span reads[] = {span_of(grad_out, d.m, d.n, d.ld_out, es, d.batch, d.stride_out), reads_pre ? span_of(pre, d.m, d.n, d.ld_pre, es, d.batch, d.stride_pre) : NO_SPAN};
        const row_span writes[] = {span_of(grad_pre, d.m, d.n, d.ld_grad, es, d.batch, d.stride_grad), span_of(grad_bias, 1, bias_len, 0, (int64_t)dtype_size(d.dtype_bias)),
                                   span_of(need ? workspace : nullptr, 1, (int64_t)need, 0, 1)};
        const int64_t read_stride[] = {d.stride_out, d.stride_pre};
        for (int w = 0; w < 3; ++w) {
            for (int r = 0; r < 2; ++r) {
                const int rel = spans_relation(writes[w], reads[r]);
                if (rel == SPANS_OVERLAP || (rel == SPANS_SAME && (w != 0 || (d.batch > 1 && read_stride[r] != d.stride_grad))))
                    return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: an output overlaps an operand");
            }
            for (int v = 0; v < w; ++v)
                if (spans_relation(writes[w], writes[v]) != SPANS_APART) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused_grad: two outputs overlap");
        }
    }
    const fused_grad_args a{grad_out, pre, grad_pre, need ? static_cast<float *>(workspace) : nullptr, d.m, d.n, d.batch, slab_rows(d),
                            d.ld_out, d.ld_pre, d.ld_grad, d.stride_out, d.stride_pre, d.stride_grad};
    launch_fused_grad(s, d.dtype, d.activation, a);
    if (grad_bias) {
        const int64_t slabs = slab_count(d);
        if (d.batch_bias) launch_fold_columns(s, static_cast<const float *>(workspace), slabs, d.n, d.batch, grad_bias, d.dtype_bias);
        else launch_fold_columns(s, static_cast<const float *>(workspace), slabs * d.batch, d.n, 1, grad_bias, d.dtype_bias);
    }
    check_launch(ctx, "mi355_gemm_fused_grad");
    return MI355_OK;
}

// ---- norms over rows -------------------------------------------------------------------------------------------------------------------
MI355_API int32_t mi355_rms_norm(mi355_ctx *ctx, mi355_stream stream, const mi355_rms_norm_desc *desc, const void *in, const void *residual,
                                 const void *weight, void *hidden, void *out, void *scales, float *rstd)
{
    MI355_REQUIRE_CTX(ctx);
    if (!desc) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: descriptor is NULL");
    const mi355_rms_norm_desc &d = *desc;
    if (d.rows < 0 || d.cols < 0) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: negative size");
    if (!float_type(d.dtype)) return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm: unsupported input dtype %d", d.dtype);
    if (d.dtype_weight != MI355_DTYPE_F32 && d.dtype_weight != d.dtype)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm: the weight must be f32 or the input's type (got %d)", d.dtype_weight);
    const bool f8 = is_fp8(d.dtype_out);
    if (!f8 && d.dtype_out != MI355_DTYPE_F32 && d.dtype_out != d.dtype)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm: output dtype %d must be f32, the input's type or an 8-bit one", d.dtype_out);
    if (!(d.eps > 0.0f) || !(d.eps < INFINITY)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: eps must be positive and finite");
    if (f8) {
        if (d.scale_block != 0 && d.scale_block != 32) return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm: scale_block %d (0 = by row, or 32)", d.scale_block);
        if (d.scale_block == 32 && d.cols % 32) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: %lld columns are not whole blocks of 32", (long long)d.cols);
    } else if (scales) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: scales belong to an 8-bit output");
    if (d.rows == 0 || d.cols == 0) return MI355_OK;
    if (!in || !out || (f8 && !scales)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: NULL operand");
    if (d.ld_in < d.cols || d.ld_out < d.cols || (residual && d.ld_residual < d.cols) || (hidden && d.ld_hidden < d.cols) ||
        (f8 && d.scale_block && d.ld_scales < d.cols / 32))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_rms_norm: a row stride is smaller than the row");
    const int64_t es = (int64_t)dtype_size(d.dtype), eo = (int64_t)dtype_size(d.dtype_out);
    if (!aligned({{in, es}, {residual, es}, {weight, (int64_t)dtype_size(d.dtype_weight)}, {hidden, es}, {out, eo}, {scales, d.scale_block ? 1 : 4}, {rstd, 4}}))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: an operand is not aligned to its element");
    {
        const row_span reads[] = {span_of(in, d.rows, d.cols, d.ld_in, es), span_of(residual, d.rows, d.cols, d.ld_residual, es),
                                  span_of(weight, 1, d.cols, d.cols, (int64_t)dtype_size(d.dtype_weight))};
        const row_span writes[] = {span_of(hidden, d.rows, d.cols, d.ld_hidden, es), span_of(out, d.rows, d.cols, d.ld_out, eo),
                                   d.scale_block ? span_of(scales, d.rows, d.cols / 32, d.ld_scales, 1) : span_of(scales, 1, d.rows, d.rows, 4),
                                   span_of(rstd, 1, d.rows, d.rows, 4)};
        for (int w = 0; w < 4; ++w) {
            for (int r = 0; r < 3; ++r) {
                const int rel = spans_relation(writes[w], reads[r]);
                // row by row in registers: hidden and a plain output of the input's type may take the place of what is read
                if (rel == SPANS_OVERLAP || (rel == SPANS_SAME && !(w < 2 && r < 2)))
                    return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: an output overlaps an operand");
            }
            for (int v = 0; v < w; ++v)
                if (spans_relation(writes[w], writes[v]) != SPANS_APART) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm: two outputs overlap");
        }
    }
    norm_args a{in, residual, weight, hidden, out, scales, rstd, d.rows, d.cols, d.ld_in, d.ld_residual, d.ld_hidden, d.ld_out, d.ld_scales,
                d.eps, 1.0f / (float)d.cols, d.dtype_weight, d.dtype_out};
    hipStream_t s = stream_of(ctx, stream);
    const int mode = !f8 ? OUT_PLAIN : d.scale_block ? OUT_BLOCK : OUT_ROW;
    launch_rms_norm(s, d.dtype, mode, a);
    check_launch(ctx, "mi355_rms_norm");
    return MI355_OK;
}

MI355_API int32_t mi355_rms_norm_grad_workspace_bytes(const mi355_rms_norm_grad_desc *desc, uint64_t *out_bytes)
{
    if (!desc || !out_bytes || desc->rows < 0 || desc->cols < 0 || desc->cols > GRAD_MAX_COLS) return MI355_E_INVALID_ARGUMENT;
    *out_bytes = desc->rows && desc->cols ? (uint64_t)norm_grad_partials(desc->rows, desc->cols) * (uint64_t)desc->cols * sizeof(float) : 0;
    return MI355_OK;
}

MI355_API int32_t mi355_rms_norm_grad(mi355_ctx *ctx, mi355_stream stream, const mi355_rms_norm_grad_desc *desc, const void *grad_out,
                                      const void *hidden, const void *weight, const float *rstd, const void *grad_hidden, void *grad_in,
                                      void *grad_weight, void *workspace, uint64_t workspace_bytes)
{
    MI355_REQUIRE_CTX(ctx);
    if (!desc) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: descriptor is NULL");
    const mi355_rms_norm_grad_desc &d = *desc;
    if (d.rows < 0 || d.cols < 0 || d.cols > GRAD_MAX_COLS) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: a size is negative, or more than 2^31 columns");
    if (!float_type(d.dtype)) return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm_grad: unsupported dtype %d", d.dtype);
    if ((d.dtype_weight != MI355_DTYPE_F32 && d.dtype_weight != d.dtype) ||
        (grad_weight && d.dtype_grad_weight != MI355_DTYPE_F32 && d.dtype_grad_weight != d.dtype))
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_rms_norm_grad: the weight and its gradient must be f32 or of the operands' type");
    if (d.cols == 0) return MI355_OK;
    if (!aligned({{grad_weight, (int64_t)dtype_size(d.dtype_grad_weight)}})) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: grad_weight is not aligned to its element");
    hipStream_t s = stream_of(ctx, stream);
    if (d.rows == 0) {
        if (grad_weight) launch_fold_columns(s, nullptr, 0, d.cols, 1, grad_weight, d.dtype_grad_weight);      // a sum over no rows: zeros
        check_launch(ctx, "mi355_rms_norm_grad");
        return MI355_OK;
    }
    if (!grad_out || !hidden || !rstd || !grad_in) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: NULL operand");
    if (d.ld_out < d.cols || d.ld_hidden < d.cols || d.ld_in < d.cols || (grad_hidden && d.ld_stream < d.cols))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_rms_norm_grad: a row stride is smaller than the row");
    {
        const int64_t es = (int64_t)dtype_size(d.dtype);
        if (!aligned({{grad_out, es}, {hidden, es}, {weight, (int64_t)dtype_size(d.dtype_weight)}, {rstd, 4}, {grad_hidden, es}, {grad_in, es}}))
            return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: an operand is not aligned to its element");
    }
    const uint64_t need = (uint64_t)norm_grad_partials(d.rows, d.cols) * (uint64_t)d.cols * sizeof(float);
    if (grad_weight && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: the workspace has %llu of %llu bytes", (unsigned long long)workspace_bytes, (unsigned long long)need);
    {
        const int64_t es = (int64_t)dtype_size(d.dtype);
        const row_span reads[] = {span_of(grad_out, d.rows, d.cols, d.ld_out, es), span_of(hidden, d.rows, d.cols, d.ld_hidden, es),
                                  span_of(grad_hidden, d.rows, d.cols, d.ld_stream, es), span_of(rstd, 1, d.rows, d.rows, 4),
                                  span_of(weight, 1, d.cols, d.cols, (int64_t)dtype_size(d.dtype_weight))};
        const row_span writes[] = {span_of(grad_in, d.rows, d.cols, d.ld_in, es),
                                   span_of(grad_weight, 1, d.cols, d.cols, (int64_t)dtype_size(d.dtype_grad_weight)),
                                   span_of(grad_weight ? workspace : nullptr, 1, (int64_t)(need / 4), 0, 4)};
        for (int w = 0; w < 3; ++w) {
            for (int r = 0; r < 5; ++r) {
                const int rel = spans_relation(writes[w], reads[r]);
                if (rel == SPANS_OVERLAP || (rel == SPANS_SAME && !(w == 0 && r < 3)))
                    return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: an output overlaps an operand");
            }
            for (int v = 0; v < w; ++v)
                if (spans_relation(writes[w], writes[v]) != SPANS_APART) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_rms_norm_grad: two outputs overlap");
        }
    }
    norm_grad_args a{grad_out, hidden, weight, grad_hidden, rstd, grad_in, grad_weight ? static_cast<float *>(workspace) : nullptr, d.rows, d.cols,
                     d.ld_out, d.ld_hidden, d.ld_in, d.ld_stream, 1.0f / (float)d.cols, d.dtype_weight};
    launch_rms_norm_grad(s, d.dtype, a);
    if (grad_weight) launch_fold_columns(s, static_cast<const float *>(workspace), norm_grad_partials(d.rows, d.cols), d.cols, 1, grad_weight, d.dtype_grad_weight);
    check_launch(ctx, "mi355_rms_norm_grad");
    return MI355_OK;
}

// ---- norms over tensor lists ------------------------------------------------------------------------------------------------------------
namespace {

bool span_flat(const mi355_tensor_span &t) { return t.rows == 1 || t.row_stride == t.cols; }

struct plan {
    std::vector<flat_table> flat;
    std::vector<rows_table> rows;
};

// The launches a list needs; false: it does not fit the workspace's partial sums.
bool make_plan(const mi355_tensor_span *in, const mi355_tensor_span *out, uint32_t count, plan &p)
{
    for (uint32_t i = 0; i < count; ++i) {
        const mi355_tensor_span &t = in[i];
        if (t.rows == 0 || t.cols == 0) continue;
        const bool flat = span_flat(t) && (!out || span_flat(out[i]));
        const int64_t cols = (int64_t)(flat ? t.rows * t.cols : t.cols), rows = flat ? 1 : (int64_t)t.rows;
        const int64_t per_row = (cols + CHUNK - 1) / CHUNK;
        // a launch counts its chunks in 32 bits; longer tensors (2^45 elements) do not exist
        const int64_t chunks = flat || cols >= CHUNK ? rows * per_row : (rows + rows_per_chunk(cols) - 1) / rows_per_chunk(cols);
        if (chunks > 0x3FFFFFFF) return false;
        if (flat) {
            if (p.flat.empty() || p.flat.back().count == FLAT_MAX || (int64_t)p.flat.back().chunks + chunks > 0x7FFFFFFF) p.flat.push_back(flat_table{});
            flat_table &f = p.flat.back();
            f.t[f.count++] = {t.data, out ? out[i].data : nullptr, cols, f.chunks, t.dtype};
            f.chunks += (uint32_t)chunks;
        } else {
            if (p.rows.empty() || p.rows.back().count == ROWS_MAX || (int64_t)p.rows.back().chunks + chunks > 0x7FFFFFFF) p.rows.push_back(rows_table{});
            rows_table &f = p.rows.back();
            f.t[f.count++] = {t.data, out ? out[i].data : nullptr, rows, cols, (int64_t)t.row_stride, (int64_t)(out ? out[i].row_stride : t.row_stride), f.chunks, t.dtype};
            f.chunks += (uint32_t)chunks;
        }
    }
    return true;
}

int32_t validate_spans(mi355_ctx *ctx, const char *what, const mi355_tensor_span *in, const mi355_tensor_span *out, uint32_t count)
{
    for (uint32_t i = 0; i < count; ++i)
        for (int side = 0; side < (out ? 2 : 1); ++side) {
            const mi355_tensor_span &t = side ? out[i] : in[i];
            if (t.dtype != MI355_DTYPE_F32 && t.dtype != MI355_DTYPE_BF16 && t.dtype != MI355_DTYPE_F16)
                return fail(ctx, MI355_E_UNSUPPORTED, "%s: tensor %u has unsupported dtype %d", what, i, t.dtype);
            if (side && (t.dtype != in[i].dtype || t.rows != in[i].rows || t.cols != in[i].cols))
                return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: output %u differs from its input in shape or type", what, i);
            if (t.rows == 0 || t.cols == 0) continue;
            if (!t.data) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: tensor %u is NULL", what, i);
            if (t.rows > 1 && t.row_stride < t.cols) return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "%s: the rows of tensor %u overlap", what, i);
            if (reinterpret_cast<uintptr_t>(t.data) & (dtype_size(t.dtype) - 1)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: tensor %u is not aligned to its element", what, i);
            if (t.rows > (1ull << 45) / t.cols || (t.rows > 1 && t.row_stride > (1ull << 45) / t.rows)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: tensor %u is too large", what, i);
        }
    return MI355_OK;
}

// Outputs against each other and against the inputs, in the order of their first bytes: only neighbours whose ranges meet are looked at closely.
bool outputs_apart(const mi355_tensor_span *in, const mi355_tensor_span *out, uint32_t count)
{
    struct item { row_span s; uint32_t i; bool is_out; };
    std::vector<item> v;
    v.reserve(2 * (size_t)count);
    for (uint32_t i = 0; i < count; ++i) {
        if (in[i].rows == 0 || in[i].cols == 0) continue;
        const int64_t es = (int64_t)dtype_size(in[i].dtype);
        v.push_back({span_of(in[i].data, in[i].rows, in[i].cols, in[i].row_stride, es), i, false});
        v.push_back({span_of(out[i].data, out[i].rows, out[i].cols, out[i].row_stride, es), i, true});
    }
    std::sort(v.begin(), v.end(), [](const item &a, const item &b) { return a.s.at < b.s.at; });
    // `open`: items whose range has not ended before the current one begins
    std::vector<const item *> open;
    for (const item &x : v) {
        open.erase(std::remove_if(open.begin(), open.end(), [&](const item *o) { return o->s.end() <= x.s.at; }), open.end());
        for (const item *o : open) {
            if (!o->is_out && !x.is_out) continue;
            const int rel = spans_relation(o->s, x.s);
            if (rel == SPANS_APART || (rel == SPANS_SAME && o->i == x.i && o->is_out != x.is_out)) continue;
            return false;
        }
        open.push_back(&x);
    }
    return true;
}

template <class TABLE>
uint32_t grid_of(const TABLE &t, size_t launches) { return std::min<uint32_t>({t.chunks, GRID, (uint32_t)(MAX_PARTIALS / launches)}); }

int32_t run(mi355_ctx *ctx, mi355_stream stream, const char *what, const mi355_tensor_span *in, const mi355_tensor_span *out, uint32_t count, float max_norm,
            float *out_norm, void *workspace, uint64_t workspace_bytes)
{
    if (count && (!in || (max_norm > 0.0f && !out))) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: NULL tensor list", what);
    const int32_t rc = validate_spans(ctx, what, in, out, count);
    if (rc != MI355_OK) return rc;
    if (!workspace || workspace_bytes < MAX_PARTIALS * sizeof(double) || (reinterpret_cast<uintptr_t>(workspace) & 7))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: the workspace has %llu of %llu bytes, or is not 8-byte aligned", what, (unsigned long long)workspace_bytes,
                    (unsigned long long)(MAX_PARTIALS * sizeof(double)));
    if (!aligned({{out_norm, 4}})) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: the norm is not aligned to its element", what);
    if (out && !outputs_apart(in, out, count))
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: an output overlaps another tensor of the list", what);
    {
        const row_span own[] = {span_of(workspace, 1, MAX_PARTIALS, MAX_PARTIALS, 8), span_of(out_norm, 1, 1, 1, 4)};
        bool apart = spans_relation(own[0], own[1]) == SPANS_APART;
        for (uint32_t i = 0; apart && i < count; ++i)
            for (int side = 0; side < (out ? 2 : 1); ++side) {
                const mi355_tensor_span &t = side ? out[i] : in[i];
                const row_span at = span_of(t.data, t.rows, t.cols, t.row_stride, (int64_t)dtype_size(t.dtype));
                apart = apart && spans_relation(at, own[0]) == SPANS_APART && spans_relation(at, own[1]) == SPANS_APART;
            }
        if (!apart) return fail(ctx, MI355_E_INVALID_ARGUMENT, "%s: the norm or the workspace overlaps a tensor", what);
    }
    plan p;
    if (!make_plan(in, out, count, p) || p.flat.size() + p.rows.size() > MAX_PARTIALS)
        return fail(ctx, MI355_E_UNSUPPORTED, "%s: the list is too long", what);
    hipStream_t s = stream_of(ctx, stream);
    double *partial = static_cast<double *>(workspace);
    const size_t launches = p.flat.size() + p.rows.size();
    uint32_t sums = 0;
    for (const flat_table &t : p.flat) {
        const uint32_t g = grid_of(t, launches);
        launch_square_sums(s, t, g, partial + sums);
        sums += g;
    }
    for (const rows_table &t : p.rows) {
        const uint32_t g = grid_of(t, launches);
        launch_square_sums(s, t, g, partial + sums);
        sums += g;
    }
    if (!out || launches == 0) {
        if (out_norm) launch_finish_norm(s, partial, sums, out_norm);
    } else {
        for (size_t i = p.rows.size(); i-- > 0;) {
            launch_scale(s, p.rows[i], std::min(p.rows[i].chunks, GRID), partial, sums, max_norm, out_norm);
            out_norm = nullptr;                             // one launch writes it
        }
        for (size_t i = p.flat.size(); i-- > 0;) {
            launch_scale(s, p.flat[i], std::min(p.flat[i].chunks, GRID), partial, sums, max_norm, out_norm);
            out_norm = nullptr;
        }
    }
    check_launch(ctx, what);
    return MI355_OK;
}

}  // namespace

MI355_API int32_t mi355_global_norm_workspace_bytes(uint64_t *out_bytes)
{
    if (!out_bytes) return MI355_E_INVALID_ARGUMENT;
    *out_bytes = MAX_PARTIALS * sizeof(double);
    return MI355_OK;
}

MI355_API int32_t mi355_global_norm(mi355_ctx *ctx, mi355_stream stream, const mi355_tensor_span *tensors, uint32_t count, float *out_norm, void *workspace,
                                    uint64_t workspace_bytes)
{
    MI355_REQUIRE_CTX(ctx);
    if (!out_norm) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_global_norm: NULL output");
    try {
        return run(ctx, stream, "mi355_global_norm", tensors, nullptr, count, 0.0f, out_norm, workspace, workspace_bytes);
    } catch (...) {
        return fail(ctx, MI355_E_OUT_OF_MEMORY, "mi355_global_norm: out of host memory");
    }
}

MI355_API int32_t mi355_clip_by_global_norm(mi355_ctx *ctx, mi355_stream stream, const mi355_tensor_span *in, const mi355_tensor_span *out, uint32_t count,
                                            float max_norm, float *out_norm, void *workspace, uint64_t workspace_bytes)
{
    MI355_REQUIRE_CTX(ctx);
    if (!(max_norm > 0.0f)) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_clip_by_global_norm: max_norm must be positive");
    try {
        return run(ctx, stream, "mi355_clip_by_global_norm", in, out, count, max_norm, out_norm, workspace, workspace_bytes);
    } catch (...) {
        return fail(ctx, MI355_E_OUT_OF_MEMORY, "mi355_clip_by_global_norm: out of host memory");
    }
}
