// linear_ops.hpp -- what linear_ops.cpp (argument checks, sizes, launch order) and the kernels' files share.
#pragma once

#include <algorithm>

#include "internal.hpp"

namespace mi355 {

// ---- rms_norm.hip
enum { OUT_PLAIN = 0, OUT_ROW = 1, OUT_BLOCK = 2 };

struct norm_args {
    const void *in, *residual, *weight;
    void *hidden, *out, *scales;
    float *rstd;
    int64_t rows, cols, ld_in, ld_residual, ld_hidden, ld_out, ld_scales;
    float eps, inv_cols;
    int32_t dtype_weight, dtype_out;
};
struct norm_grad_args {
    const void *grad_out, *hidden, *weight, *grad_hidden;
    const float *rstd;
    void *grad_in;
    float *partial;           // [workgroups][cols], NULL: no weight gradient
    int64_t rows, cols, ld_out, ld_hidden, ld_in, ld_stream;
    float inv_cols;
    int32_t dtype_weight;
};

// Threads and pieces for rows of `cols` elements (0 threads: the looping kernels).  Few rows leave most of the chip idle, and then
// the row's own latency is what is waited for: as many threads as hold it in one piece.  bf16, us, 1024 threads / 256: 8 x 8192 3.7 / 5.1,
// 256 x 4096 4.5 / 5.0, 512 x 8192 7.5 / 7.9, but 1024 x 4096 11.1 / 6.6, 1024 x 8192 13.6 / 11.6, 8192 x 4096 67 / 29 (a barrier's wait for sixteen
// waves has no other workgroup on the CU to hide behind).  One wave / 256 threads for 4096 rows of 1024: 6.7 / 9.3.
struct row_shape { int threads, pieces; };
inline row_shape shape_for(int64_t rows, int64_t cols)
{
    if (cols > 16384) return {0, 0};
    if (cols <= 512) return {64, 1};
    const bool few = rows <= 512;
    if (cols <= 1024 && !few) return {64, 2};
    if (cols <= 2048) return {256, 1};
    if (few && cols <= 8192) return {1024, 1};
    if (cols <= 4096) return {256, 2};
    if (cols <= 8192) return {256, 4};
    return {1024, 2};
}

// The gradient keeps the weight and its gradient in registers too: rows above 4096 are held by 1024 threads in one piece (us, 1024 / 256
// threads: 512 x 8192 13.7 / 17.8, 1024 x 8192 18.3 / 21.6, 4096 x 8192 45.2 / 48.5, but 2048 x 4096 18.9 / 18.1 and 8192 x 4096 51.5 / 42.8), the
// longest by half the threads with twice the registers each (1024 x 2 pieces spills).
inline row_shape grad_shape_for(int64_t rows, int64_t cols)
{
    if (cols > 4096 && cols <= 8192) return {1024, 1};
    const row_shape sh = shape_for(rows, cols);
    return sh.threads == 1024 && sh.pieces == 2 ? row_shape{512, 4} : sh;
}

// workgroups of the gradient: each walks rows / grid of them and leaves one partial row of the weight's gradient.  Two (512 threads and up: one)
// a CU; us, 512 / 256 workgroups: 2048 x 4096 18.1 / 20.7, 8192 x 4096 42.8 / 56.9, 512 x 8192 13.7 / 15.2; 1024 workgroups leave
// twice the partial rows to fold: 2048 x 4096 19.9, 8192 x 4096 49.4, 512 x 8192 15.9.
constexpr int64_t GRAD_WGS = 512;
inline int64_t norm_grad_wgs(int64_t rows, const row_shape &sh)
{
    return std::min(sh.threads == 64 ? (rows + 3) / 4 : rows, sh.threads >= 512 ? GRAD_WGS / 2 : GRAD_WGS);
}
// ... and of the kernel for rows beyond the registers, eight columns a thread: slabs of rows, so that a launch keeps below 2^32 threads
constexpr int64_t LONG_SLABS = 64, GRAD_MAX_COLS = 1ll << 31;
inline int64_t norm_grad_slabs(int64_t rows, int64_t cols)
{
    return std::min(rows, std::clamp<int64_t>((1ll << 31) / ((cols + 2047) / 2048 * 256), 1, LONG_SLABS));
}
inline int64_t norm_grad_partials(int64_t rows, int64_t cols)
{
    const row_shape sh = grad_shape_for(rows, cols);
    if (sh.threads == 0) return norm_grad_slabs(rows, cols);
    return norm_grad_wgs(rows, sh);
}

void launch_rms_norm(hipStream_t s, int32_t dtype, int mode, const norm_args &a);
void launch_rms_norm_grad(hipStream_t s, int32_t dtype, const norm_grad_args &a);
// Column sums take 1024 threads for 64 columns and a launch holds fewer than 2^32 threads: f(first column, workgroups wide, first batch entry,
// batch entries) for each launch that `cols` columns of `batch` entries need.
constexpr int64_t FOLD_COLS = 64, FOLD_WGS = 1 << 21;
template <class F>
void each_fold_launch(int64_t cols, int64_t batch, F f)
{
    for (int64_t c = 0; c < cols; c += FOLD_COLS * FOLD_WGS) {
        const int64_t wide = (std::min(cols - c, FOLD_COLS * FOLD_WGS) + FOLD_COLS - 1) / FOLD_COLS, most = std::clamp<int64_t>(FOLD_WGS / wide, 1, 65535);
        for (int64_t b = 0; b < batch; b += most) f(c, wide, b, std::min(most, batch - b));
    }
}
// column sums of f32 partial rows, [batch][count][cols] -> out [batch][cols] in `dtype`; count 0: zeros
void launch_fold_columns(hipStream_t s, const float *partial, int64_t count, int64_t cols, int64_t batch, void *out, int32_t dtype);

// ---- the epilogue of mi355_gemm_fused: gemm_epilogue.hpp inside the GEMM kernels, gemm_epilogue.hip as a pass over a product
constexpr float GELU_C0 = 0.797884560802865356f, GELU_C1 = 0.044715f;    // sqrt(2 / pi) and the cubic term of gelu's tanh form
enum { ACT_LINEAR = 0, ACT_SIGMOID = 1, ACT_ERF = 2 };                   // rowops.hpp
struct epilogue_args {
    mi355_gemm_epilogue p;
    float a, b, floor;
    int32_t kind, dtype_c;
    int32_t swapped;          // a kernel that calls its operands small and large: the small one is B
};
inline epilogue_args make_epilogue(const mi355_gemm_epilogue &ep, int32_t dtype_c)
{
    constexpr float LOG2E = 1.44269504088896340736f;
    epilogue_args e{};
    e.p = ep;
    e.dtype_c = dtype_c;
    e.floor = ep.activation == MI355_ACT_RELU ? 0.0f : -__builtin_inff();
    e.kind = ep.activation == MI355_ACT_SILU || ep.activation == MI355_ACT_GELU_TANH ? ACT_SIGMOID : ep.activation == MI355_ACT_GELU ? ACT_ERF : ACT_LINEAR;
    e.a = ep.activation == MI355_ACT_SILU ? -LOG2E : -2.0f * GELU_C0 * LOG2E;
    e.b = ep.activation == MI355_ACT_SILU ? 0.0f : -2.0f * GELU_C0 * GELU_C1 * LOG2E;
    return e;
}
inline bool has_parts(const epilogue_args &e)
{
    return e.p.bias || e.p.residual || e.p.pre || e.p.row_scale || e.p.col_scale || e.p.activation != MI355_ACT_NONE;
}
// the same for the part of the output that begins at (row, col)
inline epilogue_args epilogue_at(epilogue_args e, int64_t row, int64_t col)
{
    const int64_t ec = (int64_t)dtype_size(e.dtype_c);
    auto by = [](const void *p, int64_t bytes) { return p ? static_cast<const char *>(p) + bytes : nullptr; };
    if (e.p.bias) e.p.bias = by(e.p.bias, col * (int64_t)dtype_size(e.p.dtype_bias));
    e.p.residual = by(e.p.residual, (row * e.p.ld_residual + col) * ec);
    e.p.pre = const_cast<void *>(static_cast<const void *>(by(e.p.pre, (row * e.p.ld_pre + col) * ec)));
    if (e.p.row_scale) e.p.row_scale += row * e.p.inc_row_scale;
    if (e.p.col_scale) e.p.col_scale += col * e.p.inc_col_scale;
    return e;
}
// what mi355_gemm_fused refuses of an epilogue (linear_ops.cpp); `d` has been validated and is not empty
int32_t validate_epilogue(mi355_ctx *ctx, const mi355_gemm_desc &d, const mi355_gemm_epilogue &ep, const void *a, const void *b, const void *c);
// c = the epilogue of the sum of `slabs` f32 products, slab_stride elements apart, [batch][m][n] each, added in order
void launch_epilogue(hipStream_t s, const float *prod, uint32_t slabs, int64_t slab_stride, const epilogue_args &ep, void *c, int64_t batch, int64_t m,
                     int64_t n, int64_t ldc, int64_t stride_c);
struct fused_grad_args {
    const void *grad_out, *pre;
    void *grad_pre;
    float *partial;
    int64_t m, n, batch, slab;
    int64_t ld_out, ld_pre, ld_grad, stride_out, stride_pre, stride_grad;
};
void launch_fused_grad(hipStream_t s, int32_t dtype, int32_t activation, const fused_grad_args &a);

// ---- global_norm.hip
constexpr int64_t CHUNK = 16384;               // elements: 32 KiB of 16-bit, 64 KiB of f32 values
constexpr uint32_t GRID = 1024;                // workgroups of a launch at most
constexpr uint32_t MAX_PARTIALS = 4096;        // partial sums the workspace holds
constexpr int FLAT_MAX = 112, ROWS_MAX = 56;

struct flat_span {                             // one contiguous tensor
    const void *in;
    void *out;
    int64_t n;
    uint32_t first;                            // its first chunk in the launch's sequence
    int32_t dtype;
};
struct rows_span {                             // rows of `cols` elements; a chunk is `rows_per` of them
    const void *in;
    void *out;
    int64_t rows, cols, ld_in, ld_out;
    uint32_t first;
    int32_t dtype;
};
struct flat_table { uint32_t count, chunks; flat_span t[FLAT_MAX]; };
struct rows_table { uint32_t count, chunks; rows_span t[ROWS_MAX]; };
static_assert(sizeof(flat_table) <= 3840 && sizeof(rows_table) <= 3840, "the tables are kernel arguments");

#ifdef __HIPCC__
__host__ __device__
#endif
inline int64_t rows_per_chunk(int64_t cols) { return cols >= CHUNK ? 1 : CHUNK / cols; }

// one partial sum a workgroup; the norm from `count` of them; the tensors times min(1, max_norm / norm)
void launch_square_sums(hipStream_t s, const flat_table &t, uint32_t grid, double *partial);
void launch_square_sums(hipStream_t s, const rows_table &t, uint32_t grid, double *partial);
void launch_finish_norm(hipStream_t s, const double *partial, uint32_t count, float *out_norm);
void launch_scale(hipStream_t s, const flat_table &t, uint32_t grid, const double *partial, uint32_t count, float max_norm, float *out_norm);
void launch_scale(hipStream_t s, const rows_table &t, uint32_t grid, const double *partial, uint32_t count, float max_norm, float *out_norm);

}  // namespace mi355
