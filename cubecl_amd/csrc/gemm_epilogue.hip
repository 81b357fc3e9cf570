// gemm_epilogue.hip -- mi355_gemm_fused's epilogue as a pass of its own over an f32 product, and the epilogue's gradient.
//
//     z = rs[m] cs[n] (A B)[m][n] + bias[n]      c = act(z) + residual      grad_pre = grad_out act'(z)      grad_bias = sum over rows of it
//
// Both are HBM-bound passes: 4 bytes of product read and 2 (4) written per output, and 2 x 2 read + 2 written per element.  Kernels that run
// the epilogue on their accumulators (gemm_common.hpp, gemm_epilogue_args) do not come here.  Eight columns a thread, whole 16-byte accesses.
#include <algorithm>
#include <type_traits>

#include "rowops.hpp"

using namespace mi355;

namespace {

// one call for the activation the launch was made for: the switch is uniform, the eight elements go through straight-line code
__device__ __forceinline__ void act8(int32_t act, float (&z)[8])
{
#define ACT(A) case A: { _Pragma("unroll") for (int e = 0; e < 8; ++e) z[e] = act_of<A>(z[e]); } break
    switch (act) { ACT(MI355_ACT_RELU); ACT(MI355_ACT_GELU); ACT(MI355_ACT_GELU_TANH); ACT(MI355_ACT_SILU); default: break; }
#undef ACT
}

// grid.x: columns in 2048s, grid.y: rows, grid.z: batch
__global__ void __launch_bounds__(256)
epilogue_kernel(const float *__restrict__ prod, mi355_gemm_epilogue ep, void *c, int64_t m, int64_t n, int64_t batch, int64_t ldc,
                int64_t stride_c, int32_t dtype_c)
{
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) return;
    const int valid = (int)min((int64_t)8, n - i);
    for (int64_t b = blockIdx.z; b < batch; b += gridDim.z) {
        float bias[8], cs[8];
        if (ep.bias) load8_any(ep.bias, ep.dtype_bias, b * ep.stride_bias + i, valid, bias);
        if (ep.col_scale) {
#pragma unroll
            for (int e = 0; e < 8; ++e) cs[e] = e < valid ? ep.col_scale[b * ep.stride_col_scale + (i + e) * ep.inc_col_scale] : 0.0f;
        }
        for (int64_t row = blockIdx.y; row < m; row += gridDim.y) {
            const vec8<MI355_DTYPE_F32> p = load8<MI355_DTYPE_F32>(prod + (b * m + row) * n, i, valid);
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = get(p, e);
            if (ep.row_scale) {
                const float rs = ep.row_scale[b * ep.stride_row_scale + row * ep.inc_row_scale];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] *= rs;
            }
            if (ep.col_scale) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] *= cs[e];
            }
            if (ep.bias) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += bias[e];
            }
            if (ep.pre) store8_any(ep.pre, dtype_c, b * ep.stride_pre + row * ep.ld_pre + i, valid, z);
            act8(ep.activation, z);
            if (ep.residual) {
                float r[8];
                load8_any(ep.residual, dtype_c, b * ep.stride_residual + row * ep.ld_residual + i, valid, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += r[e];
            }
            store8_any(c, dtype_c, b * stride_c + row * ldc + i, valid, z);
        }
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------------
// A workgroup is 64 lanes x 8 columns wide and four rows (waves) deep; blockIdx.y walks slabs of `slab` rows, blockIdx.z the batch.  The
// column sums stay in registers over the slab, meet in LDS in wave order, and leave as one partial row.
template <int DT, int ACT>
__global__ void __launch_bounds__(256)
fused_grad_kernel(fused_grad_args a)
{
    __shared__ float part[3][64][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = ((int64_t)blockIdx.x * 64 + lane) * 8;
    const int valid = (int)min((int64_t)8, max((int64_t)0, a.n - i));
    const int64_t b = blockIdx.z, first = (int64_t)blockIdx.y * a.slab, last = min(a.m, first + a.slab);
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid > 0)
        for (int64_t row = first + wave; row < last; row += 4) {
            const vec8<DT> g = load8<DT>(a.grad_out, b * a.stride_out + row * a.ld_out + i, valid);
            float d[8];
            if constexpr (ACT == MI355_ACT_NONE) {
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = get(g, e);
            } else {
                const vec8<DT> z = load8<DT>(a.pre, b * a.stride_pre + row * a.ld_pre + i, valid);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = get(g, e) * act_grad_of<ACT>(get(z, e));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += d[e];
            if (a.grad_pre) store8<DT>(a.grad_pre, b * a.stride_grad + row * a.ld_grad + i, valid, d);
        }
    if (!a.partial) return;
    if (wave > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) part[wave - 1][lane][e] = sum[e];
    }
    __syncthreads();
    if (wave > 0 || valid <= 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += part[w][lane][e];
    store8<MI355_DTYPE_F32>(a.partial + (b * gridDim.y + blockIdx.y) * a.n, i, valid, sum);
}

template <int DT>
void launch_grad(hipStream_t s, int32_t activation, const fused_grad_args &a)
{
    const dim3 grid((uint32_t)((a.n + 511) / 512), (uint32_t)((a.m + a.slab - 1) / a.slab), (uint32_t)a.batch);
#define GRAD(A) hipLaunchKernelGGL((fused_grad_kernel<DT, A>), grid, dim3(256), 0, s, a)
    switch (activation) {
    case MI355_ACT_RELU: GRAD(MI355_ACT_RELU); break;
    case MI355_ACT_GELU: GRAD(MI355_ACT_GELU); break;
    case MI355_ACT_GELU_TANH: GRAD(MI355_ACT_GELU_TANH); break;
    case MI355_ACT_SILU: GRAD(MI355_ACT_SILU); break;
    default: GRAD(MI355_ACT_NONE); break;
    }
#undef GRAD
}

}  // namespace

namespace mi355 {

void launch_epilogue(hipStream_t s, const float *prod, const mi355_gemm_epilogue &ep, void *c, int64_t batch, int64_t m, int64_t n, int32_t dtype_c,
                     int64_t ldc, int64_t stride_c)
{
    const dim3 grid((uint32_t)((n + 2047) / 2048), (uint32_t)std::min<int64_t>(m, 65535), (uint32_t)std::min<int64_t>(batch, 1024));
    hipLaunchKernelGGL(epilogue_kernel, grid, dim3(256), 0, s, prod, ep, c, m, n, batch, ldc, stride_c, dtype_c);
}

void launch_fused_grad(hipStream_t s, int32_t dtype, int32_t activation, const fused_grad_args &a)
{
    if (dtype == MI355_DTYPE_F32) launch_grad<MI355_DTYPE_F32>(s, activation, a);
    else if (dtype == MI355_DTYPE_BF16) launch_grad<MI355_DTYPE_BF16>(s, activation, a);
    else launch_grad<MI355_DTYPE_F16>(s, activation, a);
}

}  // namespace mi355
