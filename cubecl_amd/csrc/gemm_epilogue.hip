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

template <bool WIDE>
__device__ __forceinline__ void act8(const epilogue_args &ep, float (&z)[8])
{
    if (ep.kind == ACT_SIGMOID) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = act_sigmoid<WIDE>(z[e], ep.a, ep.b);
    } else if (ep.kind == ACT_ERF) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = act_erf<WIDE>(z[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = act_linear(z[e], ep.floor);
    }
}

// One run of eight columns a thread, runs counted along the rows (grid.x), batch entries in grid.y; slabs in fours, so that four loads fly.
template <class INDEX>
__global__ void __launch_bounds__(256)
epilogue_kernel(const float *__restrict__ prod, uint32_t slabs, int64_t slab_stride, epilogue_args ep, void *c, INDEX runs, INDEX per_row, int64_t m, int64_t n,
                int64_t ldc, int64_t stride_c)
{
    const int64_t b = blockIdx.y;
    for (INDEX id = (INDEX)blockIdx.x * 256 + threadIdx.x; id < runs; id += (INDEX)gridDim.x * 256) {
        const INDEX q = id / per_row;
        const int64_t row = (int64_t)q, i = (int64_t)(id - q * per_row) * 8;
        const int valid = (int)min((int64_t)8, n - i);
        const float *p = prod + (b * m + row) * n;
        float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t s = 0;
        for (; s + 4 <= slabs; s += 4) {
            vec8<MI355_DTYPE_F32> t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = load8<MI355_DTYPE_F32>(p + (int64_t)(s + k) * slab_stride, i, valid);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] += get(t[k], e);
        }
        for (; s < slabs; ++s) {
            const vec8<MI355_DTYPE_F32> t = load8<MI355_DTYPE_F32>(p + (int64_t)s * slab_stride, i, valid);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += get(t, e);
        }
        float v[8];
        const float rs = ep.p.row_scale ? ep.p.row_scale[b * ep.p.stride_row_scale + row * ep.p.inc_row_scale] : 1.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e)      // (one after the other, as on the accumulators: the scales' product may leave the range where the value does not)
            z[e] = z[e] * rs * (ep.p.col_scale && e < valid ? ep.p.col_scale[b * ep.p.stride_col_scale + (i + e) * ep.p.inc_col_scale] : 1.0f);
        if (ep.p.bias) {
            load8_any(ep.p.bias, ep.p.dtype_bias, b * ep.p.stride_bias + i, valid, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += v[e];
        }
        if (ep.p.pre) store8_any(ep.p.pre, ep.dtype_c, b * ep.p.stride_pre + row * ep.p.ld_pre + i, valid, z);
        if (ep.dtype_c == MI355_DTYPE_F32) act8<true>(ep, z);
        else act8<false>(ep, z);
        if (ep.p.residual) {
            load8_any(ep.p.residual, ep.dtype_c, b * ep.p.stride_residual + row * ep.p.ld_residual + i, valid, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += v[e];
        }
        store8_any(c, ep.dtype_c, b * stride_c + row * ldc + i, valid, z);
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------------
// A workgroup is 64 lanes x 8 columns wide and four rows (waves) deep; blockIdx.y walks slabs of `slab` rows, blockIdx.z the batch.  The
// column sums stay in registers over the slab, meet in LDS in wave order, and leave as one partial row.  Measured: 4096 x 8192 bf16, gelu, 201 MB
// in 36 us (5.6 TB/s; 48 with operands that have left the caches, 4.2), f32 98, 512 x 1024 6.0 us with the fold (two launches' latency).
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
                for (int e = 0; e < 8; ++e) d[e] = get(g, e) * act_grad_of<ACT, DT == MI355_DTYPE_F32>(get(z, e));
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

void launch_epilogue(hipStream_t s, const float *prod, uint32_t slabs, int64_t slab_stride, const epilogue_args &ep, void *c, int64_t batch, int64_t m,
                     int64_t n, int64_t ldc, int64_t stride_c)
{
    const int64_t per_row = (n + 7) / 8, runs = m * per_row;
    const dim3 grid((uint32_t)std::min<int64_t>((runs + 255) / 256, std::max<int64_t>(1, (1 << 20) / batch)), (uint32_t)batch);
    if (runs < (1ll << 31)) hipLaunchKernelGGL((epilogue_kernel<uint32_t>), grid, dim3(256), 0, s, prod, slabs, slab_stride, ep, c, (uint32_t)runs, (uint32_t)per_row, m, n, ldc, stride_c);
    else hipLaunchKernelGGL((epilogue_kernel<uint64_t>), grid, dim3(256), 0, s, prod, slabs, slab_stride, ep, c, (uint64_t)runs, (uint64_t)per_row, m, n, ldc, stride_c);
}

void launch_fused_grad(hipStream_t s, int32_t dtype, int32_t activation, const fused_grad_args &a)
{
    if (dtype == MI355_DTYPE_F32) launch_grad<MI355_DTYPE_F32>(s, activation, a);
    else if (dtype == MI355_DTYPE_BF16) launch_grad<MI355_DTYPE_BF16>(s, activation, a);
    else launch_grad<MI355_DTYPE_F16>(s, activation, a);
}

}  // namespace mi355
