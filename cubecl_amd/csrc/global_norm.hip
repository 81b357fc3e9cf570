// global_norm.hip -- mi355_global_norm and mi355_clip_by_global_norm: sqrt(sum of x^2) over a list of tensors, and the list scaled by
// min(1, max_norm / norm).
//
// Roofline: HBM.  Clipping cannot start to write before the last element is read, so the list is read twice and written once (0.60 GB of bf16:
// 90 us of reading and 217 of copying at this card's rates; measured 123 and 214, 337 together, 370 in place).  Outputs are stored past the caches:
// 360 -> 334 us, since the second reading finds more of the list in the 256 MiB Infinity Cache.  (Walking the list backwards in the second pass:
// 334.0 / 335.1, not worth its code; 8 and 16 workgroups a CU instead of 4: 343 and 386.)
//   - The list travels in the kernel arguments (no device table to upload, nothing for a captured graph to find changed): up to FLAT_MAX
//     contiguous tensors or ROWS_MAX pitched ones a launch.
//   - A launch's tensors are cut into chunks of CHUNK elements, dealt to the workgroups in turn; a workgroup finds a chunk's tensor by
//     bisection over the table in its scalar registers' reach.
//   - Squares and sums are f64: v_fma_f64 runs at a rate the memory stream does not come near, and no f32 or bf16 element's square leaves the
//     range.  Every workgroup leaves one partial sum; the second pass's workgroups each add all partials again in the same order (16 KiB
//     from L2) instead of waiting for a third launch.  No atomics: the same bits from run to run.
#include <algorithm>

#include "rowops.hpp"

using namespace mi355;

namespace {

template <class TABLE>
__device__ __forceinline__ uint32_t find_span(const TABLE &tab, uint32_t chunk)
{
    uint32_t lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (tab.t[mid].first <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double *slot)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    return slot[0] + slot[1] + slot[2] + slot[3];
}

// Where a chunk's runs of eight elements lie: `count` runs, run r at element at(r) of the input and at_out(r) of the output, `len(r)` long.
struct chunk_place {
    const void *in;
    void *out;
    int64_t first_in, first_out, ld_in, ld_out, n;      // n: elements of a row from `first` on
    int32_t dtype, runs_row, count;                     // runs of a row (of the chunk, where it is one row's part)
    __device__ __forceinline__ void locate(int32_t r, int64_t &i, int64_t &o, int &valid) const
    {
        int32_t row = 0, q = r;
        if (count > runs_row) { row = r / runs_row; q = r - row * runs_row; }
        i = first_in + row * ld_in + (int64_t)q * 8;
        o = first_out + row * ld_out + (int64_t)q * 8;
        valid = (int)min((int64_t)8, n - (int64_t)q * 8);
    }
};
__device__ __forceinline__ chunk_place place_of(const flat_table &tab, uint32_t chunk)
{
    const flat_span &t = tab.t[find_span(tab, chunk)];
    const int64_t at = (int64_t)(chunk - t.first) * CHUNK, n = min(CHUNK, t.n - at);
    const int32_t runs = (int32_t)((n + 7) / 8);
    return {t.in, t.out, at, at, 0, 0, n, t.dtype, runs, runs};
}
__device__ __forceinline__ chunk_place place_of(const rows_table &tab, uint32_t chunk)
{
    const rows_span &t = tab.t[find_span(tab, chunk)];
    const uint32_t c = chunk - t.first;
    if (t.cols >= CHUNK) {                                   // a row is one chunk or several
        const int64_t per_row = (t.cols + CHUNK - 1) / CHUNK, row = c / per_row, at = (c - row * per_row) * CHUNK, n = min(CHUNK, t.cols - at);
        const int32_t runs = (int32_t)((n + 7) / 8);
        return {t.in, t.out, row * t.ld_in + at, row * t.ld_out + at, 0, 0, n, t.dtype, runs, runs};
    }
    const int64_t per = rows_per_chunk(t.cols), row = c * per, rows = min(per, t.rows - row);
    const int32_t runs = (int32_t)((t.cols + 7) / 8);        // (all of a chunk's runs fit 32 bits: at most CHUNK of them)
    return {t.in, t.out, row * t.ld_in, row * t.ld_out, t.ld_in, t.ld_out, t.cols, t.dtype, runs, (int32_t)rows * runs};
}

// Four runs of a thread at a time: all their loads are in flight before the first is used.  f(run of eight as f32, output element, valid)
template <int DT, class F>
__device__ __forceinline__ void each_run(const chunk_place &p, F f)
{
    for (int32_t r0 = threadIdx.x; r0 < p.count; r0 += 4 * 256) {
        vec8<DT> v[4];
        int64_t i, o[4];
        int valid[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            valid[u] = 0;
            if (r0 + u * 256 < p.count) {
                p.locate(r0 + u * 256, i, o[u], valid[u]);
                v[u] = load8<DT>(p.in, i, valid[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (valid[u] <= 0) continue;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = get(v[u], e);
            f(x, o[u], valid[u]);
        }
    }
}

template <class TABLE>
__global__ void __launch_bounds__(256)
square_sum_kernel(TABLE tab, double *__restrict__ partial)
{
    __shared__ double slot[4];
    double acc = 0.0;
    auto add = [&](const float (&x)[8], int64_t, int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = fma((double)x[e], (double)x[e], acc);
    };
    for (uint32_t chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
        const chunk_place p = place_of(tab, chunk);
        if (p.dtype == MI355_DTYPE_F32) each_run<MI355_DTYPE_F32>(p, add);
        else if (p.dtype == MI355_DTYPE_BF16) each_run<MI355_DTYPE_BF16>(p, add);
        else each_run<MI355_DTYPE_F16>(p, add);
    }
    acc = block_sum(acc, slot);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// the norm from the partial sums, the same in every workgroup
__device__ __forceinline__ double norm_of(const double *__restrict__ partial, uint32_t count, double *slot)
{
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += 256) acc += partial[i];
    return sqrt(block_sum(acc, slot));
}

__global__ void __launch_bounds__(256)
finish_norm_kernel(const double *__restrict__ partial, uint32_t count, float *__restrict__ out_norm)
{
    __shared__ double slot[4];
    const double norm = norm_of(partial, count, slot);
    if (threadIdx.x == 0) out_norm[0] = (float)norm;
}

template <class TABLE>
__global__ void __launch_bounds__(256)
scale_kernel(TABLE tab, const double *__restrict__ partial, uint32_t count, float max_norm, float *__restrict__ out_norm)
{
    __shared__ double slot[4];
    const double norm = norm_of(partial, count, slot);
    if (out_norm && blockIdx.x == 0 && threadIdx.x == 0) out_norm[0] = (float)norm;
    // (an infinite or NaN norm: no factor brings it to max_norm.)  A factor near the end of the f32 range, which a norm beyond that range asks for,
    // would have few bits left: `down` is a power of two, half of its exponent, and `coef` the rest.  What x * down loses there is 0 in the end.
    float coef = 1.0f, down = 1.0f;
    if (!(norm <= DBL_MAX)) coef = __uint_as_float(0x7FC00000u);
    else if (norm > (double)max_norm) {
        const double f = (double)max_norm / norm, half = f < 0x1p-100 ? ldexp(1.0, ilogb(f) / 2) : 1.0;
        down = (float)half;
        coef = (float)(f / half);
    }
    for (uint32_t k = blockIdx.x; k < tab.chunks; k += gridDim.x) {
        const chunk_place p = place_of(tab, k);
        if (coef == 1.0f && p.in == p.out) continue;              // in place and nothing to scale
        auto scale = [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            each_run<DT>(p, [&](float (&x)[8], int64_t o, int valid) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * down * coef;
                store8<DT, true>(p.out, o, valid, x);
            });
        };
        if (p.dtype == MI355_DTYPE_F32) scale(std::integral_constant<int, MI355_DTYPE_F32>{});
        else if (p.dtype == MI355_DTYPE_BF16) scale(std::integral_constant<int, MI355_DTYPE_BF16>{});
        else scale(std::integral_constant<int, MI355_DTYPE_F16>{});
    }
}

}  // namespace

namespace mi355 {

void launch_square_sums(hipStream_t s, const flat_table &t, uint32_t grid, double *partial)
{
    hipLaunchKernelGGL((square_sum_kernel<flat_table>), dim3(grid), dim3(256), 0, s, t, partial);
}
void launch_square_sums(hipStream_t s, const rows_table &t, uint32_t grid, double *partial)
{
    hipLaunchKernelGGL((square_sum_kernel<rows_table>), dim3(grid), dim3(256), 0, s, t, partial);
}
void launch_scale(hipStream_t s, const flat_table &t, uint32_t grid, const double *partial, uint32_t count, float max_norm, float *out_norm)
{
    hipLaunchKernelGGL((scale_kernel<flat_table>), dim3(grid), dim3(256), 0, s, t, partial, count, max_norm, out_norm);
}
void launch_scale(hipStream_t s, const rows_table &t, uint32_t grid, const double *partial, uint32_t count, float max_norm, float *out_norm)
{
    hipLaunchKernelGGL((scale_kernel<rows_table>), dim3(grid), dim3(256), 0, s, t, partial, count, max_norm, out_norm);
}
void launch_finish_norm(hipStream_t s, const double *partial, uint32_t count, float *out_norm)
{
    hipLaunchKernelGGL(finish_norm_kernel, dim3(1), dim3(256), 0, s, partial, count, out_norm);
}

}  // namespace mi355
