// global_norm.hip -- mi355_global_norm and mi355_clip_by_global_norm: sqrt(sum of x^2) over a list of tensors, and the list scaled by
// min(1, max_norm / norm).
//
// Roofline: HBM.  Clipping cannot start to write before the last element is read, so the list is read twice and written once; what the first
// pass read last is still in the 256 MiB Infinity Cache when the second one starts, which therefore walks the list backwards.
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

// f(i, valid) for every run of eight elements of [0, n) this thread has; `f` gets a run of fewer at the end
template <class F>
__device__ __forceinline__ void each8(int64_t n, F f)
{
    for (int64_t i = (int64_t)threadIdx.x * 8; i < n; i += 256 * 8) f(i, (int)min((int64_t)8, n - i));
}

__device__ __forceinline__ double block_sum(double v, double *slot)
{
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    return slot[0] + slot[1] + slot[2] + slot[3];
}

// the elements of one chunk: runs (tensor, index, valid) in order
template <class F>
__device__ __forceinline__ void chunk_runs(const flat_table &tab, uint32_t chunk, F f)
{
    const flat_span &t = tab.t[find_span(tab, chunk)];
    const int64_t at = (int64_t)(chunk - t.first) * CHUNK;
    each8(min(CHUNK, t.n - at), [&](int64_t i, int valid) { f(t.in, t.out, t.dtype, at + i, at + i, valid); });
}
template <class F>
__device__ __forceinline__ void chunk_runs(const rows_table &tab, uint32_t chunk, F f)
{
    const rows_span &t = tab.t[find_span(tab, chunk)];
    const uint32_t c = chunk - t.first;
    if (t.cols >= CHUNK) {                                   // a row is one chunk or several
        const int64_t per_row = (t.cols + CHUNK - 1) / CHUNK, row = c / per_row, at = (c - row * per_row) * CHUNK;
        each8(min(CHUNK, t.cols - at), [&](int64_t i, int valid) { f(t.in, t.out, t.dtype, row * t.ld_in + at + i, row * t.ld_out + at + i, valid); });
    } else {
        const int64_t per = rows_per_chunk(t.cols), row0 = c * per, rows = min(per, t.rows - row0);
        const int32_t runs = (int32_t)((t.cols + 7) / 8);    // runs of eight in a row: their count a chunk fits 32 bits
        for (int32_t r = threadIdx.x; r < (int32_t)rows * runs; r += 256) {
            const int64_t row = row0 + r / runs, i = (int64_t)(r % runs) * 8;
            f(t.in, t.out, t.dtype, row * t.ld_in + i, row * t.ld_out + i, (int)min((int64_t)8, t.cols - i));
        }
    }
}

template <class TABLE>
__global__ void __launch_bounds__(256)
square_sum_kernel(TABLE tab, double *__restrict__ partial)
{
    __shared__ double slot[4];
    double acc = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x)
        chunk_runs(tab, chunk, [&](const void *in, void *, int32_t dtype, int64_t i, int64_t, int valid) {
            float x[8];
            load8_any(in, dtype, i, valid, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc = fma((double)x[e], (double)x[e], acc);
        });
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
    // (an infinite or NaN norm: no factor brings it to max_norm)
    const float coef = !(norm <= DBL_MAX) ? __uint_as_float(0x7FC00000u) : norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.0f;
    for (uint32_t k = blockIdx.x; k < tab.chunks; k += gridDim.x)
        chunk_runs(tab, tab.chunks - 1 - k, [&](const void *in, void *out, int32_t dtype, int64_t i, int64_t o, int valid) {
            float x[8];
            load8_any(in, dtype, i, valid, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= coef;
            store8_any(out, dtype, o, valid, x);
        });
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
