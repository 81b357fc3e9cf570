// rms_norm.hip -- mi355_rms_norm and its gradient.
//
//     h = in + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w
//     grad_in = rstd (w g - x^ mean(w g x^)) + grad_hidden,  grad_w = sum over rows of g x^,   x^ = h rstd
//
// Roofline: HBM.  A row is read once into registers (f32 after the addition), reduced over its threads, and written once: in + residual +
// hidden + out bytes per element and nothing else; the weight comes out of L2.
//   - T threads hold a row, CH pieces of eight consecutive elements each: piece c of thread t is elements (c T + t) 8 .. + 7, so a wave's
//     16-byte accesses are one contiguous run.  T = 64: a wave by itself, four rows a workgroup, no barrier.
//     bf16: 8192 x 4096 29 us (134 MB: 4.6 TB/s), 16384 x 4096 with the addition and an e4m3 output in blocks of 32 85 us (470 MB, 5.5 TB/s),
//     8 x 4096 3.8 us, which is the latency of one load, one reduction and one store; the gradient of 8192 x 4096 43 us (201 MB, 4.7 TB/s, its fold included).
//   - rows longer than 16384 elements (what 1024 threads hold in two pieces) are walked in a loop and read again, from L2.
//   - 8-bit output: the scale needs the row's (block's) largest |y| first, which is in registers by then.  v_cvt_pk_fp8_f32 / _bf8_f32 round
//     to nearest even; the scale keeps every quotient at or below MAX (1 + 2^-22), which rounds to MAX, so nothing saturates.  A row is divided by
//     its scale (a product with the rounded reciprocal lands on the other side of a tie in one of 2^19 values), a block by a power of two.
//   - the gradient's workgroups walk several rows each and keep the weight's gradient in registers over them; one f32 partial row a workgroup
//     goes to the workspace, and fold_columns adds those in order.  No atomics: the same bits from run to run.
#include <algorithm>
#include <type_traits>

#include "rowops.hpp"

using namespace mi355;

namespace {

// eight f32 -> eight bytes of e4m3 / e5m2, nearest even
__device__ __forceinline__ u32x2 to_fp8(const float (&f)[8], bool e5m2)
{
    u32x2 r;
    if (e5m2) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            int v = __builtin_amdgcn_cvt_pk_bf8_f32(f[4 * w], f[4 * w + 1], 0, false);
            r[w] = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(f[4 * w + 2], f[4 * w + 3], v, true);
        }
    } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w], f[4 * w + 1], 0, false);
            r[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w + 2], f[4 * w + 3], v, true);
        }
    }
    return r;
}

__device__ __forceinline__ void store8_bytes(void *p, int64_t i, int valid, u32x2 v)
{
    uint8_t *q = static_cast<uint8_t *>(p) + i;
    if (valid >= 8) { *reinterpret_cast<u32x2_e1 *>(q) = v; return; }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < valid) q[e] = (uint8_t)(v[e >> 2] >> (8 * (e & 3)));
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// the row's scale from its largest magnitude (as bits): max / MAX, 1 for zeros, NaN for what is not finite.  Never below FLT_MIN, so its
// reciprocal is finite.
__device__ __forceinline__ float row_scale_of(uint32_t amax, bool e5m2)
{
    if (amax >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    if (amax == 0u) return 1.0f;
    return fmaxf(__uint_as_float(amax) / (e5m2 ? 57344.0f : 448.0f), FLT_MIN);
}
// f / s, the nearest f32: q = f (1 / s) and its remainder's share, f - q s being exact (P. Markstein, IBM J. Res. Dev. 34, 1990; the reciprocal is
// correctly rounded and serves the whole row).  16384 x 4096 by rows 104 us with divisions, 97.7 with the reciprocal alone, 98.5 with this.
// Remainders of rows below 2^-90 may underflow: those are divided.
struct row_quotient {
    float s, inv;
    __device__ __forceinline__ explicit row_quotient(float scale) : s(scale), inv(1.0f / scale) {}
    __device__ __forceinline__ void operator()(float (&f)[8]) const
    {
        if (s < 0x1p-90f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] /= s;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = f[e] * inv;
                f[e] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, f[e]), inv, q), f[e]);      // (a zero keeps its sign)
            }
        }
    }
};
// the block's ue8m0 byte: MAX = 1.75 * 2^8 (2^15), so max = 1.f * 2^(E - 127) needs 2^(E - 127 - 8), one more where f passes 1.75
__device__ __forceinline__ uint32_t block_scale_of(uint32_t amax, bool e5m2)
{
    if (amax >= 0x7F800000u) return 255u;
    if (amax == 0u) return 127u;
    const int e = (int)(amax >> 23) - (e5m2 ? 15 : 8) + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(e, 0);
}
__device__ __forceinline__ float inverse_of_ue8m0(uint32_t s)
{
    return s == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((254u - s) << 23);      // s <= 247: normal
}
// over the four lanes that hold a block's 32 elements
__device__ __forceinline__ uint32_t quad_max(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}

// rstd = by * scale: `by` for h * scale, kept apart because rstd itself may be subnormal where h^2 passed the f32 range
struct row_factor { float by, scale; };
__device__ __forceinline__ row_factor factor_of(float ss, float inv_cols, float eps) { return {rsqrtf(ss * inv_cols + eps), 1.0f}; }
constexpr float DOWN = 0x1p-80f;
__device__ __forceinline__ row_factor small_factor_of(float ss, float inv_cols, float eps) { return {rsqrtf(ss * inv_cols + (eps * DOWN) * DOWN), DOWN}; }

template <int DT, int MODE, int T, int CH>
__global__ void __launch_bounds__(T < 256 ? 256 : T)
rms_norm_kernel(norm_args a)
{
    constexpr int RPW = T == 64 ? 4 : 1;
    __shared__ float red[T > 64 ? 2 * (T / 64) : 1];
    __shared__ uint32_t redm[T > 64 ? T / 64 : 1];
    const int t = T == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const bool e5m2 = a.dtype_out == MI355_DTYPE_F8E5M2;
    int parity = 0;
    for (int64_t row = (int64_t)blockIdx.x * RPW + (T == 64 ? threadIdx.x >> 6 : 0); row < a.rows; row += (int64_t)gridDim.x * RPW, parity ^= 1) {
        const char *in = static_cast<const char *>(a.in) + row * a.ld_in * elem_size<DT>();
        vec8<DT> x[CH], r[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t i = ((int64_t)c * T + t) * 8;
            x[c] = load8<DT>(in, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)));
        }
        if (a.residual) {
            const char *res = static_cast<const char *>(a.residual) + row * a.ld_residual * elem_size<DT>();
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t i = ((int64_t)c * T + t) * 8;
                r[c] = load8<DT>(res, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)));
            }
        }
        float h[CH][8], ss = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[c][e] = get(x[c], e);
                if (a.residual) h[c][e] += get(r[c], e);
                ss += h[c][e] * h[c][e];
            }
        if (a.hidden) {
            char *hid = static_cast<char *>(a.hidden) + row * a.ld_hidden * elem_size<DT>();
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t i = ((int64_t)c * T + t) * 8;
                store8<DT>(hid, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)), h[c]);
            }
        }
        ss = block_reduce<T>(ss, red + (T > 64 ? parity * (T / 64) : 0), sum_of{});
        row_factor f = factor_of(ss, a.inv_cols, a.eps);
        if (!(ss < INFINITY)) {                                 // (uniform over the row's threads)
            if constexpr (T > 64) __syncthreads();              // the sums are read before their words are used again
            ss = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) { h[c][e] *= DOWN; ss += h[c][e] * h[c][e]; }
            ss = block_reduce<T>(ss, red + (T > 64 ? parity * (T / 64) : 0), sum_of{});
            f = small_factor_of(ss, a.inv_cols, a.eps);
        }
        if (a.rstd && t == 0) a.rstd[row] = f.by * f.scale;
        uint32_t amax = 0u;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t i = ((int64_t)c * T + t) * 8;
            const int valid = (int)min((int64_t)8, max((int64_t)0, a.cols - i));
            float w[8];
            if (a.weight) load8_any(a.weight, a.dtype_weight, i, valid, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[c][e] *= f.by;
                if (a.weight) h[c][e] = e < valid ? h[c][e] * w[e] : 0.0f;
                if constexpr (MODE == OUT_ROW) amax = max(amax, abs_bits(h[c][e]));
            }
            if constexpr (MODE == OUT_PLAIN)
                store8_any(a.out, a.dtype_out, row * a.ld_out + i, valid, h[c]);
            if constexpr (MODE == OUT_BLOCK) {
                uint32_t m = 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = max(m, abs_bits(h[c][e]));
                const uint32_t s = block_scale_of(quad_max(m), e5m2);
                const float inv = inverse_of_ue8m0(s);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] *= inv;
                store8_bytes(a.out, row * a.ld_out + i, valid, to_fp8(h[c], e5m2));
                if ((t & 3) == 0 && valid > 0) static_cast<uint8_t *>(a.scales)[row * a.ld_scales + (i >> 5)] = (uint8_t)s;
            }
        }
        if constexpr (MODE == OUT_ROW) {
            amax = block_reduce<T>(amax, redm, max_of{});
            const float s = row_scale_of(amax, e5m2);
            if (t == 0) static_cast<float *>(a.scales)[row] = s;
            const row_quotient by_scale(s);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t i = ((int64_t)c * T + t) * 8;
                by_scale(h[c]);
                store8_bytes(a.out, row * a.ld_out + i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)), to_fp8(h[c], e5m2));
            }
        }
    }
}

// rows longer than the registers of 1024 threads: the same steps, each a loop over the row (hidden is written last: it may be `in`)
template <int DT, int MODE>
__global__ void __launch_bounds__(1024)
rms_norm_long_kernel(norm_args a)
{
    constexpr int T = 1024;
    __shared__ float red[3][T / 64];
    __shared__ uint32_t redm[T / 64];
    const int t = threadIdx.x;
    const bool e5m2 = a.dtype_out == MI355_DTYPE_F8E5M2;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const char *in = static_cast<const char *>(a.in) + row * a.ld_in * elem_size<DT>();
        const char *res = a.residual ? static_cast<const char *>(a.residual) + row * a.ld_residual * elem_size<DT>() : nullptr;
        auto h_of = [&](int64_t i, int valid, float (&h)[8]) {
            const vec8<DT> x = load8<DT>(in, i, valid);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = get(x, e);
            if (res) {
                const vec8<DT> r = load8<DT>(res, i, valid);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] += get(r, e);
            }
        };
        auto sum_squares = [&](float scale, float *slot) {
            float ss = 0.0f;
            for (int64_t i = (int64_t)t * 8; i < a.cols; i += T * 8) {
                float h[8];
                h_of(i, (int)min((int64_t)8, a.cols - i), h);
#pragma unroll
                for (int e = 0; e < 8; ++e) { h[e] *= scale; ss += h[e] * h[e]; }
            }
            return block_reduce<T>(ss, slot, sum_of{});
        };
        float ss = sum_squares(1.0f, red[0]);
        row_factor f = factor_of(ss, a.inv_cols, a.eps);
        if (!(ss < INFINITY)) {
            ss = sum_squares(DOWN, red[1]);
            f = small_factor_of(ss, a.inv_cols, a.eps);
        }
        if (a.rstd && t == 0) a.rstd[row] = f.by * f.scale;
        auto y_of = [&](int64_t i, int valid, float (&y)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = y[e] * f.scale * f.by;
            if (a.weight) {
                float w[8];
                load8_any(a.weight, a.dtype_weight, i, valid, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = e < valid ? y[e] * w[e] : 0.0f;
            }
        };
        float scale = 1.0f;
        if constexpr (MODE == OUT_ROW) {
            uint32_t amax = 0u;
            for (int64_t i = (int64_t)t * 8; i < a.cols; i += T * 8) {
                const int valid = (int)min((int64_t)8, a.cols - i);
                float y[8];
                h_of(i, valid, y);
                y_of(i, valid, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = max(amax, abs_bits(y[e]));
            }
            amax = block_reduce<T>(amax, redm, max_of{});
            scale = row_scale_of(amax, e5m2);
            if (t == 0) static_cast<float *>(a.scales)[row] = scale;
        }
        const row_quotient by_scale(scale);
        // (block scales: a block's four lanes enter an iteration together -- cols is a multiple of 32 there)
        for (int64_t i = (int64_t)t * 8; i < a.cols; i += T * 8) {
            const int valid = (int)min((int64_t)8, a.cols - i);
            float y[8];
            h_of(i, valid, y);
            if (a.hidden) store8<DT>(static_cast<char *>(a.hidden) + row * a.ld_hidden * elem_size<DT>(), i, valid, y);
            y_of(i, valid, y);
            if constexpr (MODE == OUT_PLAIN) store8_any(a.out, a.dtype_out, row * a.ld_out + i, valid, y);
            else {
                if constexpr (MODE == OUT_BLOCK) {
                    uint32_t m = 0u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = max(m, abs_bits(y[e]));
                    const uint32_t s = block_scale_of(quad_max(m), e5m2);
                    const float inv = inverse_of_ue8m0(s);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] *= inv;
                    if ((t & 3) == 0) static_cast<uint8_t *>(a.scales)[row * a.ld_scales + (i >> 5)] = (uint8_t)s;
                }
                if constexpr (MODE == OUT_ROW) by_scale(y);
                store8_bytes(a.out, row * a.ld_out + i, valid, to_fp8(y, e5m2));
            }
        }
        __syncthreads();                                        // the LDS words are free for the next row
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------------
template <int DT, int T, int CH>
__global__ void __launch_bounds__(T < 256 ? 256 : T)
rms_norm_grad_kernel(norm_grad_args a)
{
    constexpr int RPW = T == 64 ? 4 : 1;
    __shared__ float red[T > 64 ? 2 * (T / 64) : 1];
    const int t = T == 64 ? (threadIdx.x & 63) : threadIdx.x;
    const int64_t lane_row = (int64_t)blockIdx.x * RPW + (T == 64 ? threadIdx.x >> 6 : 0);
    float w[CH][8], dw[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int64_t i = ((int64_t)c * T + t) * 8;
        if (a.weight) load8_any(a.weight, a.dtype_weight, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)), w[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!a.weight) w[c][e] = 1.0f;
            dw[c][e] = 0.0f;
        }
    }
    int parity = 0;
    for (int64_t row = lane_row; row < a.rows; row += (int64_t)gridDim.x * RPW, parity ^= 1) {
        const char *gp = static_cast<const char *>(a.grad_out) + row * a.ld_out * elem_size<DT>();
        const char *hp = static_cast<const char *>(a.hidden) + row * a.ld_hidden * elem_size<DT>();
        vec8<DT> g[CH], h[CH], s[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t i = ((int64_t)c * T + t) * 8;
            const int valid = (int)min((int64_t)8, max((int64_t)0, a.cols - i));
            g[c] = load8<DT>(gp, i, valid);
            h[c] = load8<DT>(hp, i, valid);
        }
        if (a.grad_hidden) {
            const char *sp = static_cast<const char *>(a.grad_hidden) + row * a.ld_stream * elem_size<DT>();
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t i = ((int64_t)c * T + t) * 8;
                s[c] = load8<DT>(sp, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)));
            }
        }
        const float rstd = a.rstd[row];
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gx = get(g[c], e) * (get(h[c], e) * rstd);
                dw[c][e] += gx;
                dot += w[c][e] * gx;
            }
        dot = block_reduce<T>(dot, red + (T > 64 ? parity * (T / 64) : 0), sum_of{}) * a.inv_cols;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t i = ((int64_t)c * T + t) * 8;
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                d[e] = rstd * (w[c][e] * get(g[c], e) - (get(h[c], e) * rstd) * dot);
                if (a.grad_hidden) d[e] += get(s[c], e);
            }
            store8<DT>(static_cast<char *>(a.grad_in) + row * a.ld_in * elem_size<DT>(), i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)), d);
        }
    }
    if constexpr (T == 64) {                                    // the four waves' rows meet before they leave
        __shared__ float meet[3][CH * 8][64];
        const int wave = threadIdx.x >> 6;
        if (wave > 0) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) meet[wave - 1][c * 8 + e][t] = dw[c][e];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w4 = 0; w4 < 3; ++w4)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) dw[c][e] += meet[w4][c * 8 + e][t];
    }
    if (a.partial) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t i = ((int64_t)c * T + t) * 8;
            store8<MI355_DTYPE_F32>(a.partial + (int64_t)blockIdx.x * a.cols, i, (int)min((int64_t)8, max((int64_t)0, a.cols - i)), dw[c]);
        }
    }
}

// rows longer than the registers: the row's dot product in one loop, its gradient in a second one
template <int DT>
__global__ void __launch_bounds__(1024)
rms_norm_grad_long_kernel(norm_grad_args a)
{
    constexpr int T = 1024;
    __shared__ float red[T / 64];
    const int t = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const char *gp = static_cast<const char *>(a.grad_out) + row * a.ld_out * elem_size<DT>();
        const char *hp = static_cast<const char *>(a.hidden) + row * a.ld_hidden * elem_size<DT>();
        const float rstd = a.rstd[row];
        float dot = 0.0f;
        for (int64_t i = (int64_t)t * 8; i < a.cols; i += T * 8) {
            const int valid = (int)min((int64_t)8, a.cols - i);
            const vec8<DT> g = load8<DT>(gp, i, valid), h = load8<DT>(hp, i, valid);
            float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
            if (a.weight) load8_any(a.weight, a.dtype_weight, i, valid, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += w[e] * (get(g, e) * (get(h, e) * rstd));
        }
        dot = block_reduce<T>(dot, red, sum_of{}) * a.inv_cols;
        for (int64_t i = (int64_t)t * 8; i < a.cols; i += T * 8) {
            const int valid = (int)min((int64_t)8, a.cols - i);
            const vec8<DT> g = load8<DT>(gp, i, valid), h = load8<DT>(hp, i, valid);
            float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, d[8];
            if (a.weight) load8_any(a.weight, a.dtype_weight, i, valid, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = rstd * (w[e] * get(g, e) - (get(h, e) * rstd) * dot);
            if (a.grad_hidden) {
                const vec8<DT> s = load8<DT>(static_cast<const char *>(a.grad_hidden) + row * a.ld_stream * elem_size<DT>(), i, valid);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] += get(s, e);
            }
            store8<DT>(static_cast<char *>(a.grad_in) + row * a.ld_in * elem_size<DT>(), i, valid, d);
        }
        __syncthreads();
    }
}

// ... and their weight gradient: each thread eight columns, blockIdx.y a slab of rows
template <int DT>
__global__ void __launch_bounds__(256)
rms_norm_grad_weight_long_kernel(norm_grad_args a)
{
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= a.cols) return;
    const int valid = (int)min((int64_t)8, a.cols - i);
    float dw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const vec8<DT> g = load8<DT>(static_cast<const char *>(a.grad_out) + row * a.ld_out * elem_size<DT>(), i, valid);
        const vec8<DT> h = load8<DT>(static_cast<const char *>(a.hidden) + row * a.ld_hidden * elem_size<DT>(), i, valid);
        const float rstd = a.rstd[row];
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[e] += get(g, e) * (get(h, e) * rstd);
    }
    store8<MI355_DTYPE_F32>(a.partial + (int64_t)blockIdx.y * a.cols, i, valid, dw);
}

}  // namespace

namespace {

// out[c] = partial[0][c] + partial[1][c] + ...: 64 columns x 16 slices of the partial rows a workgroup, slices in order, then across them
__global__ void __launch_bounds__(1024)
fold_columns_kernel(const float *__restrict__ partial, int64_t count, int64_t first_col, int64_t cols, void *__restrict__ out, int32_t dtype)
{
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, s = threadIdx.x >> 6;
    const int64_t c = first_col + (int64_t)blockIdx.x * FOLD_COLS + lane;
    const float *p = partial + (int64_t)blockIdx.y * count * cols + c;
    const int64_t per = (count + 15) / 16, first = s * per, last = min(count, first + per);
    float acc = 0.0f;
    if (c < cols) {
        int64_t r = first;
        for (; r + 8 <= last; r += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[(r + e) * cols];
#pragma unroll
            for (int e = 0; e < 8; ++e) acc += v[e];
        }
        for (; r < last; ++r) acc += p[r * cols];
    }
    part[s][lane] = acc;
    __syncthreads();
    if (s != 0 || c >= cols) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) acc += part[k][lane];
    store1_any(out, dtype, (int64_t)blockIdx.y * cols + c, acc);
}

}  // namespace

namespace mi355 {

// `batch` sums of `count` partial rows each, [batch][count][cols] -> out [batch][cols]
void launch_fold_columns(hipStream_t s, const float *partial, int64_t count, int64_t cols, int64_t batch, void *out, int32_t dtype)
{
    each_fold_launch(cols, batch, [&](int64_t c, int64_t wide, int64_t b, int64_t entries) {
        hipLaunchKernelGGL(fold_columns_kernel, dim3((uint32_t)wide, (uint32_t)entries), dim3(1024), 0, s, partial + b * count * cols, count, c, cols,
                           static_cast<char *>(out) + b * cols * (int64_t)dtype_size(dtype), dtype);
    });
}

}  // namespace mi355

namespace {

constexpr int64_t MAX_GRID = 1 << 20;            // rows beyond it are walked by the kernels' own loop

template <int DT, int MODE>
void launch_norm(hipStream_t s, const norm_args &a)
{
    const row_shape sh = shape_for(a.rows, a.cols);
    const int64_t wgs = sh.threads == 64 ? (a.rows + 3) / 4 : a.rows;
    const dim3 grid((uint32_t)std::min(wgs, MAX_GRID));
#define NORM(T, CH) else if (sh.threads == T && sh.pieces == CH) hipLaunchKernelGGL((rms_norm_kernel<DT, MODE, T, CH>), grid, dim3(T < 256 ? 256 : T), 0, s, a)
    if (sh.threads == 0) hipLaunchKernelGGL((rms_norm_long_kernel<DT, MODE>), grid, dim3(1024), 0, s, a);
    NORM(64, 1); NORM(64, 2); NORM(256, 1); NORM(256, 2); NORM(256, 4); NORM(1024, 1); NORM(1024, 2);
#undef NORM
}

template <int DT>
void launch_norm_grad(hipStream_t s, const norm_grad_args &a)
{
    const row_shape sh = grad_shape_for(a.rows, a.cols);
    if (sh.threads == 0) {
        // (the weight's gradient first: grad_in may be one of the operands it reads)
        if (a.partial)
            hipLaunchKernelGGL((rms_norm_grad_weight_long_kernel<DT>), dim3((uint32_t)((a.cols + 2047) / 2048), (uint32_t)norm_grad_slabs(a.rows, a.cols)), dim3(256), 0, s, a);
        hipLaunchKernelGGL((rms_norm_grad_long_kernel<DT>), dim3((uint32_t)std::min(a.rows, MAX_GRID)), dim3(1024), 0, s, a);
        return;
    }
    const dim3 grid((uint32_t)norm_grad_wgs(a.rows, sh));
#define GRAD(T, CH) else if (sh.threads == T && sh.pieces == CH) hipLaunchKernelGGL((rms_norm_grad_kernel<DT, T, CH>), grid, dim3(T < 256 ? 256 : T), 0, s, a)
    if (false) {}
    GRAD(64, 1); GRAD(64, 2); GRAD(256, 1); GRAD(256, 2); GRAD(256, 4); GRAD(512, 4); GRAD(1024, 1);
#undef GRAD
}

}  // namespace

namespace mi355 {

void launch_rms_norm(hipStream_t s, int32_t dtype, int mode, const norm_args &a)
{
#define MODES(DT)                                                      \
    do {                                                               \
        if (mode == OUT_PLAIN) launch_norm<DT, OUT_PLAIN>(s, a);        \
        else if (mode == OUT_ROW) launch_norm<DT, OUT_ROW>(s, a);       \
        else launch_norm<DT, OUT_BLOCK>(s, a);                          \
    } while (0)
    if (dtype == MI355_DTYPE_F32) MODES(MI355_DTYPE_F32);
    else if (dtype == MI355_DTYPE_BF16) MODES(MI355_DTYPE_BF16);
    else MODES(MI355_DTYPE_F16);
#undef MODES
}

void launch_rms_norm_grad(hipStream_t s, int32_t dtype, const norm_grad_args &a)
{
    if (dtype == MI355_DTYPE_F32) launch_norm_grad<MI355_DTYPE_F32>(s, a);
    else if (dtype == MI355_DTYPE_BF16) launch_norm_grad<MI355_DTYPE_BF16>(s, a);
    else launch_norm_grad<MI355_DTYPE_F16>(s, a);
}

}  // namespace mi355
