// rowops.hpp -- device helpers of the row-wise operators (gemm_epilogue.hip, rms_norm.hip, global_norm.hip): eight elements of any float type
// to and from f32, reductions over a wave and a workgroup, the activations and their derivatives.
#pragma once

#include <cfloat>

#include "gemm_common.hpp"
#include "linear_ops.hpp"

namespace mi355 {

// ---- eight consecutive elements ------------------------------------------------------------------------------------------------
// One row of a tensor may start at any element: the vectors below are declared with their element's alignment, which the gfx950 memory
// pipe serves with the same 16-byte access (it splits only where a cache line ends), so odd row lengths and offset views take this path too.
typedef uint32_t u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_e1 __attribute__((ext_vector_type(2), aligned(1)));

__device__ __forceinline__ float bf16_to_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float f16_to_f32(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

template <int DT> struct vec8;          // the raw registers of eight elements
template <> struct vec8<MI355_DTYPE_F32> { u32x4 lo, hi; };
template <> struct vec8<MI355_DTYPE_BF16> { u32x4 v; };
template <> struct vec8<MI355_DTYPE_F16> { u32x4 v; };

template <int DT> constexpr int elem_size() { return DT == MI355_DTYPE_F32 ? 4 : 2; }

// elements [i, i + 8) of `p`; where only `valid` < 8 of them exist the others read as zero
template <int DT>
__device__ __forceinline__ vec8<DT> load8(const void *p, int64_t i, int valid)
{
    vec8<DT> r;
    if constexpr (DT == MI355_DTYPE_F32) {
        const float *q = static_cast<const float *>(p) + i;
        if (valid >= 8) {
            r.lo = *reinterpret_cast<const u32x4_e4 *>(q);
            r.hi = *reinterpret_cast<const u32x4_e4 *>(q + 4);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r.lo[e] = e < valid ? __float_as_uint(q[e]) : 0u;
                r.hi[e] = e + 4 < valid ? __float_as_uint(q[e + 4]) : 0u;
            }
        }
    } else {
        const uint16_t *q = static_cast<const uint16_t *>(p) + i;
        if (valid >= 8) r.v = *reinterpret_cast<const u32x4_e2 *>(q);
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t lo = 2 * e < valid ? q[2 * e] : 0u, hi = 2 * e + 1 < valid ? q[2 * e + 1] : 0u;
                r.v[e] = lo | (hi << 16);
            }
        }
    }
    return r;
}

template <int DT>
__device__ __forceinline__ float get(const vec8<DT> &r, int e)      // e a compile-time constant after unrolling
{
    if constexpr (DT == MI355_DTYPE_F32) return __uint_as_float(e < 4 ? r.lo[e] : r.hi[e - 4]);
    else {
        const uint32_t w = r.v[e >> 1];
        if constexpr (DT == MI355_DTYPE_BF16) return __uint_as_float((e & 1) ? (w & 0xFFFF0000u) : (w << 16));
        else return f16_to_f32((uint16_t)((e & 1) ? (w >> 16) : (w & 0xFFFFu)));
    }
}

// NT: past the caches, for outputs larger than they are
template <int DT, bool NT = false>
__device__ __forceinline__ void store8(void *p, int64_t i, int valid, const float (&f)[8])
{
    if constexpr (DT == MI355_DTYPE_F32) {
        float *q = static_cast<float *>(p) + i;
        if (valid >= 8) {
            const u32x4_e4 lo = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
            const u32x4_e4 hi = {__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
            if constexpr (NT) {
                __builtin_nontemporal_store(lo, reinterpret_cast<u32x4_e4 *>(q));
                __builtin_nontemporal_store(hi, reinterpret_cast<u32x4_e4 *>(q + 4));
            } else {
                *reinterpret_cast<u32x4_e4 *>(q) = lo;
                *reinterpret_cast<u32x4_e4 *>(q + 4) = hi;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < valid) q[e] = f[e];
        }
    } else {
        uint16_t *q = static_cast<uint16_t *>(p) + i;
        if (valid >= 8) {
            const u32x4_e2 v = {f32x2_to_lp<DT>(f[0], f[1]), f32x2_to_lp<DT>(f[2], f[3]), f32x2_to_lp<DT>(f[4], f[5]), f32x2_to_lp<DT>(f[6], f[7])};
            if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_e2 *>(q));
            else *reinterpret_cast<u32x4_e2 *>(q) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < valid) q[e] = f32_to_lp<DT>(f[e]);
        }
    }
}

// the same with the type known at run time only (uniform over the launch)
__device__ __forceinline__ void load8_any(const void *p, int32_t dtype, int64_t i, int valid, float (&f)[8])
{
    if (dtype == MI355_DTYPE_F32) {
        const vec8<MI355_DTYPE_F32> r = load8<MI355_DTYPE_F32>(p, i, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = get(r, e);
    } else if (dtype == MI355_DTYPE_BF16) {
        const vec8<MI355_DTYPE_BF16> r = load8<MI355_DTYPE_BF16>(p, i, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = get(r, e);
    } else {
        const vec8<MI355_DTYPE_F16> r = load8<MI355_DTYPE_F16>(p, i, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = get(r, e);
    }
}
__device__ __forceinline__ void store8_any(void *p, int32_t dtype, int64_t i, int valid, const float (&f)[8])
{
    if (dtype == MI355_DTYPE_F32) store8<MI355_DTYPE_F32>(p, i, valid, f);
    else if (dtype == MI355_DTYPE_BF16) store8<MI355_DTYPE_BF16>(p, i, valid, f);
    else store8<MI355_DTYPE_F16>(p, i, valid, f);
}
__device__ __forceinline__ float load1_any(const void *p, int32_t dtype, int64_t i)
{
    if (dtype == MI355_DTYPE_F32) return static_cast<const float *>(p)[i];
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return dtype == MI355_DTYPE_BF16 ? bf16_to_f32(b) : f16_to_f32(b);
}
__device__ __forceinline__ void store1_any(void *p, int32_t dtype, int64_t i, float v)
{
    if (dtype == MI355_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = dtype == MI355_DTYPE_BF16 ? f32_to_bf16_rne(v) : f32_to_f16_rne(v);
}

// ---- reductions -------------------------------------------------------------------------------------------------------------------
// Over the 64 lanes: four DPP steps inside a row of 16 (no LDS traffic), two shuffles across the rows.  Every lane gets the result; the
// order is fixed, so a sum is the same bits from run to run.
template <class F, class T>
__device__ __forceinline__ T wave_reduce(T v, F f)
{
    static_assert(sizeof(T) == 4, "32-bit values");
    auto dpp = [](T x, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v = f(v, dpp(v, std::integral_constant<int, 0xB1>{}));     // quad_perm [1,0,3,2]: lane ^ 1
    v = f(v, dpp(v, std::integral_constant<int, 0x4E>{}));     // quad_perm [2,3,0,1]: lane ^ 2
    v = f(v, dpp(v, std::integral_constant<int, 0x141>{}));    // row_half_mirror: the other four of eight
    v = f(v, dpp(v, std::integral_constant<int, 0x140>{}));    // row_mirror: the other eight of sixteen
    v = f(v, __builtin_bit_cast(T, __shfl_xor(__builtin_bit_cast(int, v), 16, 64)));
    return f(v, __builtin_bit_cast(T, __shfl_xor(__builtin_bit_cast(int, v), 32, 64)));
}
struct sum_of { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
// maximum of magnitudes as bit patterns: an infinity is above every number, a NaN above the infinity
struct max_of { __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; } };

// Over T threads; `slot`: T / 64 words of LDS that nobody still reads.  T == 64: each wave by itself.
template <int T, class F, class V>
__device__ __forceinline__ V block_reduce(V v, V *slot, F f)
{
    v = wave_reduce(v, f);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) v = f(v, slot[w]);
    }
    return v;
}

// ---- activations --------------------------------------------------------------------------------------------------------------------
// Two forms.  For 16-bit outputs: exp through v_exp_f32 (2^x, 1 ulp) of the rounded product x * log2(e), which is off by |x| 2^-24 relative, and
// 1 / (1 + e) through v_rcp_f32 (1 ulp): below 2^-15 of the result wherever the type has a number for it.  WIDE, for f32 outputs: the exponent in
// two pieces, so that the tails keep their bits (2^-20 of the result; a single one is off by 2^-20 at z = -10, 2^-18 at -80).
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-x)); }
// z limited to [lo, hi]; a NaN stays
__device__ __forceinline__ float limit(float z, float lo, float hi) { return z < lo ? lo : (z > hi ? hi : z); }

// (Pieces of a product stay apart only while the compiler leaves the product alone: contraction is off where one is split.)
// 2^-(hi + lo), lo the few bits that hi has no room for; results below the normal numbers included
__device__ __forceinline__ float exp2_neg(float hi, float lo)
{
    asm("" : "+v"(hi));      // (rounded: exp2f adds 64 to what is below the normal numbers, and that sum would take hi's product in, and lo with it twice)
    const float e = exp2f(-hi);
    return __builtin_fmaf(e, lo * -0.693147182f, e);
}
// 1 / d, v_rcp_f32 and one Newton step: within 0.6 ulp for the d of [1, 8] met here
__device__ __forceinline__ float rcp_of(float d)
{
    const float r = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}
// |u| log2(e) of silu (u = z) and of gelu's tanh form (u = 2 C0 z (1 + C1 z^2)) in two pieces, for 0 <= w = |z| limited
struct exponent { float hi, lo; };
__device__ __forceinline__ exponent silu_exponent(float w)
{
#pragma clang fp contract(off)
    constexpr float L = 1.44269502f, L_LO = 1.92596303e-08f;       // log2(e)
    const float hi = w * L;
    return {hi, __builtin_fmaf(w, L_LO, __builtin_fmaf(w, L, -hi))};
}
__device__ __forceinline__ exponent gelu_tanh_exponent(float w)
{
#pragma clang fp contract(off)
    constexpr float A = 2.30220819f, A_LO = 1.29484024e-08f, B = 0.102943242f, B_LO = -2.01619832e-09f;      // 2 C0 log2(e) and its product with C1
    const float q = w * w, q_lo = __builtin_fmaf(w, w, -q);
    const float m = B * q, m_lo = __builtin_fmaf(B, q_lo, __builtin_fmaf(B_LO, q, __builtin_fmaf(B, q, -m)));
    const float s = A + m, part = s - A, s_lo = (A - (s - part)) + (m - part) + m_lo + A_LO;
    const float hi = w * s;
    return {hi, __builtin_fmaf(w, s_lo, __builtin_fmaf(w, s, -hi))};
}
// sigmoid(u) and 1 - sigmoid(u) from |u| log2(e), each with all its bits
struct sigmoid_pair { float s, c; };
__device__ __forceinline__ sigmoid_pair sigmoid_both(bool negative, exponent x)
{
    const float e = exp2_neg(x.hi, x.lo), r = rcp_of(1.0f + e), small_ = e * r;
    return negative ? sigmoid_pair{small_, r} : sigmoid_pair{r, small_};
}

// The normal distribution's upper tail Q(w) = erfc(w / sqrt 2) / 2, w >= 0, and exp(-w^2 / 2): Q = t (c0 + c1 t + ...) exp(-w^2 / 2) with
// t = 1 / (1 + p w).  The polynomials are fits of this file, minimax in the RELATIVE error over 0 <= w <= 14, beyond which both are 0: five powers
// 5.2e-6 (2^-17), eight 4.3e-8 (2.9e-7 with the rounding of its terms).  An absolute bound would not do: gelu multiplies the tail by z.
struct normal_tail { float q, e; };
template <bool WIDE>
__device__ __forceinline__ normal_tail tail_of(float w)
{
    if constexpr (WIDE) {
#pragma clang fp contract(off)
        constexpr float H = 0.721347511f, H_LO = 9.62981517e-09f;      // log2(e) / 2
        const float sq = w * w, sq_lo = __builtin_fmaf(w, w, -sq), hi = sq * H;
        const float e = exp2_neg(hi, __builtin_fmaf(sq_lo, H, __builtin_fmaf(sq, H_LO, __builtin_fmaf(sq, H, -hi))));
        const float t = rcp_of(__builtin_fmaf(0.353553385f, w, 1.0f));
        float p = -0.0295344628f;
        constexpr float C[] = {0.142287403f, -0.243599832f, 0.139033467f, -0.0133127607f, 0.101343408f, 0.121551886f, 0.141187653f, 0.141043201f};
#pragma unroll
        for (int i = 0; i < 8; ++i) p = __builtin_fmaf(p, t, C[i]);
        return {p * t * e, e};
    } else {
        const float e = __builtin_amdgcn_exp2f(w * w * -0.721347520444481704f);
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.311126977f, w, 1.0f));
        float p = -0.0730531216f;
        constexpr float C[] = {0.175327092f, 0.0203646068f, 0.131793693f, 0.121284626f, 0.12428052f};
#pragma unroll
        for (int i = 0; i < 5; ++i) p = __builtin_fmaf(p, t, C[i]);
        return {p * t * e, e};
    }
}

// Five activations in three forms, so that a kernel carries three pieces of code (their constants travel in epilogue_args):
//   linear    z, or 0 below `floor` (0: relu; -inf: none)
//   sigmoid   z sigmoid(z (p + q z^2)): silu, and gelu's tanh form, whose (1 + tanh u) / 2 is sigmoid(2 u); a, b = -p, -q times log2(e), b = 0: silu
//   erf       z Phi(z)
// At -inf the factor is 0 and the limit is 0: the multiplicand is kept finite (a NaN stays, or comes back through the factor), and so is the square
// (b may be 0).
__device__ __forceinline__ float act_linear(float z, float floor) { return z < floor ? 0.0f : z; }
template <bool WIDE>
__device__ __forceinline__ float act_sigmoid(float z, float a, float b)
{
    if constexpr (WIDE) {
        const float w = fabsf(z);
        const float f = sigmoid_both(z < 0.0f, b == 0.0f ? silu_exponent(fminf(w, 200.0f)) : gelu_tanh_exponent(fminf(w, 20.0f))).s;
        return (z < -FLT_MAX ? -FLT_MAX : z) * f;
    }
    return fmaxf(z, -FLT_MAX) * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * (a + b * fminf(z * z, 1e30f))));
}
template <bool WIDE>
__device__ __forceinline__ float act_erf(float z)
{
    const float q = tail_of<WIDE>(fminf(fabsf(z), 20.0f)).q;
    return (z < -FLT_MAX ? -FLT_MAX : z) * (z < 0.0f ? q : 1.0f - q);
}

// The derivative.  Beyond the limits it is 0 or 1 to the last bit of f32; inside them nothing overflows.
template <int ACT, bool WIDE>
__device__ __forceinline__ float act_grad_of(float z)
{
    constexpr float P = 2.0f * GELU_C0, P3 = 3.0f * GELU_C1;
    if constexpr (ACT == MI355_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    if constexpr (ACT == MI355_ACT_SILU) {
        z = limit(z, -120.0f, 120.0f);
        if constexpr (WIDE) {
            const sigmoid_pair f = sigmoid_both(z < 0.0f, silu_exponent(fminf(fabsf(z), 120.0f)));
            return f.s * (1.0f + z * f.c);
        }
        const float s = sigmoid_of(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if constexpr (ACT == MI355_ACT_GELU_TANH) {
        z = limit(z, -20.0f, 20.0f);
        if constexpr (WIDE) {
            const sigmoid_pair f = sigmoid_both(z < 0.0f, gelu_tanh_exponent(fminf(fabsf(z), 20.0f)));
            return f.s * (1.0f + z * f.c * (P * (1.0f + P3 * z * z)));
        }
        const float s = sigmoid_of(P * z * (1.0f + GELU_C1 * z * z));
        return s + z * s * (1.0f - s) * P * (1.0f + P3 * z * z);
    }
    if constexpr (ACT == MI355_ACT_GELU) {
        z = limit(z, -20.0f, 20.0f);
        const normal_tail t = tail_of<WIDE>(fminf(fabsf(z), 20.0f));
        return (z < 0.0f ? t.q : 1.0f - t.q) + z * t.e * 0.398942280401432678f;      // Phi(z) + z phi(z)
    }
    return 1.0f;
}

}  // namespace mi355
