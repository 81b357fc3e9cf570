// gemm_epilogue.hpp -- the epilogue of mi355_gemm_fused on a GEMM kernel's f32 accumulators:
//     z = rs[m] cs[n] (A B)[m][n] + bias[n]      (pre = z)      c = act(z) + residual
//
// A kernel takes it as a wider argument block, with_epilogue<its arguments>; `has_epilogue` then compiles the plain stores out and one of the two
// forms below in, and the kernels without it are what they were.
//   finish_one    one output, for kernels that store by element (few rows, few columns, edges of everything)
//   tile_finish   a wave's block of 32 rows that has been staged through LDS in f32: eight columns a lane, so the bias and the column scales
//                 stay in registers over all rows, and everything leaves in whole 16-byte pieces.  AHEAD: the residual's pieces of a block are
//                 in flight while the block before it is worked on (one workgroup a CU: nothing else hides their latency); without it a piece
//                 is fetched when it is needed (several workgroups a CU, and a third of the registers)
#pragma once

#include <type_traits>
#include <utility>

#include "rowops.hpp"

namespace mi355 {

template <class BASE> struct with_epilogue : BASE { epilogue_args ep; };
template <class G> constexpr bool has_epilogue = false;
template <class B> constexpr bool has_epilogue<with_epilogue<B>> = true;
template <class BASE>
with_epilogue<BASE> add_epilogue(const BASE &g, const epilogue_args &ep)
{
    with_epilogue<BASE> w;
    static_cast<BASE &>(w) = g;
    w.ep = ep;
    return w;
}

// The epilogue of the kernel's only argument, read from the kernel argument segment from here on: the compiler may not fetch its two dozen
// scalars above the K loop, where they would be parked in vector lanes.
template <class ARGS>
__device__ __forceinline__ const epilogue_args &epilogue_of()
{
    typedef const __attribute__((address_space(4))) char *seg_ptr;
    seg_ptr p = (seg_ptr)__builtin_amdgcn_kernarg_segment_ptr();
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winvalid-offsetof"
    p += __builtin_offsetof(ARGS, ep);
#pragma clang diagnostic pop
    asm volatile("" : "+s"(p));
    return *(const epilogue_args *)(const char *)p;
}

template <bool WIDE>
__device__ __forceinline__ float activate(const epilogue_args &ep, float z)
{
    return ep.kind == ACT_SIGMOID ? act_sigmoid<WIDE>(z, ep.a, ep.b) : ep.kind == ACT_ERF ? act_erf<WIDE>(z) : act_linear(z, ep.floor);
}

// -> the value to store at (row, col) of batch entry b; `pre` is written here
__device__ __forceinline__ float finish_one(const epilogue_args &ep, int64_t b, int64_t row, int64_t col, float v)
{
    if (ep.p.row_scale) v *= ep.p.row_scale[b * ep.p.stride_row_scale + row * ep.p.inc_row_scale];
    if (ep.p.col_scale) v *= ep.p.col_scale[b * ep.p.stride_col_scale + col * ep.p.inc_col_scale];
    if (ep.p.bias) v += load1_any(ep.p.bias, ep.p.dtype_bias, b * ep.p.stride_bias + col);
    if (ep.p.pre) store1_any(ep.p.pre, ep.dtype_c, b * ep.p.stride_pre + row * ep.p.ld_pre + col, v);
    v = ep.dtype_c == MI355_DTYPE_F32 ? activate<true>(ep, v) : activate<false>(ep, v);
    if (ep.p.residual) v += load1_any(ep.p.residual, ep.dtype_c, b * ep.p.stride_residual + row * ep.p.ld_residual + col);
    return v;
}
// ... of a kernel that knows the output as (small operand's row, large operand's row)
__device__ __forceinline__ float finish_small_big(const epilogue_args &ep, int64_t b, int64_t small_, int64_t big, float v)
{
    return finish_one(ep, b, ep.swapped ? big : small_, ep.swapped ? small_ : big, v);
}

// LPR lanes a row (columns / 8), 32 rows a block
template <int DT_C, int LPR, bool AHEAD>
struct tile_finish {
    static constexpr int RPI = 64 / LPR, PIECES = 32 / RPI;      // rows a wave instruction covers, pieces of a lane
    const epilogue_args &ep;
    int64_t b, row, col, m, ldc, stride_c;
    char *c;
    int valid;
    float bias[8], cs[8];
    static constexpr bool WIDE = DT_C == MI355_DTYPE_F32;        // the activations' precision
    static constexpr bool BUFFERED = AHEAD && DT_C != MI355_DTYPE_F32;      // a second set of pieces (f32: the registers end)
    struct pieces { float rs[AHEAD ? PIECES : 1]; vec8<DT_C> res[AHEAD ? PIECES : 1]; } now, next;

    // the lane's first row and column of the wave's block; `live` false: a lane beyond the block's columns
    __device__ __forceinline__ tile_finish(const epilogue_args &e, const gemm_args &g, int64_t batch, int64_t row_, int64_t col_, bool live)
        : ep(e), b(batch), row(row_), col(col_), m(g.m), ldc(g.ldc), stride_c(g.stride_c), c(static_cast<char *>(g.c)),
          valid(live ? (int)max((int64_t)0, min((int64_t)8, g.n - col_)) : 0)
    {
        if (ep.p.bias) load8_any(ep.p.bias, ep.p.dtype_bias, b * ep.p.stride_bias + col, valid, bias);
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) {
            if (!ep.p.bias) bias[e8] = 0.0f;
            cs[e8] = ep.p.col_scale && e8 < valid ? ep.p.col_scale[b * ep.p.stride_col_scale + (col + e8) * ep.p.inc_col_scale] : 1.0f;
        }
    }
    // the residual and the row scales of the block that begins `at` rows further down
    __device__ __forceinline__ void fetch(int at)
    {
        if constexpr (AHEAD) {
#pragma unroll
            for (int it = 0; it < PIECES; ++it) fetch_piece(BUFFERED ? next : now, it, row + at + it * RPI);
        }
    }
    __device__ __forceinline__ void fetch_piece(pieces &p, int slot, int64_t r)
    {
        const bool in = r < m && valid > 0;
        p.rs[slot] = ep.p.row_scale && in ? ep.p.row_scale[b * ep.p.stride_row_scale + r * ep.p.inc_row_scale] : 1.0f;
        if (ep.p.residual && in) p.res[slot] = load8<DT_C>(ep.p.residual, b * ep.p.stride_residual + r * ep.p.ld_residual + col, valid);
    }
    template <int KIND>
    __device__ __forceinline__ void piece(const char *rd, int64_t r, int slot)
    {
        if (r >= m || valid <= 0) return;
        const f32x4 lo = *reinterpret_cast<const f32x4 *>(rd), hi = *reinterpret_cast<const f32x4 *>(rd + 16);
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = e < 4 ? lo[e & 3] : hi[e & 3];
        if (ep.p.row_scale) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] *= now.rs[slot];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = z[e] * cs[e] + bias[e];
        if (ep.p.pre) store8<DT_C, true>(ep.p.pre, b * ep.p.stride_pre + r * ep.p.ld_pre + col, valid, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            z[e] = KIND == ACT_SIGMOID ? act_sigmoid<WIDE>(z[e], ep.a, ep.b) : KIND == ACT_ERF ? act_erf<WIDE>(z[e]) : act_linear(z[e], ep.floor);
            if (ep.p.residual) z[e] += get(now.res[slot], e);
        }
        store8<DT_C, true>(c, b * stride_c + r * ldc + col, valid, z);
    }
    template <int KIND>
    __device__ __forceinline__ void rows(const char *rd, int pitch, int at)
    {
#pragma unroll 1
        for (int it = 0; it < PIECES; ++it) {
            fetch_piece(now, 0, row + at + it * RPI);
            piece<KIND>(rd + it * RPI * pitch, row + at + it * RPI, 0);
        }
    }
    // AHEAD: GROUP pieces of the block through each step together, so that one piece's LDS reads and exponentials hide another's; INSIDE: every
    // row is one.  (Eight at once do not fit the registers beside 256 accumulators; 1 / 4: up projection of 4096 x 8192 x 2048, gelu and kept
    // pre-activation, 138.8 / 133.8 us, 8-bit 1777 x 4096 x 4096 58.8 / 55.2.)
    static constexpr int GROUP = DT_C == MI355_DTYPE_F32 ? 1 : PIECES < 4 ? PIECES : 4;
    template <int KIND>
    static __device__ __forceinline__ void act_all(float (&z)[GROUP][8], float a, float b, float floor)
    {
#pragma unroll
        for (int it = 0; it < GROUP; ++it)
#pragma unroll
            for (int e = 0; e < 8; ++e) z[it][e] = KIND == ACT_SIGMOID ? act_sigmoid<WIDE>(z[it][e], a, b) : KIND == ACT_ERF ? act_erf<WIDE>(z[it][e]) : act_linear(z[it][e], floor);
    }
    template <bool INSIDE>
    __device__ __forceinline__ void store_all(void *p, int64_t at_, int64_t ld, int64_t r0, const float (&z)[GROUP][8])
    {
#pragma unroll
        for (int it = 0; it < GROUP; ++it)
            if (INSIDE || r0 + it * RPI < m) store8<DT_C, true>(p, at_ + it * RPI * ld, INSIDE ? 8 : valid, z[it]);
    }
    template <bool INSIDE>
    __device__ __forceinline__ void together(const char *rd, int pitch, int at, const float *rs, const vec8<DT_C> *res)
    {
        float z[GROUP][8];
#pragma unroll
        for (int it = 0; it < GROUP; ++it) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(rd + it * RPI * pitch), hi = *reinterpret_cast<const f32x4 *>(rd + it * RPI * pitch + 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[it][e] = e < 4 ? lo[e & 3] : hi[e & 3];
        }
        if (valid > 0) {
            const int64_t r0 = row + at;
            if (ep.p.row_scale) {
#pragma unroll
                for (int it = 0; it < GROUP; ++it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[it][e] *= rs[it];
            }
            if (ep.p.col_scale) {
#pragma unroll
                for (int it = 0; it < GROUP; ++it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[it][e] = z[it][e] * cs[e] + bias[e];
            } else if (ep.p.bias) {
#pragma unroll
                for (int it = 0; it < GROUP; ++it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[it][e] += bias[e];
            }
            if (ep.p.pre) store_all<INSIDE>(ep.p.pre, b * ep.p.stride_pre + r0 * ep.p.ld_pre + col, ep.p.ld_pre, r0, z);
            if (ep.kind == ACT_SIGMOID) act_all<ACT_SIGMOID>(z, ep.a, ep.b, 0.0f);
            else if (ep.kind == ACT_ERF) act_all<ACT_ERF>(z, 0.0f, 0.0f, 0.0f);
            else if (ep.floor == 0.0f) act_all<ACT_LINEAR>(z, 0.0f, 0.0f, 0.0f);
            if (ep.p.residual) {
#pragma unroll
                for (int it = 0; it < GROUP; ++it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[it][e] += get(res[it], e);
            }
            store_all<INSIDE>(c, b * stride_c + r0 * ldc + col, ldc, r0, z);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    // All NB blocks: stage(block, as a constant) puts a block's accumulators into LDS, rows `pitch` bytes apart; `rd`: the lane's eight columns of
    // its first row there.  From three blocks up the loop is a loop -- the accumulators are named by a branch over the block's number, kept apart
    // by the empty statements (merged, the branches would index the accumulators at run time: out of registers) -- so that the code behind the
    // staging, a few thousand instructions, is there once.
    template <int NB, class STAGE>
    __device__ __forceinline__ void run(STAGE stage, const char *rd, int pitch)
    {
        if constexpr (NB <= 2) {
            one<0>(stage, rd, pitch);
            if constexpr (NB == 2) one<1>(stage, rd, pitch);
        } else {
            if constexpr (BUFFERED) fetch(0);
#pragma unroll 1
            for (int i = 0; i < NB; ++i) {
                if constexpr (BUFFERED) {
                    now = next;
                    if (i + 1 < NB) fetch((i + 1) * 32);
                } else fetch(i * 32);
                stage_one(std::make_integer_sequence<int, NB>{}, i, stage);
                finish_block(rd, pitch, i);
            }
        }
    }
    template <int I, class STAGE>
    __device__ __forceinline__ void one(STAGE &stage, const char *rd, int pitch)
    {
        fetch(I * 32);
        if constexpr (BUFFERED) now = next;
        stage(std::integral_constant<int, I>{});
        finish_block(rd, pitch, I);
    }
    __device__ __forceinline__ void finish_block(const char *rd, int pitch, int i)
    {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // same-wave hand-over: the DS operations of one wave execute in order
        block(rd, pitch, i * 32);
        __builtin_amdgcn_sched_barrier(0);
    }
    template <int I, class STAGE>
    static __device__ __forceinline__ void stage_apart(STAGE &stage)
    {
        asm volatile("; block %0" ::"i"(I) : "memory");
        stage(std::integral_constant<int, I>{});
        asm volatile("; block %0 staged" ::"i"(I) : "memory");
    }
    template <int... I, class STAGE>
    static __device__ __forceinline__ void stage_one(std::integer_sequence<int, I...>, int i, STAGE &stage)
    {
        ((i == I ? stage_apart<I>(stage) : (void)0), ...);
    }
    // the block's rows, staged `pitch` bytes apart; `rd`: the lane's eight columns of its first row
    __device__ __forceinline__ void block(const char *rd, int pitch, int at)
    {
        if constexpr (AHEAD) {
            const bool inside = __all((valid == 8 || valid == 0) && row + at + (PIECES - 1) * RPI < m);
#pragma unroll
            for (int g = 0; g < PIECES; g += GROUP) {
                if (inside) together<true>(rd + g * RPI * pitch, pitch, at + g * RPI, now.rs + g, now.res + g);
                else together<false>(rd + g * RPI * pitch, pitch, at + g * RPI, now.rs + g, now.res + g);
            }
        } else if (ep.kind == ACT_SIGMOID) rows<ACT_SIGMOID>(rd, pitch, at);
        else if (ep.kind == ACT_ERF) rows<ACT_ERF>(rd, pitch, at);
        else rows<ACT_LINEAR>(rd, pitch, at);
    }
};

}  // namespace mi355
