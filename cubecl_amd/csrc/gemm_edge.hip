// gemm_edge.hip -- the product of mi355_gemm_fused for operands that no other matrix-core kernel stages as they lie: a K that is no whole K-tile,
// rows that do not start on 16 bytes, an operand stored [K][M] beside one stored [N][K].
//
// The other kernels fetch by LDS-DMA, which wants whole aligned 16-byte pieces: mi355_gemm copies such operands into scratch first, zero-padded --
// one or two passes over each operand and up to four launches before the product starts, which is most of the time of a small product
// (333 x 1001 x 517 f32: 15 of 45 us).  Here a piece travels through registers: 16 bytes where they exist, at any alignment, single
// elements at the edges, zeros beyond them, and is turned into the tile's layout on its way into LDS.  So every layout, size and
// alignment is one launch, and the epilogue is in it.
//
// Tile: 2 x 2 waves of WT x WT outputs (WT = 32: 64 x 64 tiles, for few tiles; 64: 128 x 128), 128 bytes of K a step, two LDS stages; the pieces of
// step t + 1 are in flight during step t.  Matrix instructions v_mfma_f32_32x32x16_{bf16,f16} and v_mfma_f32_32x32x2_f32.  Bound: f32 the
// matrix pipe; 16-bit the LDS reads (a wave of 32 x 32 reads 4 KiB for 64 cycles of matrix work).
// Few tiles and a long K: K in slices, f32 slabs, the epilogue in their fold (launch_epilogue; slices added in order).
#include <algorithm>

#include "gemm_epilogue.hpp"

using namespace mi355;

namespace {

template <int DT> struct edge {                       // 16-bit
    typedef uint16_t elem;
    static constexpr int EPV = 8, BK = 64;            // elements of a 16-byte piece, k values of a step
};
template <> struct edge<MI355_DTYPE_F32> {
    typedef uint32_t elem;
    static constexpr int EPV = 4, BK = 32;
};

// 16 bytes at (row, col) of a [rows][cols] matrix, zeros beyond its edges
template <int DT>
__device__ __forceinline__ u32x4 piece_at(const typename edge<DT>::elem *p, int64_t ld, int64_t row, int64_t rows, int64_t col, int64_t cols)
{
    constexpr int EPV = edge<DT>::EPV;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (row >= rows || col >= cols) return v;
    const typename edge<DT>::elem *q = p + row * ld + col;
    if (col + EPV <= cols) {
        if constexpr (DT == MI355_DTYPE_F32) v = *reinterpret_cast<const u32x4_e4 *>(q);
        else v = *reinterpret_cast<const u32x4_e2 *>(q);
        return v;
    }
    const int left = (int)(cols - col);
    if constexpr (DT == MI355_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) v[e] = q[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) v[e >> 1] |= (uint32_t)q[e] << (16 * (e & 1));
    }
    return v;
}

// One operand's tile: R rows (of C or columns of C) x BK k values.  KC: it is stored with k contiguous.  In LDS
//   [row][k], 144 bytes a row          k contiguous, and 16-bit either way (two k rows of a transposed operand make whole words; the 16-byte
//                                      chunks of its rows are exchanged by row / 8, so that the eight octets of rows a wave writes at once
//                                      lie in different banks)
//   [k][row], 4 R + 16 bytes a k       f32 with the rows contiguous
template <int DT, int R, bool KC>
struct edge_tile {
    static constexpr int EPV = edge<DT>::EPV, BK = edge<DT>::BK, ESZ = 16 / EPV;
    static constexpr bool ROWS_IN = DT == MI355_DTYPE_F32 && !KC;
    static constexpr int PITCH = ROWS_IN ? 4 * R + 16 : 144;
    static constexpr int BYTES = ROWS_IN ? BK * PITCH : R * PITCH;
    static constexpr int N = R * 8 / 256;             // pieces a thread
    u32x4 v[N];

    static __device__ __forceinline__ int chunk(int row, int c) { return !KC && !ROWS_IN ? c ^ ((row >> 3) & 7) : c; }

    // step's pieces of the operand at p: element (row, k) at row * ld + k (KC) or k * ld + row
    __device__ __forceinline__ void fetch(const typename edge<DT>::elem *p, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t k_end)
    {
        const int t = threadIdx.x;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (KC) v[i] = piece_at<DT>(p, ld, row0 + (t >> 3) + 32 * i, rows, k0 + (t & 7) * EPV, k_end);
            else if constexpr (ROWS_IN) {
                const int q = t + 256 * i;             // R / 4 pieces a k row
                v[i] = piece_at<DT>(p, ld, k0 + q / (R / 4), k_end, row0 + (q % (R / 4)) * 4, rows);
            } else {                                   // pairs of k rows: thread -> (row octet, pair), pieces 2 j and 2 j + 1 its two rows
                const int q = t + 256 * (i >> 1);
                v[i] = piece_at<DT>(p, ld, k0 + 2 * (q / (R / 8)) + (i & 1), k_end, row0 + (q % (R / 8)) * 8, rows);
            }
        }
    }
    __device__ __forceinline__ void put(char *lds) const
    {
        const int t = threadIdx.x;
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4 *>(lds + ((t >> 3) + 32 * i) * PITCH + (t & 7) * 16) = v[i];
        } else if constexpr (ROWS_IN) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int q = t + 256 * i;
                *reinterpret_cast<u32x4 *>(lds + (q / (R / 4)) * PITCH + (q % (R / 4)) * 16) = v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const int q = t + 256 * j, pair = q / (R / 8), row = (q % (R / 8)) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t lo = v[2 * j][e >> 1], hi = v[2 * j + 1][e >> 1];
                    const uint32_t w = (e & 1) ? (lo >> 16) | (hi & 0xFFFF0000u) : (lo & 0xFFFFu) | (hi << 16);
                    *reinterpret_cast<uint32_t *>(lds + (row + e) * PITCH + chunk(row, pair >> 2) * 16 + (pair & 3) * 4) = w;
                }
            }
        }
    }
    // the fragment of row `row` for k-step s: 16-bit 8 values from k = 16 s + 8 h; f32 4 values from k = 8 s + 4 h
    static __device__ __forceinline__ u32x4 frag(const char *lds, int row, int s, int h)
    {
        if constexpr (ROWS_IN) {
            u32x4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const uint32_t *>(lds + (8 * s + 4 * h + j) * PITCH + row * 4);
            return r;
        } else return *reinterpret_cast<const u32x4 *>(lds + row * PITCH + chunk(row, 2 * s + h) * 16);
    }
};

template <int DT>
__device__ __forceinline__ f32x16 edge_mfma(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (DT == MI355_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    } else if constexpr (DT == MI355_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT, int DT_C, int WT, bool AKC, bool BKC, class ARGS>
__global__ void __launch_bounds__(256)
gemm_edge_kernel(ARGS g)
{
    constexpr int R = 2 * WT, F = WT / 32, BK = edge<DT>::BK;
    typedef typename edge<DT>::elem elem;
    typedef edge_tile<DT, R, AKC> TA;
    typedef edge_tile<DT, R, BKC> TB;
    constexpr int RS = WT * 4 + 16, BLOCK = 32 * RS;                      // a wave's 32 staged rows
    constexpr int STAGE = TA::BYTES + TB::BYTES;
    constexpr int LDS = 2 * STAGE > 4 * BLOCK ? 2 * STAGE : 4 * BLOCK;
    __shared__ __attribute__((aligned(16))) char smem[LDS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, h = lane >> 5, l31 = lane & 31;
    uint32_t tm, tn, batch_u;
    batched_tile_coords(g.tiles_m, g.tiles_n, g.group_m, tm, tn, batch_u);
    const int64_t batch = batch_u, m0 = (int64_t)tm * R, n0 = (int64_t)tn * R;
    const elem *A = static_cast<const elem *>(g.a) + batch * g.stride_a, *B = static_cast<const elem *>(g.b) + batch * g.stride_b;
    // K slice z of the launch: whole steps
    const int64_t steps = (g.k + BK - 1) / BK, per = (steps + g.split_k - 1) / g.split_k;
    const int64_t k_begin = (int64_t)blockIdx.z * per * BK, k_end = min(g.k, k_begin + per * BK);

    f32x16 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    TA ta;
    TB tb;
    if (k_begin < k_end) {
        ta.fetch(A, g.lda, m0, g.m, k_begin, k_end);
        tb.fetch(B, g.ldb, n0, g.n, k_begin, k_end);
        ta.put(smem);
        tb.put(smem + TA::BYTES);
    }
    __syncthreads();
    int cur = 0;
    for (int64_t k0 = k_begin; k0 < k_end; k0 += BK, cur ^= 1) {
        const bool more = k0 + BK < k_end;
        if (more) {
            ta.fetch(A, g.lda, m0, g.m, k0 + BK, k_end);
            tb.fetch(B, g.ldb, n0, g.n, k0 + BK, k_end);
        }
        const char *la = smem + cur * STAGE, *lb = la + TA::BYTES;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 fa[F], fb[F];
#pragma unroll
            for (int i = 0; i < F; ++i) {
                fa[i] = TA::frag(la, wm * WT + i * 32 + l31, s, h);
                fb[i] = TB::frag(lb, wn * WT + i * 32 + l31, s, h);
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = edge_mfma<DT>(fb[j], fa[i], acc[i][j]);      // lane: row l31, columns 8 q + 4 h .. + 3
        }
        if (more) {                                                       // the other stage: last read before the barrier of the step before
            char *st = smem + (cur ^ 1) * STAGE;
            ta.put(st);
            tb.put(st + TA::BYTES);
        }
        __syncthreads();
    }

    constexpr int LPR = WT / 8;
    gemm_args out = g;
    if (g.split_k > 1) out.c = static_cast<float *>(g.c) + (int64_t)blockIdx.z * g.split_c_stride;
    char *stage = smem + wave * BLOCK;
    char *wr = stage + l31 * RS + 4 * h * 4;
    const char *rd = stage + (lane / LPR) * RS + (lane % LPR) * 32;
    tile_finish<DT_C, LPR, false> fin(epilogue_of<ARGS>(), out, batch, m0 + wm * WT + lane / LPR, n0 + wn * WT + (lane % LPR) * 8, true);
    fin.template run<F>([&](auto ib) __attribute__((always_inline)) {
        constexpr int I = decltype(ib)::value;
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4 *>(wr + (j * 32 + 8 * q) * 4) = (f32x4){acc[I][j][4 * q + 0], acc[I][j][4 * q + 1], acc[I][j][4 * q + 2], acc[I][j][4 * q + 3]};
    }, rd, RS);
}

template <int DT, int DT_C, int WT>
void launch_layout(hipStream_t s, const mi355_gemm_desc &d, const with_epilogue<gemm_args> &g, dim3 grid)
{
    typedef with_epilogue<gemm_args> ARGS;
#define EDGE(A, B) hipLaunchKernelGGL((gemm_edge_kernel<DT, DT_C, WT, A, B, ARGS>), grid, dim3(256), 0, s, g)
    if (!d.trans_a) { if (d.trans_b) EDGE(true, true); else EDGE(true, false); }
    else { if (d.trans_b) EDGE(false, true); else EDGE(false, false); }
#undef EDGE
}

template <int DT, int DT_C>
void launch_tile(hipStream_t s, const mi355_gemm_desc &d, const with_epilogue<gemm_args> &g, dim3 grid, int wt)
{
    if (wt == 64) launch_layout<DT, DT_C, 64>(s, d, g, grid);
    else launch_layout<DT, DT_C, 32>(s, d, g, grid);
}

int64_t tiles_at(const mi355_gemm_desc &d, int64_t r) { return ((d.m + r - 1) / r) * ((d.n + r - 1) / r); }

}  // namespace

namespace mi355 {

bool gemm_edge_supports(const mi355_gemm_desc &d)
{
    if (d.dtype_ab != MI355_DTYPE_F32 && d.dtype_ab != MI355_DTYPE_BF16 && d.dtype_ab != MI355_DTYPE_F16) return false;
    return d.k > 0 && d.batch <= 65535 && tiles_at(d, 64) * d.batch < (1ll << 24);      // (a launch holds fewer than 2^32 threads)
}

int32_t launch_gemm_edge(mi355_ctx *ctx, hipStream_t s, const mi355_gemm_desc &d, const void *a, const void *b, void *c, const epilogue_args &ep)
{
    gemm_args g{};
    g.a = a; g.b = b; g.c = c;
    g.m = d.m; g.n = d.n; g.k = d.k;
    g.lda = d.lda; g.ldb = d.ldb; g.ldc = d.ldc;
    g.stride_a = d.stride_a; g.stride_b = d.stride_b; g.stride_c = d.stride_c;
    const int64_t cus = ctx->props.num_streaming_multiprocessors > 0 ? ctx->props.num_streaming_multiprocessors : 256;
    const int wt = tiles_at(d, 128) * d.batch >= cus ? 64 : 32;
    const int64_t r = 2 * wt, tiles = tiles_at(d, r) * d.batch, bk = d.dtype_ab == MI355_DTYPE_F32 ? 32 : 64, steps = (d.k + bk - 1) / bk;
    g.tiles_m = (uint32_t)((d.m + r - 1) / r);
    g.tiles_n = (uint32_t)((d.n + r - 1) / r);
    g.group_m = 8;
    g.split_k = 1;
    // K slices while the tiles leave CUs idle, four steps a slice at least: a step's latency (1.5-2 us, its pieces' way from memory through registers)
    // is what few tiles wait for.  us, eight steps a slice / four: f32 333 x 1001 x 517 20.0 / 18.2, 65 x 67 x 517 17.2 / 13.1, 30 x 2000 x 777 16.3 / 12.9,
    // bf16 333 x 517 x 1001 20.5 / 14.5, 100 x 100 x 5001 22.6 / 18.4; f32 1001 x 517 x 333 18.1 / 18.5 (a fold for six steps less).
    int64_t splits = 1;
    float *slabs = nullptr;
    if (tiles < cus && steps >= 8) {
        splits = std::min<int64_t>({2 * cus / tiles, steps / 4, 32});
        if (splits > 1) { const int64_t per = (steps + splits - 1) / splits; splits = (steps + per - 1) / per; }      // no empty slices
        if (splits > 1 && splitk_scratch(ctx, s, (size_t)(splits * d.batch * d.m * d.n) * sizeof(float), &slabs) != MI355_OK) splits = 1;
    }
    const dim3 grid(g.tiles_m * g.tiles_n, (uint32_t)d.batch, (uint32_t)splits);
    with_epilogue<gemm_args> w = add_epilogue(g, ep);
    if (splits > 1) {
        w.split_k = (uint32_t)splits;
        w.split_c_stride = d.batch * d.m * d.n;
        w.c = slabs; w.ldc = d.n; w.stride_c = d.m * d.n;
        mi355_gemm_epilogue none{};
        w.ep = make_epilogue(none, MI355_DTYPE_F32);
    }
    const bool f32c = splits > 1 || d.dtype_c == MI355_DTYPE_F32;
    if (d.dtype_ab == MI355_DTYPE_F32) launch_tile<MI355_DTYPE_F32, MI355_DTYPE_F32>(s, d, w, grid, wt);
    else if (d.dtype_ab == MI355_DTYPE_BF16) { if (f32c) launch_tile<MI355_DTYPE_BF16, MI355_DTYPE_F32>(s, d, w, grid, wt); else launch_tile<MI355_DTYPE_BF16, MI355_DTYPE_BF16>(s, d, w, grid, wt); }
    else { if (f32c) launch_tile<MI355_DTYPE_F16, MI355_DTYPE_F32>(s, d, w, grid, wt); else launch_tile<MI355_DTYPE_F16, MI355_DTYPE_F16>(s, d, w, grid, wt); }
    if (splits > 1) launch_epilogue(s, slabs, (uint32_t)splits, d.batch * d.m * d.n, ep, c, d.batch, d.m, d.n, d.ldc, d.stride_c);
    check_launch(ctx, "mi355_gemm_fused(edge)");
    return MI355_OK;
}

}  // namespace mi355
