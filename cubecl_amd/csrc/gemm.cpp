// gemm.cpp -- mi355_gemm: descriptor validation and kernel selection.
#include "gemm_common.hpp"
#include "linear_ops.hpp"

using namespace mi355;

namespace {

int32_t validate(mi355_ctx *ctx, const mi355_gemm_desc *d, const void *a, const void *b, const void *c)
{
    if (!d) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm: descriptor is NULL");
    if (d->m < 0 || d->n < 0 || d->k < 0 || d->batch < 0)
        return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm: negative dimension");
    const bool f8 = is_fp8(d->dtype_ab);
    if (d->dtype_ab != MI355_DTYPE_F32 && d->dtype_ab != MI355_DTYPE_BF16 && d->dtype_ab != MI355_DTYPE_F16 && !f8)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm: unsupported input dtype %d", d->dtype_ab);
    if (f8) {
        if (d->dtype_c != MI355_DTYPE_F32 && d->dtype_c != MI355_DTYPE_BF16 && d->dtype_c != MI355_DTYPE_F16)
            return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm: fp8 inputs write f32, bf16 or f16 (got %d)", d->dtype_c);
    } else if (d->dtype_c != MI355_DTYPE_F32 && d->dtype_c != d->dtype_ab)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm: output dtype %d must be f32 or the input dtype", d->dtype_c);
    if (d->m == 0 || d->n == 0 || d->batch == 0) return MI355_OK;
    if (!c || (d->k > 0 && (!a || !b))) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm: NULL operand");
    const int64_t a_min = d->trans_a ? d->m : d->k, b_min = d->trans_b ? d->k : d->n;
    if (d->lda < a_min || d->ldb < b_min || d->ldc < d->n)
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm: leading dimension smaller than the row (lda %lld ldb %lld ldc %lld)",
                    (long long)d->lda, (long long)d->ldb, (long long)d->ldc);
    if (d->stride_a < 0 || d->stride_b < 0 || d->stride_c < 0)
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm: negative batch stride");
    if (d->batch > 1 && d->stride_c < d->m * d->ldc - (d->ldc - d->n))
        return fail(ctx, MI355_E_UNSUPPORTED_STRIDES, "mi355_gemm: output batches overlap");
    return -1;  // proceed
}

// ---- the tile kernels' cost table (round 5) -------------------------------------------------------------------------------------
// For 16-bit operands with both extents past 128 the choice among the tile kernels is no longer a list of thresholds but the
// smallest predicted time
//     T_k = max( rounds x (K-tiles x c_k + f_k),     the workgroups' own pace: c_k us per K-tile, f_k us of prologue + epilogue + launch
//                padded FLOPs / P_k ),               the chip's pace at its power limit on uniform[-1,1) operands: P_k TFLOP/s
//     rounds = whole + (F0 + (1 - F0) x left / CUs when a last round of `left` tiles is partly filled; the idle CUs' power budget lets
//              the busy ones clock higher: F0 = 0.7, the constant of the tail-split planner below)
// with (c_k, f_k, P_k) FITTED to the committed interleaved A/B tables by tools/dev/tile_cost_model.py (`--emit` prints these rows;
// profiles/r05_tile_cost_model.txt: 400 timings of 97 shapes, median model error 2-10 % per kernel, the table's choice on average
// 0.7 % behind the measured best, one shape more than 10 %).  The 128x128 kernel's two co-resident workgroups share one CU's
// L2 -> LDS delivery: one slot per CU, two tiles deep.  Re-run the tool after a kernel changes; nothing here is tuned by hand.
struct tile_cost { int32_t algo; int tm, tn; double c_us, f_us, p_tflops; };
constexpr tile_cost TILE_COSTS[] = {
    // generated by tools/dev/tile_cost_model.py --emit from profiles/r03_tile_256x128_sweep.txt, r04_band_129_200_tiles_ab.txt,
    // r05_tile_256x192_ab.txt, r05_tile_192x192_ab.txt, r05_m16_ab.txt, r05_select_audit_cost_table_v1.txt
    {MI355_GEMM_ALGO_LP_128, 128, 128, 0.558, 1.84, 890.0},
    {MI355_GEMM_ALGO_LP_256X128, 256, 128, 0.873, 6.42, 1167.0},
    {MI355_GEMM_ALGO_LP_256W4, 256, 256, 1.313, 7.46, 1351.0},
    {MI355_GEMM_ALGO_LP_256X192, 256, 192, 1.043, 7.12, 1307.0},
    {MI355_GEMM_ALGO_LP_192X192, 192, 192, 0.829, 6.41, 1219.0},
    // (the 16x16x32 form of the square tile fits c = 1.369, f = 7.24, P = 1379: within box variance of the 32x32x16 row on one round --
    //  4096^3 measured 97.7 / 103.9, 107.8 / 108.2 and 110.3 / 105.0 us on three boxes -- so it is not a row; select_auto takes it from
    //  three rounds up, where the sustained clock decides)
};
// ... and the same kernels on a ROW-MAJOR [K][N] rhs (the layout `TensorHandle::new_contiguous` gives one): the 4-wave kernel's
// transposing-read image costs it next to nothing, the narrow tiles included (six 32-column blocks per block row); the 128-row kernels run
// it markedly slower (P 790 against 890, 1010 against 1167), which moves the crossovers -- hence rows of their own, fitted the same way.
constexpr tile_cost TILE_COSTS_ROW_MAJOR_B[] = {
    // generated by tools/dev/tile_cost_model.py --nn --emit from profiles/r05_tile_nn_ab.txt (23 shapes; the table's choice is the measured
    // best on every one).  Held out: profiles/r05_tile_nn_ab2.txt, 20 thin / multi-round / short-K shapes timed WITH this table in AUTO --
    // within 1 % of the best forced kernel on 17, 23664 x 352 x 14336 9 % behind (256 x 192 where 192^2 wins), and two outside the table's
    // domain (13096 x 128 x 512, 6144^2 x 1024); the seeded audit over 40 random shapes finds none behind (r05_random_audit_row_major_tables.txt)
    {MI355_GEMM_ALGO_LP_128, 128, 128, 0.623, 1.53, 790.0},
    {MI355_GEMM_ALGO_LP_256X128, 256, 128, 0.945, 6.95, 1010.0},
    // (late round 6: past the fit's K <= 8192 the square tile's chip pace is TILE_P_LONG_K_ROW_MAJOR_B, below)
    {MI355_GEMM_ALGO_LP_256W4, 256, 256, 1.237, 9.45, 1256.0},
    {MI355_GEMM_ALGO_LP_256X192, 256, 192, 1.014, 7.64, 1262.0},
    {MI355_GEMM_ALGO_LP_192X192, 192, 192, 0.827, 5.59, 1209.0},
};
constexpr double TILE_F0 = 0.7;
// The row-major table's fit saw no launch of the square tile past K = 8192 and its chip pace P = 1256 is 8 % low out there (the [N][K] table has
// 1351): 2320 x 5904 x 14336 went to the 192^2 tile at 396 us against 318, the seeded audit's one tile-family miss.  A refit with nine shapes at
// K = 12288 ... 16384 -- every one of them at most one round of the square tile -- (profiles/r06_long_k_tiles_nn_ab.txt; tools/dev/tile_cost_model.py
// --nn) gives 1363, c and f within 3 %.  Taken over for what the refit saw only: K-tile counts past the first fit's domain on at most one round.
// A partly filled second round runs at the first fit's 1256 at any K: 2368 x 9792 x 6144 256.3 us on the square tile = 1 225 TFLOP/s of padded
// work (227.0 on 256 x 192), 2240 x 10304 x 14336 575.9 (513.3), 4928 x 6976 x 14336 859.7 (750.5) -- with 1363 there the table took the square
// tile on all three (profiles/r06_random_audit_final2.txt, r06_random_audit_fresh_seeds.txt).  And only from seven eighths of a round (TILE_LONG_K_MIN_TILES):
// the pace of padded work follows the fill -- 240 / 256 tiles 1 418 / 1 440 TFLOP/s, 224 1 375, but 190 ... 200 tiles 1 272 ... 1 284 (4672 x 2368 x 14336: 278.7 us
// against 252.5 on 256 x 192, profiles/r06_random_audit_held_out_final.txt).
constexpr double TILE_P_LONG_K_ROW_MAJOR_B = 1363.0;
constexpr int64_t TILE_FIT_MAX_KTILES = 128, TILE_LONG_K_MIN_TILES = 224;
// the tail-split planner's cycle model against this table's microseconds: 4-8 % optimistic on the 15 shapes of profiles/
// r05_tail_split_vs_narrow_ab.txt; with this factor the table's choice is within 1 % of the measured best on all of them (was 6.6 % behind on one)
constexpr double TAIL_SPLIT_TABLE_BIAS = 1.06;
// the table's domain: both extents past TILE_MIN_EXTENT, K >= TILE_MIN_K up to one round of the square tile, K >= TILE_MIN_K_ROUNDS up to
// TILE_MAX_ROUNDS of it (further out the persistent forms, the tail split and the 16x16x32 kernel take over, all keyed to the square tile)
constexpr int64_t TILE_CUS = 256, TILE_MIN_EXTENT = 128, TILE_MIN_K = 512, TILE_MIN_K_ROUNDS = 512, TILE_MAX_ROUNDS = 3, NARROW_TILE_MIN_KTILES = 8,
                  NARROW_TILE_MIN_KTILES_ROUNDS = 8;

double tile_time_us(const tile_cost &t, const mi355_gemm_desc &d)
{
    const int64_t tiles = ((d.m + t.tm - 1) / t.tm) * ((d.n + t.tn - 1) / t.tn) * d.batch, nk = d.k / 64;
    const bool long_k_row_major_square = !d.trans_b && t.tm == 256 && t.tn == 256 && nk > TILE_FIT_MAX_KTILES && tiles >= TILE_LONG_K_MIN_TILES && tiles <= TILE_CUS;
    const double p_tflops = long_k_row_major_square ? TILE_P_LONG_K_ROW_MAJOR_B : t.p_tflops;
    const int64_t whole = tiles / TILE_CUS, left = tiles % TILE_CUS;
    const double rounds = (double)whole + (left ? TILE_F0 + (1.0 - TILE_F0) * (double)left / (double)TILE_CUS : 0.0);
    const double own = rounds * ((double)nk * t.c_us + t.f_us);
    const double chip = 2.0 * (double)tiles * t.tm * t.tn * (double)d.k / (p_tflops * 1e6);
    return std::max(own, chip);
}

// ---- f32 operands: the 128 x 128 f32 MFMA kernel (gemm_f32.hip) against the 256 x 256 tile of gemm_lp256w4.hip (late round 6) ----
// Until then one threshold chose (192 square tiles and more: the square tile).  The first seeded f32 audit (AUDIT_F32=1 tools/dev/random_audit.py, four seeds) found
// 61 of 768 cases more than 10 % behind, by up to 68 %: the square tile pays whole rounds and whole 256-wide tiles where the small one does not (4672 x 3968 x 4096:
// 304 square tiles = two rounds, 1 823 us against 1 441; 54048 x 112 x 4096 917 / 604; 96 x 57504 x 512 134 / 88).  Same model as the 16-bit tables, a K-tile = 32 values,
// and what a partly filled round costs (f0) fitted per kernel: the small kernel's rounds of 256 tiles cost a whole round however full (f0 = 1), the square tile's 0.95.
// Fitted by tools/dev/f32_tile_cost_model.py on the cases of six seeds where the two kernels are within 2 x of each other (196 + 189 of 576 + 531 timed with both), judged
// on every case of those and of four more seeds (383 + 350): median error 2.4 % / 1.1 %, mean regret 0.03 % / 0.06 %, no case more than 7 % behind (the threshold: 36 + 53
// and 23 + 28 more than 10 % behind; a first fit with f0 = 0.7 over every case: 21 of 768 on the device) -- profiles/r06_f32_tile_cost_model.txt.
// C2 (4096^3, one full round of square tiles: 932 us predicted, 912 measured; the small tile 1 180 / 1 174) stays on the square tile.
struct f32_tile_cost { int32_t algo; int tm, tn; double c_us, f_us, p_tflops, f0; };
constexpr f32_tile_cost F32_TILE_COSTS[] = {
    {MI355_GEMM_ALGO_F32_MFMA, 128, 128, 2.279, 3.48, 113.9, 1.00},
    {MI355_GEMM_ALGO_LP_256W4, 256, 256, 7.171, 14.63, 147.6, 0.95},
};
constexpr f32_tile_cost F32_TILE_COSTS_ROW_MAJOR_B[] = {
    {MI355_GEMM_ALGO_F32_MFMA, 128, 128, 2.110, 3.74, 121.9, 1.00},
    {MI355_GEMM_ALGO_LP_256W4, 256, 256, 7.134, 15.22, 175.2, 0.96},
};
constexpr double F32_TAIL_SPLIT_OVER_PLAN = 0.77;        // measured AUTO (split) / forced (plain) over tail_split_ratio: 0.70 ... 0.83 on nine shapes x two layouts
double f32_tile_time_us(const f32_tile_cost &t, const mi355_gemm_desc &d)
{
    const int64_t tiles = ((d.m + t.tm - 1) / t.tm) * ((d.n + t.tn - 1) / t.tn) * d.batch, nk = (d.k + 31) / 32;
    const int64_t whole = tiles / TILE_CUS, left = tiles % TILE_CUS;
    const double rounds = (double)whole + (left ? t.f0 + (1.0 - t.f0) * (double)left / (double)TILE_CUS : 0.0);
    return std::max(rounds * ((double)nk * t.c_us + t.f_us), 2.0 * (double)tiles * t.tm * t.tn * (double)d.k / (t.p_tflops * 1e6));
}

// what the launcher's split of a small leftover round (plan_tail_split, below) makes of the square tile's time: planned cost / plain cost
// in that planner's own model, 1 where it plans nothing.  Only the square tile has the split; without this factor the table handed
// 1.1-round shapes with a long K to a narrow tile that the split form beats (cold, us, 256 x 192 or 192^2 / 256^2 split, profiles/
// r05_tail_split_vs_narrow_ab.txt: 4608 x 4096 x 8192 265.0 / 240.9, 4864 x 4096 x 8192 270.4 / 254.4, 4096 x 4352 x 8192 236.8 / 226.0; the other way
// at K <= 4096: 4352 x 4096 x 4096 122.8 / 130.9, 5120 x 4096 x 4096 146.2 / 153.2 -- the model calls all of them)
double tail_split_ratio(const mi355_gemm_desc &d);
bool qm_takes(const mi355_gemm_desc &d, const void *a, const void *b, const void *c);
bool qm_takes_tail_main(const mi355_gemm_desc &d, const void *a, const void *b, const void *c);
constexpr double QM_OVER_W4 = 0.92, QM_OVER_W4_ONE_TILE = 0.97, QM_OVER_W4_TAIL = 0.95;
bool m16_takes_f32_c(const mi355_gemm_desc &d, const void *a, const void *b, const void *c);
constexpr double M16_OVER_W4_F32_C = 0.94, NARROW_F32_C = 1.03;

inline int64_t tiles_256(const mi355_gemm_desc &d) { return ((d.m + 255) / 256) * ((d.n + 255) / 256) * d.batch; }

// the cheapest tile kernel of the table that takes the descriptor (0: none does)
int32_t pick_tile_kernel(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    int32_t best = 0;
    double best_us = 0.0;
    const tile_cost *rows = d.trans_b ? TILE_COSTS : TILE_COSTS_ROW_MAJOR_B;
    static_assert(sizeof(TILE_COSTS) == sizeof(TILE_COSTS_ROW_MAJOR_B), "one row per kernel in both tables");
    for (size_t r = 0; r < sizeof(TILE_COSTS) / sizeof(TILE_COSTS[0]); ++r) {
        const tile_cost &t = rows[r];
        bool ok = false;
        switch (t.algo) {
        case MI355_GEMM_ALGO_LP_128: ok = gemm_lp128_supports(d, a, b, c); break;
        case MI355_GEMM_ALGO_LP_256X128: ok = gemm_lp256x128_supports(d, a, b, c); break;
        case MI355_GEMM_ALGO_LP_256W4: ok = gemm_lp256w4_supports(d, a, b, c); break;
        // (short K on at most one round is launch-bound and outside the fit; over several rounds the model holds down to K = 512:
        //  11328 x 2944 x 512 predicted 49.1 / 45.5 us for 256^2 / 256 x 192, measured 51.6 / 44.7; 3648 x 5696 x 512 32.4 / 29.8, measured 33.2 / 29.8)
        default: ok = d.k / 64 >= (tiles_256(d) > TILE_CUS ? NARROW_TILE_MIN_KTILES_ROUNDS : NARROW_TILE_MIN_KTILES) && gemm_lp256x192_supports(d, a, b, c); break;
        }
        if (!ok) continue;
        double us = tile_time_us(t, d) * (t.algo == MI355_GEMM_ALGO_LP_256W4 ? tail_split_ratio(d) : 1.0);
        // the square tile's row was fitted on gemm_lp256w4.hip; where select_auto hands the tile to the persistent 16x16x32 kernel the
        // measured ratio of the two goes on top: 0.87 ... 0.93 [N][K], 0.89 ... 0.96 row-major from one full round up (profiles/
        // r06_qm_pre_shapes_ab.txt); 0.94 ... 0.98 where a workgroup has one tile and nothing to overlap (r06_qm_sub_round_ab.txt)
        // (row-major rhs, one tile per workgroup: 0.95 ... 0.99 -- no factor)
        if (t.algo == MI355_GEMM_ALGO_LP_256W4 && qm_takes(d, a, b, c)) us *= tiles_256(d) >= TILE_CUS ? QM_OVER_W4 : d.trans_b ? QM_OVER_W4_ONE_TILE : 1.0;
        // (... and where the tail split's main part runs on it: 0.92-0.94 at K = 8192 on six shapes, 0.956 at K = 4096: profiles/r06_tail_split_main_on_qm.txt,
        //  r06_tail_split_rule_ab.txt)
        else if (t.algo == MI355_GEMM_ALGO_LP_256W4 && qm_takes_tail_main(d, a, b, c)) us *= QM_OVER_W4_TAIL;
        // 16-bit operands with an f32 C (late round 6, the seeded audit with that output: profiles/r06_random_audit_c32.txt): the square tile is the 16x16x32 kernel's where
        // select_auto hands it over (measured 0.90 ... 0.98 of the 32x32x16 kernel, median 0.94); the narrow tiles' rows, fitted with a 16-bit C, + 3 % (smallest mean
        // regret of 1.00 ... 1.09 on the audit's 737 timed cases, replayed by tools/dev/replay_audit.py --c32)
        if (d.dtype_c == MI355_DTYPE_F32 && dtype_size(d.dtype_ab) == 2) {
            if (t.algo == MI355_GEMM_ALGO_LP_256W4) { if (m16_takes_f32_c(d, a, b, c)) us *= M16_OVER_W4_F32_C; }
            else if (t.algo != MI355_GEMM_ALGO_LP_128) us *= NARROW_F32_C;      // (a second term growing towards short K, 0.1 ... 0.3 x 8 / K-tiles: no gain on three audits' 2 205 timed cases)
        }
        if (!best || us < best_us) { best = t.algo; best_us = us; }
    }
    return best;
}

// ---- the dispatcher's measured thresholds, by name (round 5) -----------------------------------------------------------------------
// Every number `select` compares against lives here; the measurement behind each one is in profiles/dispatch_rules.md under the same
// name (what was timed, against what, on which shapes).  The tile kernels are not chosen by thresholds but by the cost tables above.
namespace rule {
constexpr int64_t CUS = 256;                             // the grid unit of every "round" below
// few rows or columns: which kernel streams the large operand
constexpr int64_t DOT_MAX_ROWS = 2;                      // gemm_skinny (dot products, no MFMA): always up to here
constexpr int64_t DOT_SHORT_GRID_MAX_ROWS = 4;           // ... and with 3-4 rows while the streaming kernel would launch fewer than
constexpr int64_t DOT_SHORT_GRID_WGS = 192;              //     this many workgroups
constexpr int64_t DOT_SHORT_GRID_LONG_K = 8192, DOT_SHORT_GRID_LONG_K_MIN_TILES = 16;   //     (not past this K on fewer than this many 128-wide tiles: split-K wins, round 6)
constexpr int64_t DOT_FALLBACK_MAX_ROWS = 16;            // ... and up to here where no MFMA kernel takes the descriptor
constexpr int64_t STREAM_MIN_ROWS = 3, STREAM_MAX_ROWS = 64, STREAM_ROWS_PER_WG = 32;      // gemm_stream64
constexpr int64_t STREAM_SMALL_OPERAND_BYTES = 1ll << 21;                                  // the small operand must stay in L2
// largest grid by row count (<= 16, <= 32, <= 64).  Late round 6 (the LM head of an LLM-shape audit, tools/dev/llm_audit.py: 16 x 128256 x 4096 was 18 % behind):
// up to 16 rows 2048 -> 4800, 17-32 rows 768 -> 2560 -- the largest grids of profiles/r06_stream_large_grids_ab.txt (72 shapes, K = 2048 ... 8192), on
// every one of which the streaming kernel is ahead of or level with split K: 4 x 100000 x 2048 63.1 us / 104.1, 16 x 128256 x 4096 163.9 / 197.1,
// 16 x 152064 x 4096 194.0 / 208.7 (the gap closes with N: no further), 20 x 57344 x 2048 40.4 / 54.4, 32 x 57344 x 8192 149.9 / 157.1, 32 x 80000 x 4096
// 120.8 / 124.3, 32 x 28672 x 4096 50.7 / 49.8 (level)
constexpr int64_t STREAM_WGS_16 = 4800, STREAM_WGS_32 = 2560, STREAM_WGS_32_ONE_ROUND = 768, STREAM_WGS_64 = 512;
constexpr int64_t STREAM_K_ALONE = 48;                   // K-tiles a workgroup walks alone on any grid (round 6: was 32)
constexpr int64_t STREAM_SHORT_K = 16, STREAM_SHORT_K_MAX_WGS = 1280;                      // ... but up to this many K-tiles only on grids up to this size
constexpr int64_t STREAM_K_MID = 64, STREAM_K_MID_WGS = 96;        // up to 32 rows: this many K-tiles from this many workgroups (few columns: any)
constexpr int64_t STREAM_K_LONG = 128, STREAM_K_LONG_WGS = 192;    // ... any K (few columns: up to this many K-tiles) from this many workgroups
constexpr int64_t STREAM_WIDE_WGS_MIN = 224, STREAM_WIDE_WGS_MAX = 288;                    // 33-64 rows, 65-128 K-tiles: about one workgroup per CU
constexpr int64_t STREAM_WIDE_LONG_K_MIN = 256, STREAM_WIDE_LONG_K_MAX = 512;              // ... and 256-512 K-tiles on at most one workgroup per CU (round 6)
constexpr int64_t STREAM_MID_ROWS = 32, STREAM_FEW_ROWS = 16;
// few rows on 257 ... 320 streaming workgroups: the second round, less than a quarter full, costs a whole one (one workgroup per CU) and the 128 x 128
// kernel's split K is ahead -- 33-64 rows from 32 K-tiles (47 x 8704 x 3072 22.9 us / 17.5, 64 x 9216 x 3072 25.7 / 19.3, 64 x 8704 x 2048 17.1 / 15.8),
// 17-32 rows from 64 (31 x 8704 x 4096 24.4 / 20.4, 24 x 9216 x 4096 24.5 / 20.9; at 48 K-tiles 24 rows tie and 31 lose 2 us); from 352 workgroups
// the streaming kernel is level or ahead except 64 rows at K = 3072 (26.6 / 23.1): profiles/r06_stream64_second_round_ab.txt (108 shapes, late round 6)
// few rows whose 128-column tiles leave a second round at most a quarter full (257 ... 320 tiles, N = 33k ... 41k): the streaming kernel from 32 K-tiles
// on, up to 48 rows (until late round 6: up to 32 rows from 64 K-tiles) -- streaming / split-K, us, profiles/r06_few_rows_part_round_ab.txt (100 shapes):
// 18 x 37312 x 2048 30.5 / 41.4, 34 x 35064 x 2048 34.8 / 42.9, 47 x 38624 x 2048 37.6 / 43.3, 34 x 37312 x 8192 113.2 / 145.0, 47 x 33024 x 8192 123.3 / 138.0,
// 34 x 38624 x 4096 66.9 / 74.6; 49-64 rows: within 5 % either way except K = 2048 (61 rows 40.2 / 42.5); K = 1024: level
constexpr int64_t STREAM_PART_TILES_MAX = 320, STREAM_PART_TILES_MIN_K = 32, STREAM_PART_TILES_MAX_ROWS = 48;
// up to 16 COLUMNS (what was measured: 4 ... 16; 64 columns lose, 8192 x 64 x 14336 59.3 / 52.1) past STREAM_K_LONG K-tiles, up to K = 16384: streams from 192 workgroups on, except on a second round less than a quarter full
// (late round 6, profiles/r06_fresh_seed_fixes_ab.txt, streaming / split-K: 19152 x 6 x 14336 100.7 us / 120.2, 32768 x 6 x 14336 136.2 / 173.3,
// 19152 x 16 x 14336 102.7 / 114.3, 19152 x 8 x 16384 110.3 / 125.5, 6872 x 4 x 14336 39.2 / 43.9; 291 workgroups: 9312 x 4 ... 24 x 14336 57.8 ... 69.8 /
// 53 ... 55; half a round: 4096 x 6 x 14336 34.4 / 29.8)
constexpr int64_t STREAM_COLS_K_MAX = 256;
constexpr int64_t STREAM_PART_ROUND_MAX_WGS = 320, STREAM_PART_ROUND_MIN_K_WIDE = 32, STREAM_PART_ROUND_MIN_K_MID = 64;
constexpr int64_t PART_ROUND_MAX_TILES = 448;            // a second round of 128-column tiles filled by less than three quarters
// f32 operands
constexpr int64_t SHORT_K_FEW_COLS_F32_C_MIN_EXTENT = 16384;   // one or two K-tiles, few columns, f32 C: the 128 x 128 kernel only from here along the long side
constexpr int64_t SQUARE_MIN_TILES_F32_C = 176;          // SQUARE_MIN_TILES with an f32 C (16-bit operands)
constexpr int64_t M16_F32_C_MIN_TILES = 176;             // 16-bit operands, f32 C: the 16x16x32 one-tile kernel for the square tile from here (none audited below)
constexpr int64_t F32_DOT_MAX_ROWS = 8, F32_STREAM_MIN_ROWS = 5;   // FMA kernel below / streaming kernel's f32 form from here
constexpr int64_t F32_STRIP_MAX_ROWS = 16, F32_STRIP_MIN_WEIGHT = 1ll << 15;               // row-major weight: gemm_nnrows f32 form (2^16 until the f32 audit: 4 x 768 x 64 7.3 us on the tile / 4.3)
constexpr int64_t F32_STREAM_SHORT_K = 128, F32_SHORT_K_LONG = 16384, F32_STREAM_SHORT_K_LONG = 24576;   // K <= 64 / K <= 128 against a streamed side this long: the 128 x 128 f32 tile
// fp8 operands
constexpr int64_t FP8_SQUARE_MIN_WORK = 1ll << 21;       // m n k
constexpr int64_t FP8_SQUARE_MIN_K = 1024;               // the square tile from eight 128-value K-tiles
constexpr int64_t FP8_SQUARE_LONG_K = 4096, FP8_SQUARE_LONG_K_MIN_TILES = 96;   // ... and past this many tiles from this K
// row-major B, few rows: the strip kernel (gemm_nnrows) / what stays native / what is re-laid out
constexpr int64_t STRIP_MIN_WEIGHT = 1ll << 25;          // n k elements worth streaming
constexpr int64_t STRIP_WHOLE_COLUMNS = 256;             // with more than one row, N must be whole strips of this many columns
constexpr int64_t STRIP_NARROW_ROWS = 8, STRIP_NARROW_MAX_N = 16384;
constexpr int64_t STRIP_MAX_ROWS = 16, STRIP_WIDE_MIN_N = 8192, STRIP_WIDE_MAX_N = 16384, STRIP_HUGE_N = 65536;
// up to four rows, whole strips or not, where the 128 x 128 kernel is weakest: 129 ... 192 column tiles (no K split, a quarter to a half of the CUs idle)
// or a mostly empty second round (late round 6, profiles/r06_fresh_seed_fixes_ab.txt: 2 x 19584 x 3072 23.1 us / 28.6, 4 x 20472 x 14336 106.0 / 124.4,
// 3 x 34672 x 1536 24.5 / 28.6; outside the band the ragged strip kernel is level or behind: 4 x 14920 x 8192 48.0 / 45.4, 4 x 30000 x 4096 48.9 / 43.5)
constexpr int64_t STRIP_RAGGED_MAX_ROWS = 4, STRIP_RAGGED_MIN_TILES = 128, STRIP_RAGGED_MAX_TILES = 192;
constexpr int64_t NATIVE_NN_MID_MIN_EXTENT = 64;         // the 128 x 128 kernel stages a row-major B natively past this extent
constexpr int64_t FEW_COLUMNS_TILE_MAX_N = 16, FEW_COLUMNS_TILE_MAX_K = 4096;              // few columns of a row-major B: no re-layout pass
// tile family outside the cost tables
constexpr int64_t SQUARE_MIN_TILES = 128;                // 256 x 256 tiles above this many of them, the 128 x 128 kernel up to it
constexpr int64_t THIN_MAX_EXTENT = 128;                 // an extent up to here never takes a 256-wide tile on that side
constexpr int64_t THIN_192_MIN_EXTENT = 65;              // ... but 65-128 rows (columns) take the 192 x 192 tile where the 128 x 128 kernel would
constexpr int64_t THIN_192_MIN_K = 512, THIN_192_MAX_K = 1024;                             //     split a short K over a half-empty chip:
constexpr int64_t THIN_192_ROWS_MIN_TILES = 128, THIN_192_COLS_MIN_TILES = 56, THIN_192_SPLIT_TILES = 132;   //     this many 128-wide tiles along the long side, below the count from which that kernel never splits,
constexpr int64_t THIN_192_COLS_LONG_K = 2048;            //     (few columns from THIN_192_ROWS_MIN_TILES tiles up: to this K)
constexpr int64_t THIN_192_PART_ROUND_MIN_K = 1024;      //     or (few rows) leave a second round of them less than three quarters full at this K or longer
constexpr int64_t SHORT_K_ANY = 192, SHORT_K_BOUNDED = 256, SHORT_K_BOUNDED_TILES = 1280;  // output-bound: single-stage 128 x 128 kernel
constexpr int64_t SHORT_K_ONE_ROUND = 128;               // ... on a single round of square tiles up to this K
constexpr int64_t SHORT_K_FEW_ROWS = 128, SHORT_K_FEW_ROWS_MIN_EXTENT = 6144, SHORT_K_ONE_KTILE_MIN_EXTENT = 4096;              // ... and with few rows or columns along a long side
constexpr int64_t TALL_TILE_MIN_K = 2560, TALL_TILE_THIN_EXTENT = 512;                     // the 256 x 128 tile: long K, or one thin side
// forms of the square tile (select_auto)
constexpr int64_t PERSISTENT_MAX_KTILES = 64;            // more than one round of tiles with K up to 4096: the persistent forms
constexpr int64_t DRIP_MIN_KTILES = 16, DRIP_SHORT_MIN_KTILES = 6, DRIP_SHORT_MAX_KTILES = 8;     // ... with dripped stores (16-bit C) at these K
constexpr int64_t M16_MIN_TILES = 768;                   // three rounds up: power-bound, the 16x16x32 form of the tile (and exactly one FULL round, round 6)
}  // namespace rule

inline int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }
inline int64_t tiles_of(const mi355_gemm_desc &d, int64_t tm, int64_t tn) { return cdiv(d.m, tm) * cdiv(d.n, tn) * d.batch; }

int32_t select(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, bool strip_kernel = true);

// fp8 / MX operands: the square tile from SQUARE_MIN_TILES up (as for bf16), the 128 x 128 kernel below
int32_t select_fp8(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    const bool big4 = gemm_lp256w4_supports(d, a, b, c), mid = gemm_lp128_supports(d, a, b, c);
    // (late round 6, the first seeded fp8 audit -- 27 of 384 [N][K] cases more than 10 % behind, every one the square tile where the 128 x 128 kernel is ahead: up to four
    //  128-value K-tiles the 128 x 128 kernel is level or ahead on all 35 shapes past 100 square tiles (2304 x 8000 x 128 10.7 us / 17.5, 10688 x 3136 x 256 19.9 / 29.1,
    //  8128 x 9024 x 512 50.7 / 59.2), from K = 1024 the square tile is (0.82 ... 0.93 there, 0.50 ... 0.89 from 2048); few rows or columns stay on the 128 x 128 kernel at
    //  any K (48424 x 64 x 1024 16.9 / 19.4, 40 x 62712 x 8192 x 1.07): profiles/r06_random_audit_fp8.txt)
    // (... and from K = 4096 already past 96 square tiles: 10184 x 680 x 12288, 120 tiles, 110.1 us / 128.1; 15096 x 280 x 8192, 118, 72.1 / 82.8; 31440 x 192 x 4096, 123, 49.5 / 55.7;
    //  level at 68 ... 90 tiles: r06_random_audit_fp8_unseen.txt)
    const int64_t min_tiles = d.k >= rule::FP8_SQUARE_LONG_K ? rule::FP8_SQUARE_LONG_K_MIN_TILES : rule::SQUARE_MIN_TILES;
    const bool square_pays = tiles_of(d, 256, 256) > min_tiles && d.k >= rule::FP8_SQUARE_MIN_K && std::min(d.m, d.n) > rule::THIN_MAX_EXTENT;
    if (big4 && (square_pays || !mid) && d.m * d.n * d.k >= rule::FP8_SQUARE_MIN_WORK) return MI355_GEMM_ALGO_LP_256W4;
    if (mid) return MI355_GEMM_ALGO_LP_128;
    return MI355_GEMM_ALGO_GENERIC;
}

// f32 operands (dispatch_rules.md "f32")
int32_t select_f32(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, bool strip_kernel)
{
    const int64_t rows = std::min(d.m, d.n);
    // (no grid / K bound like stream64_wins' for 16-bit operands: the advisor of round 5 asked for one; measured at the corners -- 2 ... 4 workgroups
    // walking K = 16384 ... 65536 alone, 1280 ... 4096 workgroups on K = 256 ... 1024, three and more rounds -- the streaming form is ahead of or
    // within 6 % of the 128 x 128 f32 tile on all 14: 64 x 64 x 65536 304 / 285 us, 64 x 128 x 16384 79 / 76, 16 x 64 x 32768 52 / 145,
    // 64 x 49152 x 2048 163 / 302, 16 x 131072 x 256 47 / 81: profiles/r06_f32_stream_corners_ab.txt)
    // (late round 6, the seeded f32 audit) ... except on a short K against a long streamed side, where each workgroup's 32 streamed rows are a few KiB and the grid is
    // thousands of workgroups: 27 x 18104 x 64 10.6 us against 7.9 on the 128 x 128 tile, 7 x 49648 x 64 20.4 / 12.1, 26512 x 20 x 64 14.3 / 10.0, 53 x 25000 x 128 21.2 / 14.8;
    // below the bounds the streaming form stays ahead (15 x 14168 x 64 5.7 / 7.9, 64 x 16072 x 128 8.7 / 14.5, 25 x 11016 x 128 7.4 / 12.4)
    const bool stream_takes = rows >= rule::F32_STREAM_MIN_ROWS && rows <= rule::STREAM_MAX_ROWS && gemm_stream64_supports(d, a, b, c);
    const bool short_k_long_side = d.k <= rule::F32_STREAM_SHORT_K && std::max(d.m, d.n) >= (d.k <= 64 ? rule::F32_SHORT_K_LONG : rule::F32_STREAM_SHORT_K_LONG);
    const bool streams = stream_takes && !short_k_long_side;
    if (rows <= rule::F32_DOT_MAX_ROWS && !stream_takes && gemm_skinny_supports(d, a, b, c)) return MI355_GEMM_ALGO_SKINNY;
    // (`strip_kernel` false: the capture-window fallback of mi355_gemm -- the strip kernel's scratch / tickets cannot be created while a
    // stream is capturing -- must reach the other kernels here as it does for 16-bit operands)
    const bool strip_short_k = d.k <= 64 && d.m > rule::F32_DOT_MAX_ROWS && d.n >= rule::F32_SHORT_K_LONG;   // 15 x 21712 x 64 12.9 us / 8.1 on the tile, 11 x 35840 x 64 17.6 / 12.2
    if (strip_kernel && !d.trans_a && !d.trans_b && d.m <= rule::F32_STRIP_MAX_ROWS && d.batch == 1 && d.n * d.k >= rule::F32_STRIP_MIN_WEIGHT && !strip_short_k &&
        gemm_nnrows_supports(d, a, b, c))
        return MI355_GEMM_ALGO_NNROWS;
    if (streams) return MI355_GEMM_ALGO_STREAM64;
    const bool square = gemm_lp256w4_supports(d, a, b, c), small = gemm_f32_mfma_supports(d, a, b, c);
    if (square && small) {                   // both tiles take it: the smaller predicted time (F32_TILE_COSTS)
        const f32_tile_cost *rows = d.trans_b ? F32_TILE_COSTS : F32_TILE_COSTS_ROW_MAJOR_B;
        // (the square tile's row is the plain launch; where the launcher splits a small leftover round -- plan_tail_split, AUTO only -- its planner's ratio
        //  goes on top, times what the nine split shapes of the audit measured over it: a leftover round of f32 tiles costs 0.95 of a whole one, not the 0.7
        //  the planner was calibrated with on power-limited 16-bit tiles, so the split saves more: planned 0.75 ... 0.89, measured 0.59 ... 0.77)
        const double split = tail_split_ratio(d);
        return f32_tile_time_us(rows[0], d) <= f32_tile_time_us(rows[1], d) * (split < 1.0 ? split * F32_TAIL_SPLIT_OVER_PLAN : 1.0) ? rows[0].algo : rows[1].algo;
    }
    if (square) return MI355_GEMM_ALGO_LP_256W4;
    if (small) return MI355_GEMM_ALGO_F32_MFMA;
    if (stream_takes) return MI355_GEMM_ALGO_STREAM64;
    return MI355_GEMM_ALGO_GENERIC;
}

// A stored [K][M] with a row-major B (lhs^T . grad_out, the weight-gradient product): the 128 x 128 and 256 x 256 kernels stage both natively
// -- taken exactly when that kernel would be chosen for the same shape with a K-contiguous A; where another kernel would win, A is
// transposed into scratch first (GENERIC = "re-lay out, then select again") and B stays as it is
int32_t select_transposed_lhs(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    if (d.trans_b) return MI355_GEMM_ALGO_GENERIC;
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    mi355_gemm_desc e = d;
    e.trans_a = 0; e.lda = d.k; e.stride_a = d.stride_a == 0 ? 0 : d.m * d.k;
    const int32_t twin = select(e, &aligned_dummy, b, c);             // what the same shape takes with a K-contiguous A
    const bool mid = gemm_lp128_supports(d, a, b, c), big4 = gemm_lp256w4_supports(d, a, b, c);
    // (late round 6, the first seeded audit of this layout -- 39 of 384 cases behind, by up to 3.2 x: where the twin takes a tile kernel that has no [K][M] form (the narrow
    //  tiles of the cost tables), A was transposed into scratch first; that pass moves 4 m k bytes and is never paid back by the better tile -- 42320 x 144 x 6144 400.9 us
    //  re-laid out + 192^2 against 126.6 native on the square tile, 37648 x 192 x 4096 241.0 / 84.6, 60544 x 696 x 6144 782.8 / 441.9, 744 x 5432 x 512 20.5 / 12.6 on the
    //  128 x 128 kernel.  Any tile kernel for the twin: the cheaper of the two native forms by the cost table's rows for them; profiles/r06_random_audit_ta.txt)
    const bool twin_is_tile = twin == MI355_GEMM_ALGO_LP_128 || twin == MI355_GEMM_ALGO_LP_256W4 || twin == MI355_GEMM_ALGO_LP_256X128 || twin == MI355_GEMM_ALGO_LP_256X192 ||
                              twin == MI355_GEMM_ALGO_LP_192X192;
    if (twin_is_tile && mid && big4) {
        if (twin == MI355_GEMM_ALGO_LP_128) return MI355_GEMM_ALGO_LP_128;
        if (twin == MI355_GEMM_ALGO_LP_256W4) return MI355_GEMM_ALGO_LP_256W4;
        const tile_cost *small = nullptr, *square = nullptr;
        for (const tile_cost &t : TILE_COSTS_ROW_MAJOR_B) { if (t.algo == MI355_GEMM_ALGO_LP_128) small = &t; if (t.algo == MI355_GEMM_ALGO_LP_256W4) square = &t; }
        return small && square && tile_time_us(*small, e) < tile_time_us(*square, e) ? MI355_GEMM_ALGO_LP_128 : MI355_GEMM_ALGO_LP_256W4;
    }
    if (twin_is_tile && mid) return MI355_GEMM_ALGO_LP_128;
    if (twin_is_tile && big4) return MI355_GEMM_ALGO_LP_256W4;
    // (the twin would have its small row-major operand re-laid out -- few columns: the 128 x 128 kernel takes the descriptor as it is: 10376 x 64 x 2048 22.0 us)
    if (twin == MI355_GEMM_ALGO_GENERIC && mid) return MI355_GEMM_ALGO_LP_128;
    return MI355_GEMM_ALGO_GENERIC;
}

// 16-bit operands, row-major B, one thin side (dispatch_rules.md "row-major rhs"): the strip kernel, the native tile forms, or the
// re-layout pass (GENERIC).  0: the general rules decide.
int32_t select_row_major_rhs(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, bool strip_kernel, bool big4, bool mid)
{
    const int64_t t128 = cdiv(d.n, 128);
    const bool second_round_part = t128 > rule::CUS && t128 < rule::PART_ROUND_MAX_TILES;
    if (strip_kernel && d.batch == 1 && d.n * d.k >= rule::STRIP_MIN_WEIGHT && (d.m == 1 || d.n % rule::STRIP_WHOLE_COLUMNS == 0) &&
        ((d.m <= rule::STRIP_NARROW_ROWS && (d.n <= rule::STRIP_NARROW_MAX_N || second_round_part)) || (d.m <= rule::STRIP_MAX_ROWS && d.n > rule::STRIP_HUGE_N) ||
         (d.m <= rule::STRIP_MAX_ROWS && d.n >= rule::STRIP_WIDE_MIN_N && d.n <= rule::STRIP_WIDE_MAX_N)) &&
        gemm_nnrows_supports(d, a, b, c))
        return MI355_GEMM_ALGO_NNROWS;
    if (strip_kernel && d.batch == 1 && d.n * d.k >= rule::STRIP_MIN_WEIGHT && d.m <= rule::STRIP_RAGGED_MAX_ROWS &&
        ((t128 > rule::STRIP_RAGGED_MIN_TILES && t128 <= rule::STRIP_RAGGED_MAX_TILES) || second_round_part) && gemm_nnrows_supports(d, a, b, c))
        return MI355_GEMM_ALGO_NNROWS;
    const int64_t thin = std::min(d.m, d.n);
    const bool native = (thin > rule::THIN_MAX_EXTENT && big4 && tiles_of(d, 256, 256) > rule::SQUARE_MIN_TILES) || (thin > rule::NATIVE_NN_MID_MIN_EXTENT && mid);
    if (native) return 0;
    if (mid && d.m <= d.n) return MI355_GEMM_ALGO_LP_128;
    if (mid) {       // few COLUMNS: the re-layout pass pays only where the K-contiguous twin would then leave the 128 x 128 kernel
        static const char aligned_dummy __attribute__((aligned(16))) = 0;
        mi355_gemm_desc e = d;
        e.trans_b = 1; e.ldb = d.k; e.stride_b = d.stride_b ? d.n * d.k : 0;
        if ((d.n <= rule::FEW_COLUMNS_TILE_MAX_N && d.k <= rule::FEW_COLUMNS_TILE_MAX_K) || select(e, a, &aligned_dummy, c, false) == MI355_GEMM_ALGO_LP_128)
            return MI355_GEMM_ALGO_LP_128;
    }
    return MI355_GEMM_ALGO_GENERIC;
}

// 16-bit K-contiguous operands, 3 ... 64 rows or columns: does gemm_stream64 take the launch?  (dispatch_rules.md "streaming kernel")
bool stream64_wins(const mi355_gemm_desc &d)
{
    const int64_t rows = std::min(d.m, d.n), wgs = cdiv(std::max(d.m, d.n), rule::STREAM_ROWS_PER_WG) * d.batch, nk = d.k / 64;
    if (rows * d.k * 2 > rule::STREAM_SMALL_OPERAND_BYTES) return false;
    const bool few_rows = d.m <= d.n, upto32 = rows <= rule::STREAM_MID_ROWS;
    const int64_t t128 = cdiv(std::max(d.m, d.n), 128) * d.batch;
    // any grid: few columns up to STREAM_K_MID K-tiles; few rows whose 128-column tiles would leave a second round mostly empty
    if (upto32 && !few_rows && nk <= rule::STREAM_K_MID) return true;
    if (upto32 && few_rows && t128 > rule::CUS && t128 < rule::PART_ROUND_MAX_TILES && nk >= rule::STREAM_K_MID) return true;
    if (few_rows && rows <= rule::STREAM_PART_TILES_MAX_ROWS && t128 > rule::CUS && t128 <= rule::STREAM_PART_TILES_MAX && nk >= rule::STREAM_PART_TILES_MIN_K) return true;
    // (17-32 rows: the larger limit only where the 128 x 128 kernel needs a second round of column tiles -- on one round it is level or ahead:
    //  32 x 28672 x 4096, 224 tiles, 41.7 us against 49.7 on one box, 49.8 / 50.7 on another)
    const int64_t max_wgs = rows <= rule::STREAM_FEW_ROWS ? rule::STREAM_WGS_16 : upto32 ? (t128 > rule::CUS ? rule::STREAM_WGS_32 : rule::STREAM_WGS_32_ONE_ROUND) : rule::STREAM_WGS_64;
    if (wgs > max_wgs) return false;
    if (nk <= rule::STREAM_SHORT_K && wgs > rule::STREAM_SHORT_K_MAX_WGS) return false;
    if (few_rows && rows > rule::STREAM_FEW_ROWS && wgs > rule::CUS && wgs <= rule::STREAM_PART_ROUND_MAX_WGS &&
        nk >= (upto32 ? rule::STREAM_PART_ROUND_MIN_K_MID : rule::STREAM_PART_ROUND_MIN_K_WIDE))
        return false;
    if (nk <= rule::STREAM_K_ALONE) return true;
    if (upto32)
        return (nk <= rule::STREAM_K_MID && (wgs >= rule::STREAM_K_MID_WGS || !few_rows)) || (wgs >= rule::STREAM_K_LONG_WGS && (few_rows || nk <= rule::STREAM_K_LONG)) ||
               (!few_rows && rows <= rule::STREAM_FEW_ROWS && nk <= rule::STREAM_COLS_K_MAX && wgs >= rule::STREAM_K_LONG_WGS && !(wgs > rule::CUS && wgs <= rule::STREAM_PART_ROUND_MAX_WGS));
    if (wgs >= rule::STREAM_WIDE_WGS_MIN && wgs <= rule::CUS && nk >= rule::STREAM_WIDE_LONG_K_MIN && nk <= rule::STREAM_WIDE_LONG_K_MAX) return true;
    return wgs >= rule::STREAM_WIDE_WGS_MIN && wgs <= rule::STREAM_WIDE_WGS_MAX && nk > rule::STREAM_K_MID && nk <= rule::STREAM_K_LONG;
}

int32_t select(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, bool strip_kernel)
{
    if (d.k == 0) return MI355_GEMM_ALGO_GENERIC;  // writes zeros
    if (is_fp8(d.dtype_ab)) return select_fp8(d, a, b, c);
    if (d.dtype_ab == MI355_DTYPE_F32) return select_f32(d, a, b, c, strip_kernel);
    if (d.trans_a) return select_transposed_lhs(d, a, b, c);
    // (MI355_GEMM_ALGO_LP_256, the retired 8-wave kernel's id, is an alias of the 4-wave kernel for callers that name it)
    const bool big4 = gemm_lp256w4_supports(d, a, b, c), mid = gemm_lp128_supports(d, a, b, c);
    if (!d.trans_b) {
        const int32_t pick = select_row_major_rhs(d, a, b, c, strip_kernel, big4, mid);
        if (pick) return pick;
    }
    const int64_t thin = std::min(d.m, d.n), tiles256 = tiles_of(d, 256, 256);
    // one or two K-tiles along a long side, however few rows or columns: the streaming kernels' per-workgroup cost is not paid back
    // (few COLUMNS with an f32 C: only from a much longer side -- 9168 x 18 x 64 5.4 us here / 3.8 streaming, 4576 x 37 x 64 5.4 / 3.7, 11536 x 18 x 128 6.7 / 4.7, 9296 x 4 x 128 6.2 / 3.8,
    //  level at 48032 x 31 x 64 and 57512 x 1 x 128; few rows are right as they are: 39 x 23752 x 64 5.6 / 7.4 -- profiles/r06_random_audit_c32_held_out.txt)
    const int64_t short_k_min_extent = d.dtype_c == MI355_DTYPE_F32 && d.n < d.m ? rule::SHORT_K_FEW_COLS_F32_C_MIN_EXTENT
                                       : d.k <= 64 ? rule::SHORT_K_ONE_KTILE_MIN_EXTENT : rule::SHORT_K_FEW_ROWS_MIN_EXTENT;
    if (mid && d.trans_b && d.k <= rule::SHORT_K_FEW_ROWS && thin <= rule::STREAM_MAX_ROWS && std::max(d.m, d.n) >= short_k_min_extent)
        return MI355_GEMM_ALGO_LP_128;
    // few rows or columns: dot products, the streaming kernel, or (below) the 128 x 128 kernel's split-K
    if (thin > rule::DOT_MAX_ROWS && thin <= rule::DOT_SHORT_GRID_MAX_ROWS && cdiv(std::max(d.m, d.n), rule::STREAM_ROWS_PER_WG) * d.batch < rule::DOT_SHORT_GRID_WGS &&
        d.batch == 1 && !(mid && d.k > rule::DOT_SHORT_GRID_LONG_K && cdiv(std::max(d.m, d.n), 128) < rule::DOT_SHORT_GRID_LONG_K_MIN_TILES) && gemm_skinny_supports(d, a, b, c))
        return MI355_GEMM_ALGO_SKINNY;
    if (thin >= rule::STREAM_MIN_ROWS && thin <= rule::STREAM_MAX_ROWS && gemm_stream64_supports(d, a, b, c) && stream64_wins(d)) return MI355_GEMM_ALGO_STREAM64;
    if (thin <= rule::DOT_FALLBACK_MAX_ROWS && gemm_skinny_supports(d, a, b, c) && (thin <= rule::DOT_MAX_ROWS || !(big4 || mid))) return MI355_GEMM_ALGO_SKINNY;
    // output-bound short K: the 128 x 128 kernel's single-stage form (dispatch_rules.md "short K")
    // (the tile bound at K = 193 ... 256 is where the persistent dripped-store kernel takes over: 16-bit C only -- with an f32 C 11712 x 10624 x 256, 1932 tiles, 99.4 us here
    //  against 115.4 on the 16x16x32 tile and 137.9 on the 32x32x16 one)
    if (mid && tiles256 > rule::CUS && (d.k <= rule::SHORT_K_ANY || (d.k <= rule::SHORT_K_BOUNDED && (tiles256 <= rule::SHORT_K_BOUNDED_TILES || d.dtype_c == MI355_DTYPE_F32)))) return MI355_GEMM_ALGO_LP_128;
    if (mid && tiles256 > rule::SQUARE_MIN_TILES && d.k <= rule::SHORT_K_ONE_ROUND) return MI355_GEMM_ALGO_LP_128;
    // one thin side over many tiles: never a 256-wide tile on that side; few COLUMNS fill the 256 rows of the tall tile where one round of it exists
    if (mid && thin <= rule::THIN_MAX_EXTENT) {
        const int64_t t128 = cdiv(d.m, 128) * d.batch, tall = cdiv(d.m, 256) * d.batch;
        if (d.n <= rule::THIN_MAX_EXTENT && d.m > rule::THIN_MAX_EXTENT && t128 > rule::CUS && tall <= rule::CUS && gemm_lp256x128_supports(d, a, b, c)) return MI355_GEMM_ALGO_LP_256X128;
        // 65 ... 128 rows or columns (dispatch_rules.md "thin, 65-128"): one round of 192 x 192 tiles where the 128 x 128 kernel would split a short K
        // or run a mostly empty second round
        // (late round 6: batches too -- heads x [seq x 128 x seq], the second product of an attention layer: the tile count is what decides whether the
        //  128 x 128 kernel splits K, whatever it is made of; a batched audit found 32 x 512 x 128 x 512 at 18.5 us against 10.9.  Batches from
        //  THIN_192_COLS_MIN_TILES tiles in either orientation: profiles/r06_batched_thin_ab.txt, 112 cases)
        if (thin >= rule::THIN_192_MIN_EXTENT && gemm_lp256x192_supports(d, a, b, c)) {
            const bool few_rows = d.m <= d.n;
            const int64_t along = cdiv(std::max(d.m, d.n), 128) * d.batch;
            if (d.k >= rule::THIN_192_MIN_K && d.k <= rule::THIN_192_MAX_K && along < rule::THIN_192_SPLIT_TILES &&
                along >= (few_rows && d.batch == 1 ? rule::THIN_192_ROWS_MIN_TILES : rule::THIN_192_COLS_MIN_TILES))
                return MI355_GEMM_ALGO_LP_192X192;
            if (d.batch > 1) return MI355_GEMM_ALGO_LP_128;        // (the two rules below were measured on single matrices only)
            if (!few_rows && d.k > rule::THIN_192_MAX_K && d.k <= rule::THIN_192_COLS_LONG_K && along >= rule::THIN_192_ROWS_MIN_TILES && along < rule::THIN_192_SPLIT_TILES)
                return MI355_GEMM_ALGO_LP_192X192;
            if (few_rows && along > rule::CUS && along < rule::PART_ROUND_MAX_TILES && d.k >= rule::THIN_192_PART_ROUND_MIN_K) return MI355_GEMM_ALGO_LP_192X192;
        }
        return MI355_GEMM_ALGO_LP_128;
    }
    // both extents past TILE_MIN_EXTENT, up to TILE_MAX_ROUNDS rounds of the square tile: the fitted cost tables decide among the five tile kernels
    if (big4 && mid && thin > TILE_MIN_EXTENT &&
        ((tiles256 <= TILE_CUS && d.k >= TILE_MIN_K) || (tiles256 <= TILE_MAX_ROUNDS * TILE_CUS && d.k >= TILE_MIN_K_ROUNDS))) {
        const int32_t pick = pick_tile_kernel(d, a, b, c);
        if (pick) return pick;
    }
    // outside the tables' domain: the 256 x 128 tile (more than one 128 x 128 tile per CU, at most one of it, a long K or one thin side) ...
    if (mid && tiles_of(d, 128, 128) > rule::CUS && tiles_of(d, 256, 128) <= rule::CUS && (d.k >= rule::TALL_TILE_MIN_K || thin <= rule::TALL_TILE_THIN_EXTENT) &&
        gemm_lp256x128_supports(d, a, b, c))
        return MI355_GEMM_ALGO_LP_256X128;
    // ... the square tile once the 128 x 128 kernel would need more than its two co-resident workgroups per CU, else the 128 x 128 kernel
    // (an f32 C at K < 512: a launch of the square tile costs 18.5 us however few tiles it has, the 128 x 128 kernel's time follows the tiles -- 11304 x 720 x 256, 135 tiles,
    //  14.2 us / 18.7; 3144 x 3280 x 256, 169, 15.2 / 18.5; level from 178: 19.9 / 19.3, 234 tiles 18.6 / 18.7)
    const int64_t square_min_tiles = d.dtype_c == MI355_DTYPE_F32 ? rule::SQUARE_MIN_TILES_F32_C : rule::SQUARE_MIN_TILES;
    if (big4 && (tiles256 > square_min_tiles || !mid)) return MI355_GEMM_ALGO_LP_256W4;
    if (mid) return MI355_GEMM_ALGO_LP_128;
    return MI355_GEMM_ALGO_GENERIC;
}
}  // namespace

namespace {

// When AUTO would land on the generic scalar kernel because of an operand's LAYOUT (transposed A, 16-bit row-major
// B), its K extent (not a multiple of the K-tile) or its alignment (rows / base not 16-byte aligned), the operand is
// first re-laid out into K-contiguous, zero-padded, aligned library scratch -- what the reference's launchers do
// with into_contiguous after matrix_batch_layout -- and the MFMA kernel runs on that.  `plan_relayout` is the pure
// part (also used by mi355_gemm_select); it returns false when nothing would be gained.
struct relayout_plan {
    bool a, b;              // which operands get a scratch copy
    int64_t kpad;           // K rounded up to the K-tile (zero columns add nothing)
    mi355_gemm_desc nd;     // the descriptor the MFMA kernel sees
};

bool plan_relayout(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, relayout_plan &p)
{
    // tiny AND short: not worth extra launches.  (late round 6, the audit of lhs [K][M]: the scalar kernel walks K serially, ~0.11 us per value, whatever the work --
    // 1 x 2360 x 512 89 us, 304 x 2 x 1024 115, 10 x 304 x 256 33, 11 x 792 x 128 17.9, 14 x 328 x 64 10.7 -- where the re-layout path costs its two or three launches:
    // 3 x 992 x 1536 16.3 us, 2 x 3968 x 512 15.0.  The work bound alone kept every K on the scalar kernel: profiles/r06_random_audit_ta.txt)
    constexpr int64_t RELAYOUT_TINY_WORK = (int64_t)1 << 21, RELAYOUT_TINY_MAX_K = 64;    // (K = 128: 11 x 792 x 128 18.7 us on the scalar kernel, 11.4 for 10 x 304 x 256 through the re-layout path: profiles/r06_tiny_relayout.txt)
    if (d.k == 0 || (d.m * d.n * d.k < RELAYOUT_TINY_WORK && d.k <= RELAYOUT_TINY_MAX_K)) return false;
    const int64_t esz = (int64_t)dtype_size(d.dtype_ab);
    const int64_t ktile = 128 / esz, ve = 16 / esz;
    p.kpad = (d.k + ktile - 1) / ktile * ktile;
    const bool ragged_k = p.kpad != d.k;
    const bool a_misaligned = (d.lda % ve) || (d.stride_a % ve) || (reinterpret_cast<uintptr_t>(a) & 15u);
    const bool b_misaligned = (d.ldb % ve) || (d.stride_b % ve) || (reinterpret_cast<uintptr_t>(b) & 15u);
    p.a = d.trans_a != 0 || ragged_k || a_misaligned;
    p.b = (!d.trans_b && (d.dtype_ab != MI355_DTYPE_F32 || ragged_k || b_misaligned || (d.n & 3))) ||
          (d.trans_b && (ragged_k || b_misaligned));
    if (!p.a && !p.b) return false;
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    auto planned = [&](bool pa, bool pb) {
        p.a = pa; p.b = pb;
        p.nd = d;
        p.nd.k = p.kpad;
        if (p.a) { p.nd.trans_a = 0; p.nd.lda = p.kpad; p.nd.stride_a = d.stride_a == 0 ? 0 : d.m * p.kpad; }
        if (p.b) { p.nd.trans_b = 1; p.nd.ldb = p.kpad; p.nd.stride_b = d.stride_b == 0 ? 0 : d.n * p.kpad; }
        return select(p.nd, p.a ? &aligned_dummy : a, p.b ? &aligned_dummy : b, c) != MI355_GEMM_ALGO_GENERIC;
    };
    // A 16-bit row-major B that is only here because A needs a new layout stays where it is when a tile kernel stages it natively
    // (until late round 3 both operands were transposed: 2048 x 2048 x 8192 with A stored [K][M] 110.6 us against 95.5 with B left alone)
    if (p.a && p.b && !d.trans_b && !ragged_k && !b_misaligned && d.dtype_ab != MI355_DTYPE_F32 && planned(true, false)) return true;
    return planned(p.a, p.b);
}

int32_t relayout_for_mfma(mi355_ctx *ctx, hipStream_t s, const mi355_gemm_desc &d, const void *a, const void *b, void *c,
                          mi355_gemm_desc &nd, const void *&na, const void *&nb)
{
    relayout_plan p;
    if (!plan_relayout(d, a, b, c, p)) return MI355_E_UNSUPPORTED;
    const int esz = (int)dtype_size(d.dtype_ab);
    nd = p.nd; na = a; nb = b;
    if (p.a) {
        const int64_t nba = d.stride_a == 0 ? 1 : d.batch;
        void *q = nullptr;
        if (scratch_get(ctx, s, SCRATCH_RELAYOUT_A, (size_t)(nba * d.m * p.kpad * esz), &q) != MI355_OK) return MI355_E_UNSUPPORTED;
        if (d.trans_a) {                                                       // [K][M] -> [M][kpad], zeros in the pad columns
            if (p.kpad != d.k) launch_zero_columns(s, q, nba * d.m, d.k * esz, p.kpad * esz);
            launch_transpose(s, a, q, d.k, d.m, d.lda, p.kpad, nba, d.stride_a, d.m * p.kpad, esz);
        } else {
            launch_pad_copy(s, a, q, d.m, d.k, p.kpad, d.lda, p.kpad, nba, d.stride_a, d.m * p.kpad, esz);
        }
        na = q;
    }
    if (p.b) {
        const int64_t nbb = d.stride_b == 0 ? 1 : d.batch;
        void *q = nullptr;
        if (scratch_get(ctx, s, SCRATCH_RELAYOUT_B, (size_t)(nbb * d.n * p.kpad * esz), &q) != MI355_OK) return MI355_E_UNSUPPORTED;
        if (!d.trans_b) {                                                      // [K][N] -> [N][kpad]
            if (p.kpad != d.k) launch_zero_columns(s, q, nbb * d.n, d.k * esz, p.kpad * esz);
            launch_transpose(s, b, q, d.k, d.n, d.ldb, p.kpad, nbb, d.stride_b, d.n * p.kpad, esz);
        } else {
            launch_pad_copy(s, b, q, d.n, d.k, p.kpad, d.ldb, p.kpad, nbb, d.stride_b, d.n * p.kpad, esz);
        }
        nb = q;
    }
    check_launch(ctx, "mi355_gemm(operand re-layout)");
    return MI355_OK;
}

// ---- the last, partly filled round of 256x256 tiles ----------------------------------------------------------------------
// All tiles of a GEMM take the same time, so T tiles on 256 CUs cost ceil(T / 256) rounds: 576 tiles (6144^3) pay for
// 768.  When the leftover is at most half a round, the output is cut into a part whose tile count (nearly) fills whole
// rounds and a strip of at most 96 tiles whose K range is split `s` ways over the CUs that would otherwise idle: the
// strip runs as ONE batched launch of the same kernel (batch entry z = K slice z: operand "batch strides" of one slice
// along the rows, f32 partial slabs as the batched output) followed by the split-K fold (gemm_splitk.hip), which adds
// the slabs in slice order (deterministic) and converts.  Chosen by a cost model in K-tile units; only for batch == 1.
struct tail_plan {
    bool along_m;          // the strip is the last rows (true) or the last columns (false) of C
    int64_t main_extent;   // rows (columns) handled by the plain launch
    int64_t splits;
};

bool plan_tail_split(const mi355_gemm_desc &d, tail_plan &best, double *ratio = nullptr)
{
    if (ratio) *ratio = 1.0;
    if (d.batch != 1 || d.trans_a || (d.n & 3)) return false;
    const int64_t esz = (int64_t)dtype_size(d.dtype_ab), ktile = 128 / esz, nk = d.k / ktile;
    if (!d.trans_b && ((d.n & (16 / esz - 1)) || is_fp8(d.dtype_ab))) return false;   // row-major B: f32 and 16-bit, whole 16-byte pieces
    const int64_t tm = (d.m + 255) / 256, tn = (d.n + 255) / 256, T = tm * tn;
    if (nk < 8) return false;
    // cycles: a K-tile costs ~2 200, a tile's prologue + epilogue ~10 000, a launch ~5 000, the fold moves
    // (s + 1) x 256 KiB per strip tile at ~2 500 B per cycle of the whole chip
    const double CK = 2200.0, CFIX = 10000.0, CLAUNCH = 5000.0;
    // A partly filled round is cheaper than a full one: the idle CUs' power budget lets the busy ones clock higher
    // (64 leftover tiles cost ~0.66 of a round, 128 ~0.83: 6144^3 and 4096 x 6144 x 4096).  Calibrated interleaved against
    // the plain launch (tools/dev/tail_ab.py): with F0 = 0.7 and strips of at most 96 tiles the split is taken at
    // 1.02-1.13, 2.25, 3.06 and 4.12 rounds (+28, +18, +15, +11, +7, +7, +7 %) and left alone at 1.5-1.56, 2.44, 4.5 rounds.
    constexpr double F0 = 0.7;
    auto rounds = [](int64_t t) {
        const int64_t left = t % 256;
        return (double)(t / 256) + (left ? F0 + (1.0 - F0) * (double)left / 256.0 : 0.0);
    };
    const double now = rounds(T) * ((double)nk * CK + CFIX);
    double best_cost = now * 0.93;                          // must win by 7 % to be worth two extra launches
    bool found = false;
    for (int dir = 0; dir < 2; ++dir) {
        const int64_t t_along = dir == 0 ? tm : tn, t_other = dir == 0 ? tn : tm;
        // the strip is whole tiles of the LAST rows (columns): when that extent ends in a partly filled tile the model's tile
        // count is wrong and the split lost (4160 x 10240 x 8192: 618 us against 531 plain, tools/dev/random_audit.py)
        if ((dir == 0 ? d.m : d.n) % 256) continue;
        for (int64_t strip = 1; strip <= t_along && strip * t_other <= 96; ++strip) {
            const int64_t t_strip = strip * t_other, t_main = T - t_strip;
            for (int64_t sp = 2; sp <= 16 && sp * t_strip <= 256 && nk / sp >= 4; ++sp) {
                if (nk % sp) continue;
                const double fold = (double)t_strip * (double)(sp + 1) * 262144.0 / 2500.0;
                const double cost = rounds(t_main) * ((double)nk * CK + CFIX) + rounds(sp * t_strip) * ((double)(nk / sp) * CK + CFIX) + fold +
                                    (t_main > 0 ? 2.0 : 1.0) * CLAUNCH;
                if (cost < best_cost) {
                    best_cost = cost;
                    best.along_m = dir == 0;
                    best.main_extent = (t_along - strip) * 256;
                    best.splits = sp;
                    found = true;
                }
            }
        }
    }
    if (found && ratio) *ratio = best_cost / now;
    return found;
}

double tail_split_ratio(const mi355_gemm_desc &d)
{
    if (tiles_of(d, 256, 256) <= rule::CUS) return 1.0;       // (the planner is calibrated on leftover rounds: more than one round of tiles)
    tail_plan tp;
    double r = 1.0;
    plan_tail_split(d, tp, &r);
    return r < 1.0 ? std::min(1.0, r * TAIL_SPLIT_TABLE_BIAS) : 1.0;
}

// Several rounds of short tiles: the persistent form (gemm_lp256p.hip) streams the next tile's operands during the epilogue
// and lets the C stores drain under the next tile's MFMAs.  Measured against the one-tile-per-workgroup kernel,
// interleaved (tools/dev/p_vs_w4.py): K = 512 +10 %, 1024 +4 %, 2048 +1...4 %, 4096 +1 %, 8192 a tie; single-round
// launches -0.5...-2 %.  A leftover round that the strip split handles gains more from that and keeps the plain kernel.
bool prefers_persistent(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    if (d.dtype_ab != MI355_DTYPE_BF16 && d.dtype_ab != MI355_DTYPE_F16) return false;
    const int64_t tiles = ((d.m + 255) / 256) * ((d.n + 255) / 256) * d.batch, nk = d.k / 64;
    // more than one round of tiles (round 2: was two full rounds).  With 257-511 tiles the second round is partly empty either
    // way, and the tile hand-over of the persistent forms still hides the epilogues: 8192 x 3072 x 512 (384 tiles) 32.5 ->
    // 28.1 us, x 1024 50.0 -> 45.8, 7168 x 4096 x 1024 (448) 52.1 -> 49.9, 8192 x 2560 x 512 (320) 30.2 -> 27.2, level from
    // K = 2048 up (tools/dev/shortk_probe.py)
    if (tiles <= rule::CUS || nk > rule::PERSISTENT_MAX_KTILES) return false;
    if (!gemm_lp256p_supports(d, a, b, c)) return false;
    tail_plan tp;
    return !plan_tail_split(d, tp);
}

// 16-bit C: the persistent kernel that keeps the finished tile in registers and drips its stores into the next tile's K loop
// (gemm_lp256q.hip).  Measured against gemm_lp256p.hip, interleaved, 64 x 2048 x 2048 x K (tools/dev/q_ab.py): K = 384 / 448 /
// 512 (8 stores per K-tile) +1.5 / +2.5 / +4 %, K = 576 ... 960 (4 or 2 stores per K-tile) -5 ... -11 %, K = 1024 / 1536 / 2048 /
// 4096 +3.6 / +1.5 / +3.6 ... 4.9 / +1.2 %, 8192 a tie.
bool prefers_dripped_stores(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    const int64_t nk = d.k / 64;
    return gemm_lp256q_supports(d, a, b, c) && (nk >= rule::DRIP_MIN_KTILES || (nk >= rule::DRIP_SHORT_MIN_KTILES && nk <= rule::DRIP_SHORT_MAX_KTILES));
}

bool qm_takes(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    tail_plan tp;
    return gemm_lp256qm_supports(d, a, b, c) && !plan_tail_split(d, tp);
}

// ... or the launcher's tail split runs its main part (whole rounds of full tiles) on that kernel (run_tail_split)
bool qm_takes_tail_main(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    tail_plan tp;
    if (!plan_tail_split(d, tp) || tp.main_extent <= 0) return false;
    mi355_gemm_desc md = d;
    if (tp.along_m) md.m = tp.main_extent; else md.n = tp.main_extent;
    return gemm_lp256qm_supports(md, a, b, c);
}

// 16-bit operands, f32 C, [N][K] rhs: the one-tile-per-workgroup 16x16x32 kernel wherever the square tile is the choice and no tail split is planned
bool m16_takes_f32_c(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    tail_plan tp;
    return d.dtype_c == MI355_DTYPE_F32 && tiles_of(d, 256, 256) >= rule::M16_F32_C_MIN_TILES && gemm_lp256m16_supports(d, a, b, c) && !plan_tail_split(d, tp);
}

int32_t select_auto(const mi355_gemm_desc &d, const void *a, const void *b, const void *c, bool strip_kernel = true)
{
    const int32_t algo = select(d, a, b, c, strip_kernel);
    if (algo != MI355_GEMM_ALGO_LP_256W4) return algo;
    // Round 6: FULL square tiles of 16-bit operands with a 16-bit C, wherever the square tile is the choice -- the persistent dripped-store loop on
    // v_mfma_f32_16x16x32 (gemm_lp256qm.hip).  First K loop of the round, cold, interleaved: ahead of every other form of the tile on all 22
    // [N][K] shapes from 324 to 2304 tiles and K = 448 ... 16384 (config C5 1 275 -> 1 340 TFLOP/s: profiles/r06_qm_shapes_ab.txt,
    // r06_qm_longk_ab.txt), its row-major-rhs form only at K = 2048 ... 4096 (r06_qm_nn_ab.txt).  Second K loop -- bookkeeping in the empty
    // MFMA gaps, two-instruction DMA pieces: +4 ... +10 % on both layouts (profiles/r06_qm_pre_shapes_ab.txt: row-major rhs 8192^3 1 474
    // (lp256w4) -> 1 617 TFLOP/s, x 1024 1 281 (lp256q) -> 1 361, x 512 1 029 -> 1 084; [N][K] 8192^2 x 2048 1 391 -> 1 526; exactly one
    // round, 4096^3, 96.9 us (lp256m16) -> 93.9; 196 tiles, 3584^3, 80.2 (lp256w4) -> 75.2, r06_qm_rule_ab.txt): the K window of the row-major
    // form and the "more than one round" bound went with it.
    // (Not where the launcher splits a ragged last round off: that planner's model is the 32x32 kernel's.)
    if (qm_takes(d, a, b, c)) return MI355_GEMM_ALGO_LP_256QM;
    // (late round 6) an f32 C: the same tile on v_mfma_f32_16x16x32, one tile per workgroup (gemm_lp256m16.hip) -- 3 ... 12 % ahead of the 32x32x16 kernel on all 55
    // audited shapes from 178 tiles up where the square tile is within 10 % of the best kernel, full tiles or ragged, K = 256 ... 14336 (median 0.94), and of
    // gemm_lp256p.hip's overlap on short K (10944 x 5184 x 512 87.0 / 95.0 us): profiles/r06_random_audit_c32.txt
    if (m16_takes_f32_c(d, a, b, c)) return MI355_GEMM_ALGO_LP_256M16;
    if (prefers_persistent(d, a, b, c)) return prefers_dripped_stores(d, a, b, c) ? MI355_GEMM_ALGO_LP_256Q : MI355_GEMM_ALGO_LP_256P;
    // Round 5: several full rounds of 256x256 tiles of [N][K] 16-bit operands run at the chip's POWER limit on random data; there the
    // same tile on v_mfma_f32_16x16x32 (gemm_lp256m16.hip: half the accumulator bytes through the register file per FLOP) holds
    // 1.83-1.87 GHz where the 32x32x16 kernel holds 1.63: 8192^3 1 440 -> 1 533-1 563 TFLOP/s.  Below ~3 rounds the chip is not
    // power-bound and the wider instruction's slack per issue slot wins (4096^3 a tie, 3584^3 -4 %): profiles/r05_m16_ab.txt.
    // (Not where the launcher would split a ragged last round off: that planner's model is the 32x32 kernel's.)
    {
        tail_plan tp;
        // (round 6: ... and on exactly ONE FULL round -- every CU busy, the same power limit: 4096^2 x 1024 / 2048 / 4096 / 8192 32.5 / 54.5 /
        //  103.6 / 194.0 -> 30.7 / 51.6 / 98.1 / 183.8 us, interleaved, seven rounds, profiles/r06_one_round_m16_ab.txt; a tie on three boxes in
        //  round 5; 196 tiles the other way, 75.2 / 78.0.  The persistent form is 1-3 % behind the plain one there: nothing to overlap.)
        const int64_t t256 = tiles_of(d, 256, 256);
        if ((t256 >= rule::M16_MIN_TILES || t256 == rule::CUS) && gemm_lp256m16_supports(d, a, b, c) && !plan_tail_split(d, tp)) return MI355_GEMM_ALGO_LP_256M16;
    }
    return algo;
}

int32_t run_tail_split(mi355_ctx *ctx, hipStream_t s, const mi355_gemm_desc &d, const void *a, const void *b, void *c,
                       const tail_plan &p, const epilogue_args *ep)
{
    const int64_t esz = (int64_t)dtype_size(d.dtype_ab), csz = (int64_t)dtype_size(d.dtype_c);
    const int64_t ms = p.along_m ? d.m - p.main_extent : d.m, ns = p.along_m ? d.n : d.n - p.main_extent;   // the strip
    float *slabs = nullptr;
    if (splitk_scratch(ctx, s, (size_t)(p.splits * ms * ns) * sizeof(float), &slabs) != MI355_OK) return MI355_E_UNSUPPORTED;
    const char *a0 = static_cast<const char *>(a), *b0 = static_cast<const char *>(b);
    char *c0 = static_cast<char *>(c);
    const char *as = p.along_m ? a0 + p.main_extent * d.lda * esz : a0;
    // the strip's first column of B: a row of [N][K] storage, a column of row-major [K][N]
    const char *bs = p.along_m ? b0 : b0 + (d.trans_b ? p.main_extent * d.ldb * esz : p.main_extent * esz);
    char *cs = p.along_m ? c0 + p.main_extent * d.ldc * csz : c0 + p.main_extent * csz;
    mi355_gemm_desc sd = d;                                 // the strip: batch entry z = K slice z, f32 slab output
    sd.m = ms; sd.n = ns; sd.k = d.k / p.splits; sd.batch = p.splits;
    sd.stride_a = sd.k; sd.stride_b = d.trans_b ? sd.k : sd.k * d.ldb; sd.stride_c = ms * ns; sd.ldc = ns; sd.dtype_c = MI355_DTYPE_F32;
    if (!gemm_lp256w4_supports(sd, as, bs, slabs)) return MI355_E_UNSUPPORTED;
    if (p.main_extent > 0) {
        mi355_gemm_desc md = d;
        if (p.along_m) md.m = p.main_extent; else md.n = p.main_extent;
        if (!gemm_lp256w4_supports(md, a, b, c)) return MI355_E_UNSUPPORTED;
        // (round 6: whole rounds of full tiles with a 16-bit C -- the persistent 16x16x32 kernel where it takes the main part:
        //  4608 x 4096 x 8192 254.6 -> 240 us, profiles/r06_tail_split_main_on_qm.txt)
        const int32_t rc = !ep && gemm_lp256qm_supports(md, a, b, c) ? launch_gemm_lp256qm(ctx, s, md, a, b, c)
                           : ep && gemm_lp256m16_supports(md, a, b, c) ? launch_gemm_lp256m16(ctx, s, md, a, b, c, ep)
                                                                       : launch_gemm_lp256w4(ctx, s, md, a, b, c, nullptr, ep);
        if (rc != MI355_OK) return rc;
    }
    const int32_t rc = launch_gemm_lp256w4(ctx, s, sd, as, bs, slabs);
    if (rc != MI355_OK) return rc;
    if (ep) launch_epilogue(s, slabs, (uint32_t)p.splits, ms * ns, p.along_m ? epilogue_at(*ep, p.main_extent, 0) : epilogue_at(*ep, 0, p.main_extent), cs, 1, ms, ns, d.ldc, 0);
    else launch_splitk_fold(s, slabs, (uint32_t)p.splits, ms * ns, 1, ms, ns, cs, d.dtype_c, d.ldc, 0);
    check_launch(ctx, "mi355_gemm(tail split-K fold)");
    return MI355_OK;
}

}  // namespace

namespace {

// Operands that would be copied before a matrix-core kernel can stage them, with an epilogue: gemm_edge.hip takes them as they lie, while the
// product is small enough for its smaller tiles.  us, copies and product / edge: f32, any layout: 333 x 517 x 1001 42 / 19, 2000 x 2000 x 501 63 / 49,
// 8001 x 1001 x 333 94 / 66, but 2001 x 2003 x 2005 (16 GFLOP) 179 / 251.  16-bit, both operands k-contiguous: 333 x 517 x 1001 23 / 14, 4001 x 4003 x
// 1001 (32 GFLOP) 68 / 64, 4001 x 4003 x 4005 147 / 196; otherwise (pieces turned on their way into LDS) 8001 x 1001 x 333 50 / 26, 2001 x 2003 x
// 2005 58 / 122.
// f32 operands that the 128 x 128 kernel would take, too few such tiles for the chip and no long K to slice: 512^3 25 / 16, 1024 x 1024 x 512 40 / 20,
// 2048 x 1024 x 512 41 / 28, 512 x 512 x 2048 29 / 22; not 1024^3 31 / 33 (K in slices there too), nor 2048 x 2048 x 256 27 / 31 (256 tiles).
bool edge_wins(const mi355_gemm_desc &d, const void *a, const void *b, const void *c)
{
    const int32_t algo = select_auto(d, a, b, c);
    const double flops = 2.0 * (double)d.m * (double)d.n * (double)d.k * (double)d.batch;
    if (algo == MI355_GEMM_ALGO_F32_MFMA) return tiles_of(d, 128, 128) <= rule::CUS / 2 && (flops <= 1.1e9 || d.k <= 512);
    if (algo != MI355_GEMM_ALGO_GENERIC) return false;
    return flops <= (d.dtype_ab != MI355_DTYPE_F32 && !d.trans_a && d.trans_b ? 40e9 : 8e9);
}

// mi355_gemm of a validated descriptor, with the epilogue `ep` where one is given (it may have no parts)
int32_t run_gemm(mi355_ctx *ctx, hipStream_t s, const mi355_gemm_desc &desc, const void *a, const void *b, void *c, const epilogue_args *ep)
{
    mi355_gemm_desc d = desc;
    if (ep && gemm_edge_supports(d) && (d.algo == MI355_GEMM_ALGO_EDGE || (d.algo == MI355_GEMM_ALGO_AUTO && edge_wins(d, a, b, c))))
        return launch_gemm_edge(ctx, s, d, a, b, c, *ep);
    if (d.algo == MI355_GEMM_ALGO_EDGE)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm: the edge kernel belongs to mi355_gemm_fused and takes f32, bf16 and f16 operands with k > 0");
    // nothing to do on the accumulators: the plain product on its own kernels, the persistent ones among them (the products of a gradient)
    if (ep && !has_parts(*ep)) ep = nullptr;
    int32_t algo = d.algo == MI355_GEMM_ALGO_AUTO ? select_auto(d, a, b, c) : d.algo;
    if (d.algo == MI355_GEMM_ALGO_AUTO && algo == MI355_GEMM_ALGO_GENERIC) {
        mi355_gemm_desc nd;
        const void *na, *nb;
        if (relayout_for_mfma(ctx, s, d, a, b, c, nd, na, nb) == MI355_OK) {
            d = nd; a = na; b = nb;
            algo = select_auto(d, a, b, c);
        }
    }
    // the strip kernel needs scratch + ticket words that cannot be created inside a capture window: AUTO then takes what it took
    // before that kernel existed (as the split-K paths fall back to their unsplit forms)
    // -- through the same AUTO pipeline (persistent-kernel promotion; GENERIC = "re-lay out, then select again"), so that a
    // captured graph replays the kernel AUTO would have taken, not the scalar correctness net
    if (d.algo == MI355_GEMM_ALGO_AUTO && algo == MI355_GEMM_ALGO_NNROWS && !gemm_nnrows_ready(ctx, s, d)) {
        algo = select_auto(d, a, b, c, false);
        if (algo == MI355_GEMM_ALGO_GENERIC) {
            mi355_gemm_desc nd;
            const void *na, *nb;
            if (relayout_for_mfma(ctx, s, d, a, b, c, nd, na, nb) == MI355_OK) {
                d = nd; a = na; b = nb;
                algo = select_auto(d, a, b, c, false);
            }
        }
    }
    // 8-bit operands, at most two 128 x 128 tiles a CU: two co-resident workgroups hide each other's epilogue where the square tile waits for its
    // own (us, square / 128: 1777 x 4096 x 4096 with silu and residual 55.6 / 45.1, 2048 x 4096 x 4096 56.8 / 47.4; three tiles a CU the other way,
    // 2560 x 4096 x 4096 57.3 / 79.6; without parts the square tile's own stores, 41.3 for 1777 x 4096 x 4096)
    if (ep && d.algo == MI355_GEMM_ALGO_AUTO && algo == MI355_GEMM_ALGO_LP_256W4 && is_fp8(d.dtype_ab) && tiles_of(d, 128, 128) <= 2 * rule::CUS &&
        gemm_lp128_supports(d, a, b, c))
        algo = MI355_GEMM_ALGO_LP_128;
    // the persistent kernels carry no epilogue: the same tile, one tile a workgroup
    if (ep && (algo == MI355_GEMM_ALGO_LP_256P || algo == MI355_GEMM_ALGO_LP_256Q || algo == MI355_GEMM_ALGO_LP_256QM))
        algo = gemm_lp256m16_supports(d, a, b, c) ? MI355_GEMM_ALGO_LP_256M16 : MI355_GEMM_ALGO_LP_256W4;
    // (MI355_W4_TAIL_SPLIT=1, dev: a FORCED 256x256 launch is split as well -- lets tools/ab_algos.py time the split form against the other tiles)
    static const bool split_forced_too = [] { const char *e = getenv("MI355_W4_TAIL_SPLIT"); return e && atoi(e) == 1; }();
    if ((d.algo == MI355_GEMM_ALGO_AUTO || split_forced_too) && algo == MI355_GEMM_ALGO_LP_256W4) {
        tail_plan tp;
        if (plan_tail_split(d, tp) && run_tail_split(ctx, s, d, a, b, c, tp, ep) == MI355_OK) return MI355_OK;
    }
    switch (algo) {
    case MI355_GEMM_ALGO_GENERIC: return launch_gemm_generic(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_F32_MFMA: return launch_gemm_f32_mfma(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_LP_128: return launch_gemm_lp128(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_LP_256: return launch_gemm_lp256w4(ctx, s, d, a, b, c, nullptr, ep);      // retired 8-wave kernel: an alias since ABI 8
    case MI355_GEMM_ALGO_LP_256W4: return launch_gemm_lp256w4(ctx, s, d, a, b, c, nullptr, ep);
    case MI355_GEMM_ALGO_LP_256P: return launch_gemm_lp256p(ctx, s, d, a, b, c);
    case MI355_GEMM_ALGO_LP_256Q: return launch_gemm_lp256q(ctx, s, d, a, b, c);
    case MI355_GEMM_ALGO_SKINNY: return launch_gemm_skinny(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_STREAM64: return launch_gemm_stream64(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_LP_256X128: return launch_gemm_lp256x128(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_NNROWS: return launch_gemm_nnrows(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_LP_256X192: return launch_gemm_lp256x192(ctx, s, d, a, b, c, 256, ep);
    case MI355_GEMM_ALGO_LP_192X192: return launch_gemm_lp256x192(ctx, s, d, a, b, c, 192, ep);
    case MI355_GEMM_ALGO_LP_256M16: return launch_gemm_lp256m16(ctx, s, d, a, b, c, ep);
    case MI355_GEMM_ALGO_LP_256QM: return launch_gemm_lp256qm(ctx, s, d, a, b, c);
    default: return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm: unknown algo %d", algo);
    }
}

}  // namespace

MI355_API int32_t mi355_gemm(mi355_ctx *ctx, mi355_stream stream, const mi355_gemm_desc *desc, const void *a,
                             const void *b, void *c)
{
    MI355_REQUIRE_CTX(ctx);
    const int32_t rc = validate(ctx, desc, a, b, c);
    if (rc != -1) return rc;
    return run_gemm(ctx, stream_of(ctx, stream), *desc, a, b, c, nullptr);
}

// cmma::execute(a, b, c, d) at tensor level: D = A * B + C.  The selected kernel writes the f32 product into
// library-owned per-stream scratch; gemm_add.hip adds C in f32 and rounds once to dtype_c.
MI355_API int32_t mi355_gemm_add(mi355_ctx *ctx, mi355_stream stream, const mi355_gemm_desc *desc, const void *a, const void *b,
                                 const void *c, void *d_out)
{
    MI355_REQUIRE_CTX(ctx);
    int32_t rc = validate(ctx, desc, a, b, d_out);
    if (rc != -1) return rc;
    if (!c) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_add: the C operand is NULL");
    hipStream_t s = stream_of(ctx, stream);
    const mi355_gemm_desc &d = *desc;
    // f32 output on the 256x256 kernel: C is added inside the kernel's epilogue (one extra read of C, nothing else)
    // (every form of the square tile AUTO may name for an f32 C -- the plain kernel, its persistent form, the 16x16x32 form since round 5 --
    // is answered by the plain kernel's fused epilogue: no 4-bytes-per-output scratch product, no second pass, nothing to allocate inside
    // a capture window.  8192^3 bf16 + f32 C was fused until round 5's AUTO rule for the 16x16x32 kernel silently took it off this path.)
    if (d.dtype_c == MI355_DTYPE_F32 && (d.algo == MI355_GEMM_ALGO_AUTO || d.algo == MI355_GEMM_ALGO_LP_256W4) &&
        (reinterpret_cast<uintptr_t>(c) & 15u) == 0 && gemm_lp256w4_supports(d, a, b, d_out)) {
        const int32_t pick = d.algo == MI355_GEMM_ALGO_LP_256W4 ? MI355_GEMM_ALGO_LP_256W4 : select_auto(d, a, b, d_out);
        if (pick == MI355_GEMM_ALGO_LP_256W4 || pick == MI355_GEMM_ALGO_LP_256P || pick == MI355_GEMM_ALGO_LP_256M16)
            return launch_gemm_lp256w4(ctx, s, d, a, b, d_out, c);
    }
    void *prod = nullptr;
    const size_t bytes = (size_t)d.batch * (size_t)d.m * (size_t)d.n * sizeof(float);
    if (scratch_get(ctx, s, SCRATCH_PRODUCT, bytes, &prod) != MI355_OK)
        return fail(ctx, MI355_E_UNSUPPORTED, "mi355_gemm_add: no scratch for the %zu-byte f32 product (inside a capture window?)", bytes);
    mi355_gemm_desc pd = d;
    pd.dtype_c = MI355_DTYPE_F32;
    pd.ldc = d.n;
    pd.stride_c = d.m * d.n;
    rc = mi355_gemm(ctx, stream, &pd, a, b, prod);
    if (rc != MI355_OK) return rc;
    launch_add_c(s, static_cast<const float *>(prod), c, d_out, d.batch, d.m, d.n, d.dtype_c, d.ldc, d.stride_c);
    check_launch(ctx, "mi355_gemm_add");
    return MI355_OK;
}

// act(rs cs (A B) + bias) + residual: the kernel that mi355_gemm would take runs the epilogue on its accumulators (or in the fold of its K slices).
MI355_API int32_t mi355_gemm_fused(mi355_ctx *ctx, mi355_stream stream, const mi355_gemm_desc *desc, const mi355_gemm_epilogue *epilogue, const void *a,
                                   const void *b, void *c)
{
    MI355_REQUIRE_CTX(ctx);
    if (!epilogue) return fail(ctx, MI355_E_INVALID_ARGUMENT, "mi355_gemm_fused: the epilogue is NULL");
    int32_t rc = validate(ctx, desc, a, b, c);
    if (rc != -1) return rc;
    rc = validate_epilogue(ctx, *desc, *epilogue, a, b, c);
    if (rc != MI355_OK) return rc;
    const epilogue_args ep = make_epilogue(*epilogue, desc->dtype_c);
    return run_gemm(ctx, stream_of(ctx, stream), *desc, a, b, c, &ep);
}

// Introspection (no device needed): how mi355_gemm would cut a descriptor that AUTO resolves to the 256x256 kernel.
MI355_API int32_t mi355_gemm_split_plan(const mi355_gemm_desc *desc, int32_t compute_units, int32_t *out_slices)
{
    if (!desc || !out_slices || compute_units < 0) return MI355_E_INVALID_ARGUMENT;
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    *out_slices = 1;
    if (desc->m <= 0 || desc->n <= 0 || desc->k <= 0 || desc->batch <= 0) return MI355_OK;
    if (!gemm_lp128_supports(*desc, &aligned_dummy, &aligned_dummy, &aligned_dummy)) return MI355_OK;   // the launcher would never see it
    *out_slices = (int32_t)lp128_split_count(*desc, compute_units ? compute_units : 256);
    return MI355_OK;
}

MI355_API int32_t mi355_gemm_tail_plan(const mi355_gemm_desc *desc, int32_t *out_along_m, int64_t *out_main_extent, int32_t *out_splits)
{
    if (!desc || !out_along_m || !out_main_extent || !out_splits) return MI355_E_INVALID_ARGUMENT;
    tail_plan tp{};
    // (the split belongs to the 256x256 kernel: a descriptor AUTO hands to another kernel -- a narrow tile of the cost table since
    // round 5 -- is launched whole, exactly as mi355_gemm does it)
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    const bool split = (desc->algo != MI355_GEMM_ALGO_AUTO || select_auto(*desc, &aligned_dummy, &aligned_dummy, &aligned_dummy) == MI355_GEMM_ALGO_LP_256W4) &&
                       plan_tail_split(*desc, tp);
    *out_along_m = split ? (tp.along_m ? 1 : 0) : 0;
    *out_main_extent = split ? tp.main_extent : 0;
    *out_splits = split ? (int32_t)tp.splits : 1;
    return MI355_OK;
}

MI355_API int32_t mi355_gemm_relayout_plan(const mi355_gemm_desc *desc, int32_t *out_relayout_a, int32_t *out_relayout_b)
{
    if (!desc || !out_relayout_a || !out_relayout_b) return MI355_E_INVALID_ARGUMENT;
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    *out_relayout_a = *out_relayout_b = 0;
    if (desc->m <= 0 || desc->n <= 0 || desc->batch <= 0) return MI355_OK;
    if (select_auto(*desc, &aligned_dummy, &aligned_dummy, &aligned_dummy) != MI355_GEMM_ALGO_GENERIC) return MI355_OK;
    relayout_plan p;                  // exactly what mi355_gemm does before it settles for the scalar kernel
    if (plan_relayout(*desc, &aligned_dummy, &aligned_dummy, &aligned_dummy, p)) {
        *out_relayout_a = p.a ? 1 : 0;
        *out_relayout_b = p.b ? 1 : 0;
    }
    return MI355_OK;
}

MI355_API int32_t mi355_gemm_select(mi355_ctx *ctx, const mi355_gemm_desc *desc, int32_t *out_algo)
{
    (void)ctx;                           // may be NULL: nothing below asks the device
    if (!desc || !out_algo) return MI355_E_INVALID_ARGUMENT;
    // alignment-dependent choices are evaluated for 16-byte aligned operands
    static const char aligned_dummy __attribute__((aligned(16))) = 0;
    const mi355_gemm_desc &d = *desc;
    int32_t algo = select_auto(d, &aligned_dummy, &aligned_dummy, &aligned_dummy);
    if (algo == MI355_GEMM_ALGO_GENERIC) {
        relayout_plan p;                  // what mi355_gemm does before it settles for the scalar kernel
        if (plan_relayout(d, &aligned_dummy, &aligned_dummy, &aligned_dummy, p))
            algo = select_auto(p.nd, &aligned_dummy, &aligned_dummy, &aligned_dummy);
    }
    *out_algo = algo;
    return MI355_OK;
}
