// Runs the kernels of the operators around a linear layer on the CPU (hip/hip_runtime.h beside this file) with every operand flush against pages
// that may not be touched, at its end or at its start, workspaces of exactly the size the entry points ask for.  An access outside an operand ends
// the program behind the line that names the case; each case runs twice over different contents, so that an element of an output that is not
// written, or a byte between its rows that is, shows too.  Products are compared with sums in 64 bits.
#include <sys/mman.h>
#include <unistd.h>

#include <cstdarg>
#include <random>

#include "linear_ops.hpp"
#include "rowops.hpp"
#include "gemm_epilogue.hpp"

using namespace mi355;

static bool front;
static int failures = 0;
static std::string message;
static std::mt19937 rng(1);

struct guarded {
    char *map, *p;
    size_t bytes, span;
    explicit guarded(size_t n) : bytes(n)
    {
        const size_t page = (size_t)sysconf(_SC_PAGESIZE), inner = (n + page - 1) / page * page;
        span = inner + 2 * page;
        map = (char *)mmap(nullptr, span, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
        if (inner) mprotect(map + page, inner, PROT_READ | PROT_WRITE);
        p = front ? map + page : map + page + inner - n;
    }
    ~guarded() { munmap(map, span); }
    guarded(const guarded &) = delete;
};
static std::vector<std::unique_ptr<guarded>> scratch;
static void *fresh(size_t n) { scratch.push_back(std::make_unique<guarded>(n)); return scratch.back()->p; }

namespace mi355 {
int32_t fail(mi355_ctx *, int32_t code, const char *fmt, ...)
{
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    message = text;
    return code;
}
void check_launch(mi355_ctx *, const char *) {}
int32_t splitk_scratch(mi355_ctx *, hipStream_t, size_t bytes, float **out) { *out = (float *)fresh(bytes); return MI355_OK; }
}  // namespace mi355
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }
extern "C" const char *hipGetErrorString(hipError_t) { return ""; }

static mi355_ctx ctx;
static const char *now = "";
#define CHECK(x, ...) do { if (!(x)) { ++failures; printf("%s: ", now); printf(__VA_ARGS__); printf("\n"); } } while (0)

static float value() { return (float)((int)(rng() % 4001) - 2000) / 1000.0f; }
static void put(void *p, int64_t i, int32_t dt, float v)
{
    if (dt == MI355_DTYPE_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = dt == MI355_DTYPE_BF16 ? f32_to_bf16_rne(v) : f32_to_f16_rne(v);
}
static double get_at(const void *p, int64_t i, int32_t dt) { return load1_any(p, dt, i); }

// `batch` matrices of rows x cols; the operand ends with its last element
struct matrix {
    int64_t rows, cols, ld, batch, stride;
    int32_t dt;
    size_t esz;
    std::unique_ptr<guarded> g;
    matrix(int64_t r, int64_t c, int64_t pad, int32_t dtype, int64_t b = 1, bool in_turn = false) : rows(r), cols(c), batch(b), dt(dtype), esz(dtype_size(dtype))
    {
        ld = in_turn ? (c + pad) * b : c + pad;
        stride = in_turn ? c + pad : b > 1 ? r * ld + pad : 0;
        g = std::make_unique<guarded>(((b - 1) * stride + (r - 1) * ld + c) * esz);
    }
    matrix &random()
    {
        for (size_t i = 0; i < g->bytes / esz; ++i) put(g->p, (int64_t)i, dt, value());
        return *this;
    }
    char *p() const { return g->p; }
    double at(int64_t b, int64_t r, int64_t c) const { return get_at(p(), b * stride + r * ld + c, dt); }
};
using outputs = std::vector<matrix *>;

// run(): twice over outputs filled with different bytes
template <class F>
static void twice(const outputs &outs, F run)
{
    std::vector<std::vector<char>> first;
    for (int pass = 0; pass < 2; ++pass) {
        const int fill = pass ? 0x5A : 0xA5;
        for (matrix *m : outs) memset(m->p(), fill, m->g->bytes);
        message.clear();
        const int32_t rc = run();
        scratch.clear();
        CHECK(rc == MI355_OK, "refused: %s", message.c_str());
        for (size_t k = 0; k < outs.size(); ++k) {
            const matrix &m = *outs[k];
            std::vector<char> got(m.p(), m.p() + m.g->bytes);
            if (pass == 0) { first.push_back(got); continue; }
            std::vector<char> mine(got.size(), 0);
            for (int64_t b = 0; b < m.batch; ++b)
                for (int64_t r = 0; r < m.rows; ++r) memset(mine.data() + (b * m.stride + r * m.ld) * m.esz, 1, m.cols * m.esz);
            size_t missed = 0, touched = 0;
            for (size_t i = 0; i < got.size(); ++i) {
                if (mine[i]) missed += got[i] != first[k][i];
                else touched += got[i] != (char)0x5A || first[k][i] != (char)0xA5;
            }
            CHECK(missed == 0 && touched == 0, "output %zu: %zu bytes not written, %zu written between rows", k, missed, touched);
        }
    }
}

static char label[256];
#define CASE(...) do { snprintf(label, sizeof label, __VA_ARGS__); now = label; puts(label); fflush(stdout); } while (0)
static const int32_t FLOATS[] = {MI355_DTYPE_F32, MI355_DTYPE_BF16, MI355_DTYPE_F16};

static void norms(int64_t rows, int64_t cols, int32_t dt, int pad)
{
    CASE("rms_norm %lld x %lld type %d pad %d", (long long)rows, (long long)cols, dt, pad);
    const int32_t wt = cols % 2 ? dt : MI355_DTYPE_F32;
    matrix x(rows, cols, pad, dt), r(rows, cols, pad + 1, dt), w(1, cols, 0, wt), hid(rows, cols, pad + 2, dt), rstd(1, rows, 0, MI355_DTYPE_F32);
    x.random(), r.random(), w.random();
    for (int mode = 0; mode < 3; ++mode) {
        if (mode == 2 && cols % 32) continue;
        const int32_t ot = mode == 0 ? (rows % 2 ? dt : MI355_DTYPE_F32) : mode == 1 ? MI355_DTYPE_F8E4M3 : MI355_DTYPE_F8E5M2;
        matrix out(rows, cols, pad + 3, ot), scales(mode == 2 ? rows : 1, mode == 2 ? cols / 32 : rows, mode == 2 ? pad : 0, mode == 2 ? MI355_DTYPE_UE8M0 : MI355_DTYPE_F32);
        mi355_rms_norm_desc d{rows, cols, x.ld, r.ld, hid.ld, out.ld, scales.ld, 1e-6f, dt, wt, ot, mode == 2 ? 32 : 0, 0};
        outputs outs{&hid, &out, &rstd};
        if (mode) outs.push_back(&scales);
        twice(outs, [&] { return mi355_rms_norm(&ctx, nullptr, &d, x.p(), r.p(), w.p(), hid.p(), out.p(), mode ? scales.p() : nullptr, (float *)rstd.p()); });
        d.ld_residual = d.ld_hidden = 0;
        twice({&out}, [&] { return mi355_rms_norm(&ctx, nullptr, &d, x.p(), nullptr, nullptr, nullptr, out.p(), mode ? scales.p() : nullptr, nullptr); });
    }
    matrix g(rows, cols, pad, dt), s(rows, cols, pad + 1, dt), dx(rows, cols, pad + 2, dt), dw(1, cols, 0, wt);
    g.random(), s.random();
    for (int64_t i = 0; i < rows; ++i) ((float *)rstd.p())[i] = 0.5f;
    mi355_rms_norm_grad_desc gd{rows, cols, g.ld, x.ld, dx.ld, s.ld, dt, wt, wt, 0};
    uint64_t need = 0;
    mi355_rms_norm_grad_workspace_bytes(&gd, &need);
    twice({&dx, &dw}, [&] {
        return mi355_rms_norm_grad(&ctx, nullptr, &gd, g.p(), x.p(), w.p(), (float *)rstd.p(), s.p(), dx.p(), dw.p(), fresh(need), need);
    });
    for (int64_t c = 0; c < cols; c += 1 + cols / 7) {
        double sum = 0, size = 0;
        for (int64_t i = 0; i < rows; ++i) sum += g.at(0, i, c) * x.at(0, i, c) * 0.5, size += fabs(g.at(0, i, c) * x.at(0, i, c) * 0.5);
        CHECK(fabs(dw.at(0, 0, c) - sum) <= size * 1e-4 + fabs(sum) * 0.004 + 1e-6, "grad_weight %g for %g", dw.at(0, 0, c), sum);
    }
    twice({&dx}, [&] { return mi355_rms_norm_grad(&ctx, nullptr, &gd, g.p(), x.p(), nullptr, (float *)rstd.p(), nullptr, dx.p(), nullptr, nullptr, 0); });
}

static void epilogue_gradient(int64_t m, int64_t n, int64_t batch, int32_t dt, int act, int pad, bool in_turn)
{
    CASE("epilogue gradient %lld x %lld x %lld type %d act %d pad %d in turn %d", (long long)batch, (long long)m, (long long)n, dt, act, pad, in_turn);
    matrix g(m, n, pad, dt, batch, in_turn), z(m, n, pad + 1, dt, batch), o(m, n, pad + 2, dt, batch, in_turn);
    g.random(), z.random();
    for (int each = 0; each < (batch > 1 ? 2 : 1); ++each) {
        matrix db(1, n * (each ? batch : 1), 0, each ? dt : MI355_DTYPE_F32);
        mi355_gemm_fused_grad_desc d{m, n, batch, g.ld, z.ld, o.ld, g.stride, z.stride, o.stride, dt, act, each ? dt : MI355_DTYPE_F32, each};
        uint64_t need = 0;
        mi355_gemm_fused_grad_workspace_bytes(&d, &need);
        twice({&o, &db}, [&] { return mi355_gemm_fused_grad(&ctx, nullptr, &d, g.p(), z.p(), o.p(), db.p(), fresh(need), need); });
    }
}

static void lists()
{
    struct shape { int64_t rows, cols, pad; int32_t dt; };
    const std::vector<std::vector<shape>> all = {
        {{1, 1, 0, MI355_DTYPE_F32}}, {{1, CHUNK, 0, MI355_DTYPE_BF16}}, {{1, CHUNK + 1, 0, MI355_DTYPE_F32}, {1, CHUNK - 1, 0, MI355_DTYPE_F16}, {3, 7, 0, MI355_DTYPE_BF16}},
        {{300, 33, 5, MI355_DTYPE_BF16}, {2, CHUNK, 3, MI355_DTYPE_F32}, {2, CHUNK + 9, 1, MI355_DTYPE_F16}, {5000, 3, 1, MI355_DTYPE_F32}, {1, 5 * CHUNK + 3, 0, MI355_DTYPE_BF16}},
        std::vector<shape>(130, {2, 9, 0, MI355_DTYPE_F16}), std::vector<shape>(70, {3, 11, 2, MI355_DTYPE_F32})};
    for (size_t i = 0; i < all.size(); ++i) {
        CASE("list %zu", i);
        std::vector<std::unique_ptr<matrix>> in, out;
        std::vector<mi355_tensor_span> a, b;
        outputs outs;
        for (const shape &s : all[i]) {
            in.push_back(std::make_unique<matrix>(s.rows, s.cols, s.pad, s.dt));
            out.push_back(std::make_unique<matrix>(s.rows, s.cols, s.pad ? s.pad + 1 : 0, s.dt));
            in.back()->random();
            a.push_back({in.back()->p(), (uint64_t)s.rows, (uint64_t)s.cols, (uint64_t)in.back()->ld, s.dt, 0});
            b.push_back({out.back()->p(), (uint64_t)s.rows, (uint64_t)s.cols, (uint64_t)out.back()->ld, s.dt, 0});
            outs.push_back(out.back().get());
        }
        matrix norm(1, 1, 0, MI355_DTYPE_F32);
        outs.push_back(&norm);
        uint64_t need = 0;
        mi355_global_norm_workspace_bytes(&need);
        double sum = 0;
        for (auto &m : in)
            for (int64_t r = 0; r < m->rows; ++r)
                for (int64_t c = 0; c < m->cols; ++c) sum += m->at(0, r, c) * m->at(0, r, c);
        twice(outs, [&] { return mi355_clip_by_global_norm(&ctx, nullptr, a.data(), b.data(), (uint32_t)a.size(), 0.5f, (float *)norm.p(), fresh(need), need); });
        CHECK(fabs(norm.at(0, 0, 0) - sqrt(sum)) <= sqrt(sum) * 1e-6, "norm %g for %g", norm.at(0, 0, 0), sqrt(sum));
        twice({&norm}, [&] { return mi355_global_norm(&ctx, nullptr, a.data(), (uint32_t)a.size(), (float *)norm.p(), fresh(need), need); });
    }
}

struct parts {
    matrix bias, residual, pre, rs, cs;
    mi355_gemm_epilogue ep{};
    parts(int64_t m, int64_t n, int64_t batch, int32_t dt, int act, int pad, bool in_turn)
        : bias(1, n * batch, 0, pad % 2 ? dt : MI355_DTYPE_F32), residual(m, n, pad, dt, batch), pre(m, n, pad + 1, dt, batch, in_turn), rs(1, m * batch, 0, MI355_DTYPE_F32),
          cs(1, n, 0, MI355_DTYPE_F32)
    {
        bias.random(), residual.random(), rs.random(), cs.random();
        ep.bias = bias.p(), ep.residual = residual.p(), ep.pre = pre.p(), ep.row_scale = (float *)rs.p(), ep.col_scale = (float *)cs.p();
        ep.stride_bias = n, ep.ld_residual = residual.ld, ep.stride_residual = residual.stride, ep.ld_pre = pre.ld, ep.stride_pre = pre.stride;
        ep.inc_row_scale = 1, ep.stride_row_scale = m, ep.inc_col_scale = 1;
        ep.activation = act, ep.dtype_bias = bias.dt;
    }
    double z(int64_t b, int64_t i, int64_t j, double product) const { return product * rs.at(0, 0, b * rs.cols / std::max<int64_t>(1, residual.batch) + i) * cs.at(0, 0, j) + bias.at(0, 0, b * cs.cols + j); }
};

static void folds(int64_t m, int64_t n, int64_t batch, uint32_t slabs, int32_t dt, int act)
{
    CASE("fold %u x %lld x %lld x %lld type %d act %d", slabs, (long long)batch, (long long)m, (long long)n, dt, act);
    matrix prod(1, slabs * batch * m * n, 0, MI355_DTYPE_F32), c(m, n, 3, dt, batch);
    parts e(m, n, batch, dt, act, 2, true);
    prod.random();
    twice({&c, &e.pre}, [&] { launch_epilogue(nullptr, (float *)prod.p(), slabs, batch * m * n, make_epilogue(e.ep, dt), c.p(), batch, m, n, c.ld, c.stride); return MI355_OK; });
}

static void edge(int64_t m, int64_t n, int64_t k, int64_t batch, int32_t dt, int32_t ct, int ta, int tb, int act, int pad, int cus)
{
    CASE("edge %lld x %lld x %lld x %lld type %d -> %d layout %d%d act %d pad %d on %d", (long long)batch, (long long)m, (long long)n, (long long)k, dt, ct, ta, tb, act, pad, cus);
    ctx.props.num_streaming_multiprocessors = (uint32_t)cus;
    matrix a(ta ? k : m, ta ? m : k, pad, dt, batch), b(tb ? n : k, tb ? k : n, pad + 1, dt, batch), c(m, n, pad + 2, ct, batch);
    a.random(), b.random();
    parts e(m, n, batch, ct, act, pad, batch > 1);
    mi355_gemm_desc d{};
    d.m = m, d.n = n, d.k = k, d.batch = batch, d.lda = a.ld, d.ldb = b.ld, d.ldc = c.ld, d.stride_a = a.stride, d.stride_b = b.stride, d.stride_c = c.stride;
    d.dtype_ab = dt, d.dtype_c = ct, d.trans_a = ta, d.trans_b = tb;
    if (validate_epilogue(&ctx, d, e.ep, a.p(), b.p(), c.p()) != MI355_OK) { CHECK(false, "refused: %s", message.c_str()); return; }
    twice({&c, &e.pre}, [&] { return launch_gemm_edge(&ctx, nullptr, d, a.p(), b.p(), c.p(), make_epilogue(e.ep, ct)); });
    const double half = ct == MI355_DTYPE_F32 ? 0x1p-24 : ct == MI355_DTYPE_BF16 ? 0x1p-8 : 0x1p-11;
    for (int64_t q = 0; q < batch; ++q)
        for (int64_t i = 0; i < m; i += 1 + m / 9)
            for (int64_t j = 0; j < n; j += 1 + n / 11) {
                double p = 0, size = 0;
                for (int64_t x = 0; x < k; ++x) {
                    const double t = (ta ? a.at(q, x, i) : a.at(q, i, x)) * (tb ? b.at(q, j, x) : b.at(q, x, j));
                    p += t, size += fabs(t);
                }
                const double z = e.z(q, i, j, p), y = act == MI355_ACT_RELU ? (z < 0 ? 0 : z) : act == MI355_ACT_SILU ? z / (1 + exp(-z)) : z, want = y + e.residual.at(q, i, j);
                const double tol = 1e-5 * fabs(e.z(q, i, j, size) - e.z(q, i, j, 0)) + 1e-6 * (fabs(z) + fabs(want) + 1);
                CHECK(fabs(c.at(q, i, j) - want) <= 1.2 * tol + half * fabs(want), "(%lld, %lld) %g for %g", (long long)i, (long long)j, c.at(q, i, j), want);
                CHECK(fabs(e.pre.at(q, i, j) - z) <= tol + half * fabs(z), "argument (%lld, %lld) %g for %g", (long long)i, (long long)j, e.pre.at(q, i, j), z);
            }
}

// the two forms of the tile epilogue on a workgroup's staged blocks, NB blocks of 32 rows a wave, as the kernels of 128 and 256 rows call them
template <int DT_C, int LPR, bool AHEAD, int NB, class ARGS>
static void tile_kernel(ARGS g)
{
    constexpr int RS = LPR * 32 + 16;
    static char stage[4][32 * RS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
    const int64_t row = (int64_t)blockIdx.x * 64 * NB + (wave >> 1) * 32 * NB, col = (int64_t)blockIdx.y * 16 * LPR + (wave & 1) * 8 * LPR;
    tile_finish<DT_C, LPR, AHEAD> fin(epilogue_of<ARGS>(), g, blockIdx.z, row + lane / LPR, col + (lane % LPR) * 8, true);
    fin.template run<NB>([&](auto ib) {
        for (int c = 4 * h; c < 8 * LPR; c += 8)
            for (int e = 0; e < 4; ++e) reinterpret_cast<float *>(stage[wave] + l31 * RS)[c + e] = (float)(row + ib.value * 32 + l31) * 0.01f + (float)(col + c + e) * 0.1f;
    }, stage[wave] + (lane / LPR) * RS + (lane % LPR) * 32, RS);
}
template <int DT_C, int LPR, bool AHEAD, int NB>
static void tiles(int64_t m, int64_t n, int64_t batch, int act, int pad)
{
    CASE("tile %d lanes ahead %d blocks %d: %lld x %lld x %lld type %d act %d pad %d", LPR, AHEAD, NB, (long long)batch, (long long)m, (long long)n, DT_C, act, pad);
    matrix c(m, n, pad, DT_C, batch);
    parts e(m, n, batch, DT_C, act, pad, batch > 1);
    gemm_args g{};
    g.c = c.p(), g.m = m, g.n = n, g.ldc = c.ld, g.stride_c = c.stride;
    typedef with_epilogue<gemm_args> ARGS;
    twice({&c, &e.pre}, [&] {
        emu::launch(tile_kernel<DT_C, LPR, AHEAD, NB, ARGS>, dim3((m + 64 * NB - 1) / (64 * NB), (n + 16 * LPR - 1) / (16 * LPR), batch), dim3(256), add_epilogue(g, make_epilogue(e.ep, DT_C)));
        return MI355_OK;
    });
    const double half = DT_C == MI355_DTYPE_F32 ? 0x1p-24 : DT_C == MI355_DTYPE_BF16 ? 0x1p-8 : 0x1p-11;
    for (int64_t q = 0; q < batch; ++q)
        for (int64_t i = 0; i < m; ++i)
            for (int64_t j = 0; j < n; ++j) {
                const double z = e.z(q, i, j, (double)i * 0.01f + (double)j * 0.1f);
                CHECK(fabs(e.pre.at(q, i, j) - z) <= half * fabs(z) + 1e-5 * (fabs(z) + 1 + (double)(i + j)), "argument (%lld, %lld) %g for %g", (long long)i, (long long)j, e.pre.at(q, i, j), z);
            }
}

int main(int argc, char **argv)
{
    front = argc > 1 && !strcmp(argv[1], "front");
    int turn = 0;
    for (int64_t cols : {1, 7, 8, 31, 32, 33, 96, 512, 513, 1000, 1024, 1025, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16385, 20000, 20480})
        for (int64_t rows : {1, 3, 5}) norms(rows, cols, FLOATS[turn % 3], turn % 4), ++turn;
    for (int64_t cols : {40, 1000, 4096, 8184}) norms(513, cols, FLOATS[turn % 3], turn % 3), ++turn;      // many rows: fewer threads hold a row
    norms(2051, 24, MI355_DTYPE_F32, 1);                                                                   // ... and a thread several of them
    for (int64_t n : {1, 7, 8, 511, 512, 513, 1030})
        for (int64_t m : {1, 3, 5, 64, 261}) epilogue_gradient(m, n, 1 + turn % 3, FLOATS[turn % 3], turn % 5, turn % 4, turn % 2), ++turn;
    epilogue_gradient(4099, 24, 1, MI355_DTYPE_BF16, MI355_ACT_SILU, 1, false);
    lists();
    for (int64_t n : {1, 8, 9, 130})
        for (uint32_t slabs : {1u, 3u, 4u, 6u}) folds(5, n, 1 + turn % 3, slabs, FLOATS[turn % 3], turn % 5), ++turn;
    const int ACTS[] = {MI355_ACT_NONE, MI355_ACT_RELU, MI355_ACT_SILU};
    for (int layout = 0; layout < 4; ++layout)
        for (int32_t dt : FLOATS)
            for (auto [m, n, k] : {std::tuple<int, int, int>{1, 1, 1}, {3, 5, 2}, {31, 33, 7}, {64, 64, 64}, {65, 67, 63}, {70, 130, 65}, {33, 40, 1100}, {130, 129, 72}})
                edge(m, n, k, 1 + turn % 2, dt, turn % 3 ? dt : MI355_DTYPE_F32, layout & 1, layout >> 1, ACTS[turn % 3], turn % 4, m == 130 ? 1 : 256), ++turn;
    for (int64_t n : {1, 8, 63, 64, 127, 136})
        for (int64_t m : {1, 33, 130}) {
            tiles<MI355_DTYPE_F32, 8, false, 2>(m, n, 1 + turn % 2, ACTS[turn % 3], turn % 4);
            tiles<MI355_DTYPE_BF16, 8, false, 1>(m, n, 1, ACTS[turn % 3], turn % 4);
            tiles<MI355_DTYPE_F16, 16, true, 4>(m, n, 1 + turn % 2, ACTS[turn % 3], turn % 4);
            tiles<MI355_DTYPE_F32, 16, true, 4>(m, n, 1, ACTS[turn % 3], turn % 4);
            tiles<MI355_DTYPE_BF16, 16, true, 3>(m, n, 1, ACTS[turn % 3], turn % 4);
            ++turn;
        }
    printf(failures ? "%d failures\n" : "clean\n", failures);
    return failures != 0;
}
