"""Calls that the operators around a linear layer once answered wrongly, or accepted and should not have, without a device: the host side on
the fake HIP runtime, as in tests/test_linear_ops_cpu.py.  Their GPU side is tests/test_gpu_linear_ops_mends.py."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from cubecl_amd import ElemType, TensorHandle, ops
from cubecl_amd import _native as N
from test_linear_ops_cpu import client, lib, log, make, refused  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]
F32, BF16, F16, E4M3, UE8M0 = ElemType.F32, ElemType.BF16, ElemType.F16, ElemType.F8E4M3, ElemType.UE8M0


# ---- a batch's rows as one matrix -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,strides", [
    ((3, 8, 16), (128, 16, 1)), ((3, 8, 16), (0, 0, 1)), ((3, 8, 16), (0, 16, 1)), ((3, 8, 16), (16, 0, 1)), ((3, 8, 16), (128, 1, 8)), ((3, 8, 16), (64, 8, 1)),
    ((3, 1, 16), (16, 0, 1)), ((3, 1, 16), (20, 1, 1)), ((1, 8, 16), (0, 20, 1)), ((2, 3, 8, 16), (480, 160, 20, 1)), ((2, 3, 8, 16), (160, 320, 20, 1)), ((3, 8, 1), (24, 3, 7)),
    ((3, 8, 1), (0, 0, 0)), ((1, 1, 16), (0, 0, 1)), ((0, 8, 16), (128, 16, 1))])
def test_a_batch_as_rows_is_the_same_elements(client, monkeypatch, shape, strides):  # noqa: F811
    """Every element of the one matrix lies where the view has it, whichever axes are broadcast, overlap or have one entry."""
    copied = []

    def copy(_, t):
        copied.append(t)
        return make(client, t.shape, t.dtype)

    monkeypatch.setattr(ops, "into_contiguous", copy)
    t = make(client, shape, F32, strides)
    got = ops._as_rows(client, t)
    assert got.shape == (int(np.prod(shape[:-1])), shape[-1])
    places = lambda shape, strides: np.array([int(np.dot(i, strides)) for i in np.ndindex(*shape)])      # noqa: E731
    want = places(shape, make(client, shape).strides if copied else strides)
    assert np.array_equal(places(got.shape, got.strides), want)
    assert got.shape[0] <= 1 or got.strides[0] >= got.shape[1]


# ---- a batch of no entries --------------------------------------------------------------------------------------------------------
def test_gradients_of_shared_operands_over_an_empty_batch_are_written(client, monkeypatch):  # noqa: F811
    """The sum over no entries is zeros: a product without a K axis, not whatever the memory held."""
    done = []
    monkeypatch.setattr(ops, "matmul", lambda c, a, b, out, acc=None: done.append((a.shape, b.shape, out.shape, acc)))
    monkeypatch.setattr(ops, "copy_into", lambda c, a, out: done.append((a.shape, out.shape)))
    g, d = make(client, (0, 4, 6)), make(client, (0, 4, 6))
    a, b, da, db = make(client, (4, 5)), make(client, (5, 6)), make(client, (4, 5)), make(client, (5, 6))
    ops.matmul_fused_backward(client, g, None, d, lhs=a, rhs=b, grad_lhs=da, grad_rhs=db)
    assert done == [((4, 0), (0, 5), (4, 5), None), ((4, 5), (4, 5)), ((5, 0), (0, 6), (5, 6), None), ((5, 6), (5, 6))]


def test_a_bias_gradient_of_no_entries_is_not_written(client):  # noqa: F811
    """[0, n]: one bias for each of no entries holds nothing, unlike [n], which is the sum over none."""
    ops.matmul_fused_backward(client, make(client, (0, 4, 6)), None, make(client, (0, 4, 6)), grad_bias=make(client, (0, 6)))
    assert log(client)["fold"] == 0
    ops.matmul_fused_backward(client, make(client, (0, 4, 6)), None, make(client, (0, 4, 6)), grad_bias=make(client, (6,)))
    ops.matmul_fused_backward(client, make(client, (3, 0, 6)), None, make(client, (3, 0, 6)), grad_bias=make(client, (3, 6)))
    assert log(client)["fold"] == 2


# ---- launch limits ------------------------------------------------------------------------------------------------------------------
GEOMETRY = r"""
#include "../../cubecl_amd/csrc/linear_ops.hpp"
#include <cstdio>
using namespace mi355;
int main()
{
    for (int64_t cols : {1ll, 63ll, 64ll, 65ll, 1ll << 20, (1ll << 27) - 1, 1ll << 27, (1ll << 27) + 1, 1ll << 28, (1ll << 30) + 7, 1ll << 31})
        for (int64_t batch : {1ll, 2ll, 65535ll, 70000ll}) {
            int64_t done = 0;
            each_fold_launch(cols, batch, [&](int64_t c, int64_t wide, int64_t b, int64_t entries) {
                const int64_t here = std::min(wide * FOLD_COLS, cols - c);
                if (wide * 1024 * entries >= 1ll << 32 || entries > 65535 || b + entries > batch || c + (wide - 1) * FOLD_COLS >= cols) printf("fold %lld %lld\n", (long long)cols, (long long)batch);
                done += here * entries;
            });
            if (done != cols * batch) printf("fold covers %lld of %lld x %lld\n", (long long)done, (long long)cols, (long long)batch);
        }
    for (int64_t cols : {1ll, 512ll, 16385ll, 1ll << 27, 1ll << 29, (long long)GRAD_MAX_COLS})
        for (int64_t rows : {1ll, 3ll, 600ll, 1ll << 20}) {
            const row_shape sh = grad_shape_for(rows, cols);
            const int64_t wgs = norm_grad_partials(rows, cols), threads = sh.threads ? std::max(sh.threads, 256) * wgs : (cols + 2047) / 2048 * 256 * wgs;
            if (wgs < 1 || wgs > rows || threads >= 1ll << 32) printf("grad %lld %lld\n", (long long)rows, (long long)cols);
            if (sh.threads && (int64_t)sh.threads * sh.pieces * 8 < cols) printf("shape %lld %lld\n", (long long)rows, (long long)cols);
            const row_shape f = shape_for(rows, cols);
            if (f.threads && (int64_t)f.threads * f.pieces * 8 < cols) printf("forward shape %lld %lld\n", (long long)rows, (long long)cols);
        }
    for (int64_t cols = 1; cols <= 16384; ++cols)          // every row length that registers hold is held
        for (int64_t rows : {1ll, 512ll, 513ll}) {
            const row_shape f = shape_for(rows, cols), g = grad_shape_for(rows, cols);
            if ((int64_t)f.threads * f.pieces * 8 < cols || (int64_t)g.threads * g.pieces * 8 < cols) printf("registers %lld\n", (long long)cols);
        }
    puts("done");
}
"""


def test_launches_stay_below_the_thread_limit_and_cover_every_column(tmp_path):
    src, exe = tmp_path / "geometry.cpp", tmp_path / "geometry"
    src.write_text(GEOMETRY.replace("../../cubecl_amd", str(ROOT / "cubecl_amd")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", str(ROOT / "tests" / "fake_hip"), "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "done\n"


def test_norm_gradient_refuses_more_columns_than_its_launches_hold(client):  # noqa: F811
    need, d = C.c_uint64(), N.RmsNormGradDesc(rows=1, cols=(1 << 31) + 1, ld_out=1 << 32, ld_hidden=1 << 32, ld_in=1 << 32, dtype=BF16, dtype_weight=BF16, dtype_grad_weight=F32)
    assert client.lib.mi355_rms_norm_grad_workspace_bytes(C.byref(d), C.byref(need)) == N.E_INVALID_ARGUMENT
    held = make(client, (64,))
    p = held.device_ptr()
    assert client.lib.mi355_rms_norm_grad(client.ctx, None, C.byref(d), p, p, None, p, None, p, None, None, 0) == N.E_INVALID_ARGUMENT
    assert log(client)["norm_grad"] == 0


# ---- which calls share memory -------------------------------------------------------------------------------------------------------
SPANS = r"""
#include "ROOT/cubecl_amd/csrc/row_span.hpp"
#include <cstdio>
#include <random>
#include <vector>
using namespace mi355;
struct set { int64_t at, rows, cols, ld, batch, stride; };
static char base[1];
static std::vector<char> bytes(const set &s, int64_t esz)
{
    std::vector<char> v(4096, 0);
    for (int64_t b = 0; b < s.batch; ++b)
        for (int64_t r = 0; r < s.rows; ++r)
            for (int64_t k = 0; k < s.cols * esz; ++k) v[s.at + (b * s.stride + r * s.ld) * esz + k] = 1;
    return v;
}
int main()
{
    std::mt19937 g(7);
    auto upto = [&](int64_t lo, int64_t hi) { return lo + (int64_t)(g() % (uint64_t)(hi - lo + 1)); };
    int apart = 0, exact = 0, same = 0;
    for (int t = 0; t < 200000; ++t) {
        const int64_t esz = 1 << upto(0, 2), ld = upto(1, 12), stride = upto(0, 40);
        auto one = [&](bool alike) {
            set s{upto(0, 60), upto(0, 4), upto(0, 5), alike ? ld : upto(0, 12), upto(0, 3), alike ? stride : upto(0, 40)};
            if (alike && t % 3 == 0) std::swap(s.ld, s.stride);
            return s;
        };
        const bool alike = t & 1;
        const set a = one(alike), b = t % 16 == 3 ? a : one(alike);
        const row_span x = span_of(base + a.at, a.rows, a.cols, a.ld, esz, a.batch, a.stride), y = span_of(base + b.at, b.rows, b.cols, b.ld, esz, b.batch, b.stride);
        const std::vector<char> p = bytes(a, esz), q = bytes(b, esz);
        bool meet = false, equal = p == q;
        for (size_t i = 0; i < p.size(); ++i) meet = meet || (p[i] && q[i]);
        const int rel = spans_relation(x, y);
        if (meet && rel == SPANS_APART) { puts("a shared byte was missed"); return 0; }
        if (rel == SPANS_SAME && !equal) { puts("not the same bytes"); return 0; }
        if (alike && !meet && rel != SPANS_APART) { puts("apart, and taken as overlapping"); return 0; }
        if (spans_relation(y, x) != rel) { puts("one way is not the other"); return 0; }
        apart += rel == SPANS_APART && x.row_bytes && y.row_bytes; exact += alike && !meet; same += rel == SPANS_SAME;
    }
    printf(apart > 1000 && exact > 1000 && same > 1000 ? "done\n" : "too few of a kind: %d %d %d\n", apart, exact, same);
}
"""


def test_shared_bytes_are_seen_in_random_row_sets(tmp_path):
    """Against the bytes themselves: no overlap is missed, and sets that step by the same distances are told apart exactly."""
    src, exe = tmp_path / "spans.cpp", tmp_path / "spans"
    src.write_text(SPANS.replace("ROOT", str(ROOT)))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "done\n"


def in_turn(client, handle, m, n, batch, dt=F32, at=0, width=None):  # noqa: F811
    """[batch, m, n] stored [m][batch][width]."""
    width = width or n
    return TensorHandle.new(handle.offset_start_by(at * dt.size()), (batch, m, n), (width, batch * width, 1), dt)


def test_outputs_on_interleaved_operands_are_refused(client):  # noqa: F811
    m, n, k, batch = 4, 8, 8, 3
    buf = client.empty(4 * (m * n * batch + 64))
    lhs, rhs, out = in_turn(client, buf, m, k, batch), make(client, (k, n)), make(client, (batch, m, n))
    # (the C entry: ops.matmul_fused copies such an lhs first)
    d = N.GemmDesc(m=m, n=n, k=k, batch=batch, lda=batch * k, ldb=n, ldc=n, stride_a=k, stride_c=m * n, dtype_ab=F32, dtype_c=F32)
    call = lambda c: client.lib.mi355_gemm_fused(client.ctx, None, C.byref(d), C.byref(N.GemmEpilogue()), lhs.device_ptr(), rhs.device_ptr(), c)      # noqa: E731
    assert call(out.device_ptr()) == N.OK
    assert [call(buf.offset_start_by(at).device_ptr()) for at in (0, 8, 4 * n)] == [N.E_INVALID_ARGUMENT] * 3
    refused(ops.matmul_fused, client, make(client, (batch, m, k)), rhs, out, residual=in_turn(client, out.handle, m, n, batch), match="overlaps")
    refused(ops.matmul_fused, client, make(client, (batch, m, k)), rhs, out, residual=lhs, pre_activation=in_turn(client, buf, m, n, batch, at=4), match="overlaps")
    log(client, clear=True)
    # the gradient's pass: in place is in place, anything else on its operands is not
    g = in_turn(client, buf, m, n, batch)
    ops.matmul_fused_backward(client, g, None, g)
    refused(ops.matmul_fused_backward, client, g, None, in_turn(client, buf, m, n, batch, at=2), match="overlaps")
    refused(ops.matmul_fused_backward, client, g, None, make(client, (batch, m, n), F32, None, buf), match="overlaps")
    square = client.empty(4 * 3 * 3 * n)
    a, b = make(client, (3, 3, n), F32, None, square), in_turn(client, square, 3, n, 3)
    refused(ops.matmul_fused_backward, client, a, None, b, match="overlaps")      # the same bytes, entries and rows exchanged
    assert log(client)["fused_grad"] == 1


def test_interleaved_entries_and_parts_of_one_tensor_are_taken(client):  # noqa: F811
    m, n, k, batch = 4, 8, 5, 3
    a, b, out = make(client, (batch, m, k)), make(client, (k, n)), make(client, (batch, m, n))
    whole = client.empty(4 * m * batch * 3 * n)
    q, r, s = (in_turn(client, whole, m, n, batch, at=i * n, width=3 * n) for i in range(3))
    ops.matmul_fused(client, a, b, out, activation="silu", pre_activation=in_turn(client, client.empty(4 * m * n * batch), m, n, batch))
    ops.matmul_fused(client, a, b, out, activation="silu", pre_activation=q, residual=r)
    ops.matmul_fused_backward(client, q, r, s, activation="silu")
    ops.matmul_fused_backward(client, q, r, r, activation="silu")
    # a column of scales beside an output in the same rows
    wide = client.empty(4 * m * (n + 1))
    ops.matmul_fused(client, make(client, (m, k)), b, make(client, (m, n), F32, (n + 1, 1), wide), lhs_scale=make(client, (m,), F32, (n + 1,), wide.offset_start_by(4 * n)))
    assert log(client)["epilogue"] == 3 and log(client)["fused_grad"] == 2
    refused(ops.matmul_fused, client, make(client, (m, k)), b, make(client, (m, n), F32, (n + 1, 1), wide),
            lhs_scale=make(client, (m,), F32, (n + 1,), wide.offset_start_by(4 * n - 4)), match="overlaps")
    # entries that do share memory
    for stride, ld in ((n - 1, batch * n), (n, batch * n - 1), (0, n)):
        refused(ops.matmul_fused, client, a, b, out, pre_activation=make(client, (batch, m, n), F32, (stride, ld, 1)), code=N.E_UNSUPPORTED_STRIDES)
        refused(ops.matmul_fused_backward, client, out, None, make(client, (batch, m, n), F32, (stride, ld, 1)), code=N.E_UNSUPPORTED_STRIDES)


# ---- alignment and missing operands ---------------------------------------------------------------------------------------------------
def test_pointers_off_their_element_are_refused(client):  # noqa: F811
    """Each operand of the C entry points half an element off, the others as they should be; one element off is fine."""
    held = [make(client, (64,), F32) for _ in range(8)]
    p = [t.device_ptr() for t in held]
    d = N.RmsNormDesc(rows=2, cols=8, ld_in=8, ld_residual=8, ld_hidden=8, ld_out=8, eps=1e-6, dtype=BF16, dtype_weight=F32, dtype_out=BF16)
    norm = lambda off, d=d: client.lib.mi355_rms_norm(client.ctx, None, C.byref(d), *[x + o for x, o in zip(p, off)][:5], p[5] + off[5] if d.dtype_out == E4M3 else None, p[6] + off[6])      # noqa: E731
    assert norm([2, 2, 4, 2, 2, 0, 4]) == N.OK
    for i, o in enumerate((1, 1, 2, 1, 1, None, 2)):
        assert o is None or norm([o if j == i else 0 for j in range(7)]) == N.E_INVALID_ARGUMENT, i
    d8 = N.RmsNormDesc(rows=2, cols=8, ld_in=8, ld_residual=8, ld_hidden=8, ld_out=8, eps=1e-6, dtype=BF16, dtype_weight=F32, dtype_out=E4M3)
    assert norm([0, 0, 0, 0, 1, 4, 0], d8) == N.OK and norm([0, 0, 0, 0, 1, 2, 0], d8) == N.E_INVALID_ARGUMENT
    g = N.RmsNormGradDesc(rows=2, cols=8, ld_out=8, ld_hidden=8, ld_in=8, ld_stream=8, dtype=BF16, dtype_weight=F32, dtype_grad_weight=F32)
    need = C.c_uint64()
    assert client.lib.mi355_rms_norm_grad_workspace_bytes(C.byref(g), C.byref(need)) == N.OK
    ws = client.empty(need.value)
    grad = lambda off: client.lib.mi355_rms_norm_grad(client.ctx, None, C.byref(g), *[x + o for x, o in zip(p, off)], ws.device_ptr(), need.value)      # noqa: E731
    assert grad([2, 2, 4, 4, 2, 2, 4]) == N.OK
    for i, o in enumerate((1, 1, 2, 2, 1, 1, 2)):
        assert grad([o if j == i else 0 for j in range(7)]) == N.E_INVALID_ARGUMENT, i
    f = N.GemmFusedGradDesc(m=2, n=8, batch=1, ld_out=8, ld_pre=8, ld_grad=8, dtype=BF16, activation=N.ACT_SILU, dtype_bias=F32)
    assert client.lib.mi355_gemm_fused_grad_workspace_bytes(C.byref(f), C.byref(need)) == N.OK
    ws = client.empty(need.value)
    fused = lambda off: client.lib.mi355_gemm_fused_grad(client.ctx, None, C.byref(f), *[x + o for x, o in zip(p, off)], ws.device_ptr(), need.value)      # noqa: E731
    assert fused([2, 2, 2, 4]) == N.OK
    for i, o in enumerate((1, 1, 1, 2)):
        assert fused([o if j == i else 0 for j in range(4)]) == N.E_INVALID_ARGUMENT, i
    spans, ws = ops.TensorList([make(client, (8,))]).spans, client.empty(1 << 16)
    assert client.lib.mi355_global_norm(client.ctx, None, spans, 1, p[0] + 2, ws.device_ptr(), 1 << 16) == N.E_INVALID_ARGUMENT
    got = log(client)
    assert (got["norm"], got["norm_grad"], got["fused_grad"], got["sums"]) == (2, 1, 1, 0)


def test_missing_operands_are_refused(client):  # noqa: F811
    g, w, r, dx = make(client, (5, 64), F16), make(client, (64,), F16), make(client, (5,)), make(client, (5, 64), F16)
    refused(ops.rms_norm_backward, client, g, g, w, None, dx, match="NULL")
    refused(ops.rms_norm_backward, client, g, None, w, r, dx, match="NULL")
    refused(ops.global_norm, client, [g], None, match="NULL")
    assert log(client)["norm_grad"] == 0 and log(client)["sums"] == 0
