"""What the operators around a linear layer refuse, and how they cut their work, without a device: cubecl_amd/csrc/linear_ops.cpp and the host
runtime on the fake HIP runtime (tests/fake_hip/), launches counted instead of made.  The same entry points run on the MI355X in
tests/test_gpu_linear_ops.py."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from cubecl_amd import ElemType, ServerError, TensorHandle, ops
from cubecl_amd import _native as N
from cubecl_amd.runtime import ComputeClient, DeviceId, _Server

ROOT = Path(__file__).resolve().parents[1]
FAKE, CSRC = ROOT / "tests" / "fake_hip", ROOT / "cubecl_amd" / "csrc"
F32, BF16, F16, E4M3, E5M2, UE8M0 = ElemType.F32, ElemType.BF16, ElemType.F16, ElemType.F8E4M3, ElemType.F8E5M2, ElemType.UE8M0
LOG = ("norm", "norm_grad", "fold", "epilogue", "fused_grad", "sums", "scale", "finish", "chunks", "partials")


def build_lib() -> Path:
    so = FAKE / "liblinearopstest.so"
    srcs = [CSRC / "runtime.cpp", CSRC / "pool.cpp", CSRC / "comm.cpp", CSRC / "linear_ops.cpp", FAKE / "fake_hip.cpp", FAKE / "fake_linear_kernels.cpp"]
    deps = srcs + [CSRC / "internal.hpp", CSRC / "linear_ops.hpp", FAKE / "hip" / "hip_runtime.h", ROOT / "include" / "mi355cube.h", Path(__file__)]
    if not so.exists() or so.stat().st_mtime < max(d.stat().st_mtime for d in deps):
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-format-truncation", "-DFAKE_WITH_RUNTIME", "-shared", "-fPIC", "-Wl,-Bsymbolic",
                        "-I", str(FAKE), "-o", str(so)] + [str(s) for s in srcs] + ["-ldl"], check=True)
    return so


@pytest.fixture(scope="module")
def lib():
    lib = C.CDLL(str(build_lib()))
    for name, (restype, argtypes) in N.PROTOTYPES.items():
        if hasattr(lib, name):
            getattr(lib, name).restype, getattr(lib, name).argtypes = restype, argtypes
    lib.faketest_set_device.argtypes = [C.c_char_p, C.c_int32, C.c_int32]
    lib.pooltest_set_capacity.argtypes = [C.c_uint64]
    lib.lineartest_log.argtypes = [C.POINTER(C.c_uint64), C.c_int32]
    lib.lineartest_log.restype = None
    return lib


@pytest.fixture()
def client(lib):
    lib.faketest_set_device(b"gfx950:sramecc+:xnack-", 64, 1)
    lib.pooltest_set_capacity(288 << 30)
    server = _Server(DeviceId(0, 0), lib=lib)
    client = ComputeClient(server)
    log(client, clear=True)
    yield client
    server.close()


def log(client, clear=False):
    out = (C.c_uint64 * len(LOG))()
    client.lib.lineartest_log(out, int(clear))
    return dict(zip(LOG, out))


def make(client, shape, dtype=F32, strides=None, handle=None):
    n = sum((d - 1) * s for d, s in zip(shape, strides)) + 1 if strides and np.prod(shape) else int(np.prod(shape))
    handle = handle or client.empty(max(n, 1) * dtype.size())
    if strides is None:
        return TensorHandle.new_contiguous(shape, handle, dtype)
    return TensorHandle.new(handle, shape, strides, dtype)


def refused(fn, *args, code=N.E_INVALID_ARGUMENT, match=None, **kw):
    with pytest.raises(ServerError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value


# ---- matmul_fused -----------------------------------------------------------------------------------------------------------------
def fused_operands(client, m=4, n=6, k=5, dt=BF16):
    return make(client, (m, k), dt), make(client, (k, n), dt), make(client, (m, n), dt)


def test_fused_takes_what_it_documents(client):
    a, b, c = fused_operands(client)
    ops.matmul_fused(client, a, b, c)
    ops.matmul_fused(client, a, b, c, bias=make(client, (6,), F32), activation="silu", residual=c, pre_activation=make(client, (4, 6), BF16),
                     lhs_scale=make(client, (4,)), rhs_scale=make(client, (1,)))
    # residual and output as column ranges of one wider matrix
    wide = client.empty(4 * 12 * 2)
    left, right = make(client, (4, 6), BF16, (12, 1), wide), make(client, (4, 6), BF16, (12, 1), wide.offset_start_by(12))
    ops.matmul_fused(client, a, b, left, residual=right)
    assert log(client)["epilogue"] == 3
    # nothing to do
    ops.matmul_fused(client, make(client, (0, 5), BF16), b, make(client, (0, 6), BF16))
    assert log(client)["epilogue"] == 3


def test_fused_refusals(client):
    a, b, c = fused_operands(client)
    go = lambda **kw: refused(ops.matmul_fused, client, a, b, c, **kw)
    refused(ops.matmul_fused, client, a, b, make(client, (4, 7), BF16))
    refused(ops.matmul_fused, client, a, make(client, (5, 6), F16), c)
    go(activation="swish", code=N.E_UNSUPPORTED)
    go(bias=make(client, (5,), F32))
    go(bias=make(client, (1,), F32))                        # one value for six columns
    go(bias=make(client, (6,), F16), code=N.E_UNSUPPORTED)
    go(bias=make(client, (3, 6), F32))                      # a batch of three for one matrix
    go(residual=make(client, (4, 6), F32))
    go(residual=make(client, (1, 6), BF16))
    go(pre_activation=make(client, (6, 4), BF16))
    go(lhs_scale=make(client, (3,)))
    go(lhs_scale=make(client, (4,), BF16))
    go(rhs_scale=make(client, (7,)))
    go(pre_activation=c, match="overlaps")
    pre = make(client, (4, 6), BF16)
    go(residual=pre, pre_activation=pre, match="overlaps")
    shifted = client.empty(4 * 6 * 2 + 2)
    refused(ops.matmul_fused, client, a, b, make(client, (4, 6), BF16, handle=shifted), residual=make(client, (4, 6), BF16, handle=shifted.offset_start_by(2)), match="overlaps")
    refused(ops.matmul_fused, client, a, b, make(client, (4, 6), BF16, handle=b.handle), match="overlaps an operand")
    refused(ops.matmul_fused, client, a, b, make(client, (4, 6), BF16, (1, 4)), code=N.E_UNSUPPORTED_STRIDES)
    ep = N.GemmEpilogue(activation=9)
    d = N.GemmDesc(m=4, n=6, k=5, batch=1, lda=5, ldb=6, ldc=6, dtype_ab=BF16, dtype_c=BF16)
    assert client.lib.mi355_gemm_fused(client.ctx, None, C.byref(d), C.byref(ep), a.device_ptr(), b.device_ptr(), c.device_ptr()) == N.E_UNSUPPORTED
    ep = N.GemmEpilogue(residual=c.device_ptr() + 1, ld_residual=6)
    assert client.lib.mi355_gemm_fused(client.ctx, None, C.byref(d), C.byref(ep), a.device_ptr(), b.device_ptr(), c.device_ptr()) == N.E_INVALID_ARGUMENT
    ep = N.GemmEpilogue(bias=pre.device_ptr(), stride_bias=-6, dtype_bias=BF16)
    assert client.lib.mi355_gemm_fused(client.ctx, None, C.byref(d), C.byref(ep), a.device_ptr(), b.device_ptr(), c.device_ptr()) == N.E_UNSUPPORTED_STRIDES
    assert client.lib.mi355_gemm_fused(client.ctx, None, C.byref(d), None, a.device_ptr(), b.device_ptr(), c.device_ptr()) == N.E_INVALID_ARGUMENT
    assert log(client)["epilogue"] == 0


def test_fused_batches(client):
    a, b, c = make(client, (3, 4, 5)), make(client, (5, 6)), make(client, (3, 4, 6))
    ops.matmul_fused(client, a, b, c, bias=make(client, (3, 6)), lhs_scale=make(client, (3, 4)), residual=c)
    refused(ops.matmul_fused, client, a, b, c, bias=make(client, (2, 6)))
    refused(ops.matmul_fused, client, a, make(client, (2, 5, 6)), c)
    # a residual that all entries share is not the output
    refused(ops.matmul_fused, client, a, b, c, residual=make(client, (3, 4, 6), F32, (0, 6, 1), c.handle), match="overlaps")
    # entries of an output that share memory
    refused(ops.matmul_fused, client, a, b, c, pre_activation=make(client, (3, 4, 6), F32, (0, 6, 1)), code=N.E_UNSUPPORTED_STRIDES)


# ---- its gradient -----------------------------------------------------------------------------------------------------------------
def test_fused_backward_refusals(client):
    g, z, d = make(client, (4, 6), BF16), make(client, (4, 6), BF16), make(client, (4, 6), BF16)
    ops.matmul_fused_backward(client, g, z, d, activation="gelu", grad_bias=make(client, (6,)))
    ops.matmul_fused_backward(client, g, None, d)
    ops.matmul_fused_backward(client, g, z, g, activation="relu")               # in place
    ops.matmul_fused_backward(client, g, z, None, activation="relu", grad_bias=make(client, (6,), BF16))
    assert log(client)["fused_grad"] == 4 and log(client)["fold"] == 2
    log(client, clear=True)
    f = lambda *args, **kw: refused(ops.matmul_fused_backward, client, *args, **kw)
    f(g, None, d, activation="gelu")
    f(g, make(client, (4, 6), F16), d, activation="gelu")
    f(g, z, make(client, (6, 4), BF16), activation="gelu")
    f(g, z, d, activation="tanh", code=N.E_UNSUPPORTED)
    f(g, z, d, activation="relu", grad_bias=make(client, (4,)))
    f(g, z, d, activation="relu", grad_bias=make(client, (6,), F16), code=N.E_UNSUPPORTED)
    f(g, z, d, activation="relu", grad_bias=make(client, (2, 6)))
    f(g, z, None, activation="relu", grad_lhs=make(client, (4, 5), BF16), rhs=make(client, (5, 6), BF16))
    f(g, z, d, activation="relu", grad_lhs=make(client, (4, 5), BF16))
    f(g, z, d, activation="relu", grad_lhs=make(client, (4, 5), BF16), rhs=make(client, (7, 6), BF16))
    f(g, z, d, activation="relu", grad_rhs=make(client, (5, 6), F16), lhs=make(client, (4, 5), BF16))
    f(g, z, d, activation="relu", grad_rhs=make(client, (5, 6), BF16), lhs=make(client, (3, 5), BF16))
    f(make(client, (6,), BF16), None, None)
    buf = client.empty(4 * 6 * 2 + 2)
    f(make(client, (4, 6), BF16, handle=buf), None, make(client, (4, 6), BF16, handle=buf.offset_start_by(2)), match="overlaps")
    desc = N.GemmFusedGradDesc(m=4, n=6, batch=1, ld_out=6, ld_pre=6, ld_grad=6, dtype=BF16, activation=1, dtype_bias=F32)
    need = C.c_uint64()
    assert client.lib.mi355_gemm_fused_grad_workspace_bytes(C.byref(desc), C.byref(need)) == N.OK and need.value >= 24
    ws, bias = client.empty(need.value), make(client, (6,))
    call = lambda b, w, nb: client.lib.mi355_gemm_fused_grad(client.ctx, None, C.byref(desc), g.device_ptr(), z.device_ptr(), d.device_ptr(), b, w, nb)
    assert call(bias.device_ptr(), ws.device_ptr(), need.value - 1) == N.E_INVALID_ARGUMENT
    assert call(bias.device_ptr(), None, need.value) == N.E_INVALID_ARGUMENT
    assert call(ws.device_ptr(), ws.device_ptr(), need.value) == N.E_INVALID_ARGUMENT
    assert log(client)["fused_grad"] == 0
    desc.batch = -1
    assert client.lib.mi355_gemm_fused_grad_workspace_bytes(C.byref(desc), C.byref(need)) == N.E_INVALID_ARGUMENT


def test_fused_backward_refuses_outputs_on_what_a_later_launch_reads(client):
    """grad_lhs is complete before grad_rhs reads lhs, and grad_pre before either product reads the operands."""
    m, n, k = 4, 6, 5
    g, d = make(client, (m, n), BF16), make(client, (m, n), BF16)
    a, b, da, db = make(client, (m, k), BF16), make(client, (k, n), BF16), make(client, (m, k), BF16), make(client, (k, n), BF16)
    f = lambda pre, **kw: refused(ops.matmul_fused_backward, client, g, None, pre, match="overlaps", **{**dict(lhs=a, rhs=b, grad_lhs=da, grad_rhs=db), **kw})
    f(d, grad_lhs=a)
    f(d, grad_rhs=b)
    f(d, grad_lhs=d, lhs=make(client, (m, n), BF16), rhs=make(client, (n, n), BF16), grad_rhs=None)
    f(d, grad_rhs=make(client, (k, n), BF16, handle=da.handle))
    f(d, grad_bias=make(client, (n,), BF16, handle=b.handle))
    f(make(client, (m, n), BF16, handle=client.empty(256)), lhs=make(client, (m, k), BF16, (20, 1), d.handle), grad_lhs=make(client, (m, k), BF16, (20, 1), d.handle))
    assert log(client)["fused_grad"] == 0
    # column ranges of one wider matrix lie beside each other
    wide = client.empty(m * 20 * 2)
    left, right = TensorHandle.new(wide, (m, k), (20, 1), BF16), TensorHandle.new(wide.offset_start_by(2 * k), (m, k), (20, 1), BF16)
    assert not ops._meshed(left, right, 2 * k) and not ops._meshed(right, left, -2 * k)
    assert ops._meshed(left, right, 2 * k - 2) and ops._meshed(right, left, 2 - 2 * k)


@pytest.mark.parametrize("m,n,batch", [(1, 1, 1), (4096, 8192, 1), (100000, 8, 1), (3, 100001, 1), (17, 40, 65535), (1 << 20, 512, 2)])
def test_fused_backward_workspace_covers_its_slabs(client, m, n, batch):
    desc = N.GemmFusedGradDesc(m=m, n=n, batch=batch, ld_out=n, ld_pre=n, ld_grad=n, dtype=BF16, dtype_bias=F32)
    need = C.c_uint64()
    assert client.lib.mi355_gemm_fused_grad_workspace_bytes(C.byref(desc), C.byref(need)) == N.OK
    assert need.value % (4 * n * batch) == 0 and 1 <= need.value // (4 * n * batch) <= min(256, m)


# ---- rms_norm ---------------------------------------------------------------------------------------------------------------------
def test_rms_norm_takes_what_it_documents(client):
    x, w = make(client, (3, 5, 64), BF16), make(client, (64,), BF16)
    ops.rms_norm(client, x, w, make(client, (3, 5, 64), BF16), rstd=make(client, (3, 5)))
    ops.rms_norm(client, x, None, make(client, (3, 5, 64), F32), residual=x, residual_out=x)
    ops.rms_norm(client, x, make(client, (64,)), x)                                     # in place
    ops.rms_norm(client, x, w, make(client, (3, 5, 64), E4M3), scales=make(client, (3, 5)))
    ops.rms_norm(client, x, w, make(client, (3, 5, 64), E5M2), scales=make(client, (3, 5, 2), UE8M0))
    ops.rms_norm(client, make(client, (15, 64), BF16, (80, 1)), w, make(client, (15, 64), BF16, (72, 1)))
    assert log(client)["norm"] == 6
    ops.rms_norm(client, make(client, (0, 64), BF16), w, make(client, (0, 64), BF16))
    ops.rms_norm(client, make(client, (4, 0), BF16), None, make(client, (4, 0), BF16))
    assert log(client)["norm"] == 6


def test_rms_norm_refusals(client):
    x, w, y = make(client, (5, 64), BF16), make(client, (64,), BF16), make(client, (5, 64), BF16)
    f = lambda *args, **kw: refused(ops.rms_norm, client, *args, **kw)
    f(make(client, (5, 64), ElemType.I32), w, y, code=N.E_UNSUPPORTED)
    f(x, w, make(client, (64, 5), BF16))
    f(x, w, make(client, (5, 64), F16), code=N.E_UNSUPPORTED)
    f(x, make(client, (63,), BF16), y)
    f(x, make(client, (64,), F16), y)
    for eps in (0.0, -1e-6, float("nan"), float("inf")):
        f(x, w, y, eps=eps)
    f(x, w, y, residual=make(client, (4, 64), BF16))
    f(x, w, y, residual_out=make(client, (5, 64), F32))
    f(x, w, y, rstd=make(client, (4,)))
    f(x, w, y, rstd=make(client, (5,), BF16))
    f(x, w, y, scales=make(client, (5,)))
    q = make(client, (5, 64), E4M3)
    f(x, w, q)
    f(x, w, q, scales=make(client, (5,), BF16))
    f(x, w, q, scales=make(client, (5, 3), UE8M0))
    x48 = make(client, (5, 48), BF16)
    f(x48, None, make(client, (5, 48), E4M3), scales=make(client, (5, 1), UE8M0))       # 48 columns are not whole blocks
    f(x, w, y, residual_out=y, match="outputs overlap")
    buf = client.empty(5 * 64 * 2 + 2)
    f(make(client, (5, 64), BF16, handle=buf), w, make(client, (5, 64), BF16, handle=buf.offset_start_by(2)), match="overlaps")
    f(x, make(client, (64,), BF16, handle=y.handle), y, match="overlaps")
    f(x, w, make(client, (5, 64), BF16, (1, 5)), code=N.E_UNSUPPORTED_STRIDES)
    f(x, w, make(client, (5, 64), BF16, (0, 1)), code=N.E_UNSUPPORTED_STRIDES)
    assert log(client)["norm"] == 0
    d = N.RmsNormDesc(rows=5, cols=64, ld_in=64, ld_out=64, eps=1e-6, dtype=BF16, dtype_weight=BF16, dtype_out=E4M3, scale_block=16)
    assert client.lib.mi355_rms_norm(client.ctx, None, C.byref(d), x.device_ptr(), None, None, None, q.device_ptr(), q.device_ptr(), None) == N.E_UNSUPPORTED


def test_rms_norm_backward_refusals(client):
    g, h, w, r, dx = make(client, (5, 64), F16), make(client, (5, 64), F16), make(client, (64,), F16), make(client, (5,)), make(client, (5, 64), F16)
    ops.rms_norm_backward(client, g, h, w, r, dx, grad_weight=make(client, (64,)), grad_hidden=dx)
    ops.rms_norm_backward(client, g, h, None, r, h)
    assert log(client)["norm_grad"] == 2 and log(client)["fold"] == 1
    ops.rms_norm_backward(client, make(client, (0, 64), F16), make(client, (0, 64), F16), w, make(client, (0,)), make(client, (0, 64), F16), grad_weight=make(client, (64,)))
    assert log(client)["norm_grad"] == 2 and log(client)["fold"] == 2                   # a sum over no rows is still written
    log(client, clear=True)
    f = lambda *args, **kw: refused(ops.rms_norm_backward, client, *args, **kw)
    f(g, make(client, (5, 64), BF16), w, r, dx)
    f(g, h, make(client, (64,), BF16), r, dx)
    f(g, h, w, make(client, (5,), F16), dx)
    f(g, h, w, make(client, (6,)), dx)
    f(g, h, w, r, make(client, (5, 64), F32))
    f(g, h, w, r, dx, grad_weight=make(client, (64,), BF16))
    f(g, h, w, r, dx, grad_weight=w, match="overlaps")
    f(g, h, w, r, dx, grad_hidden=make(client, (4, 64), F16))
    buf = client.empty(5 * 64 * 2 + 2)
    f(make(client, (5, 64), F16, handle=buf), h, w, r, make(client, (5, 64), F16, handle=buf.offset_start_by(2)), match="overlaps")
    d = N.RmsNormGradDesc(rows=5, cols=64, ld_out=64, ld_hidden=64, ld_in=64, dtype=F16, dtype_weight=F16, dtype_grad_weight=F32)
    need = C.c_uint64()
    assert client.lib.mi355_rms_norm_grad_workspace_bytes(C.byref(d), C.byref(need)) == N.OK and need.value >= 4 * 64
    ws, dw = client.empty(need.value), make(client, (64,))
    assert client.lib.mi355_rms_norm_grad(client.ctx, None, C.byref(d), g.device_ptr(), h.device_ptr(), w.device_ptr(), r.device_ptr(), None, dx.device_ptr(),
                                          dw.device_ptr(), ws.device_ptr(), need.value - 4) == N.E_INVALID_ARGUMENT
    assert log(client)["norm_grad"] == 0


# ---- global_norm and clip_by_global_norm ----------------------------------------------------------------------------------------------
def test_lists_are_cut_into_few_launches(client):
    ts = [make(client, (7, 9), BF16) for _ in range(300)] + [make(client, (0, 4)), make(client, (), F32)]
    out = make(client, (1,))
    ops.global_norm(client, ts, out)
    got = log(client, clear=True)
    assert got["sums"] == 3 and got["finish"] == 1 and got["chunks"] == 301 and got["scale"] == 0
    ops.clip_by_global_norm(client, ops.TensorList(ts), 1.0)
    got = log(client, clear=True)
    assert got["sums"] == got["scale"] == 3 and got["finish"] == 0 and got["partials"] <= 4096
    ops.clip_by_global_norm(client, [make(client, (40000, 3), F32, (4, 1)), make(client, (2, 40000), F16, (40008, 1))], 1.0)
    got = log(client, clear=True)
    assert got["sums"] == got["scale"] == 1 and got["chunks"] == -(-40000 // (16384 // 3)) + 2 * 3
    ops.global_norm(client, [], out)
    ops.clip_by_global_norm(client, [], 1.0, total_norm=out)
    assert log(client)["finish"] == 2 and log(client)["sums"] == 0


def test_a_long_list_leaves_no_more_partial_sums_than_the_workspace_holds(client):
    ts = [make(client, (3,))] * 6000 + [make(client, (1 << 20,))]
    ops.global_norm(client, ts, make(client, (1,)))                       # (the same tensor again only counts again)
    assert log(client)["sums"] == 54 and log(client)["partials"] <= 4096


def test_list_refusals(client):
    t, u, out = make(client, (8, 8)), make(client, (8, 8)), make(client, (1,))
    f = lambda *args, **kw: refused(ops.clip_by_global_norm, client, *args, **kw)
    refused(ops.global_norm, client, [make(client, (4,), E4M3)], out, code=N.E_UNSUPPORTED)
    refused(ops.global_norm, client, [make(client, (8, 8), F32, (1, 8))], out, code=N.E_UNSUPPORTED_STRIDES)
    refused(ops.global_norm, client, [t], make(client, (1,), BF16))
    refused(ops.global_norm, client, [t], make(client, (1,), F32, handle=t.handle), match="overlaps")
    for bad in (0.0, -1.0, float("nan")):
        f([t], bad)
    f([t, u], 1.0, outputs=[t])
    f([t], 1.0, outputs=[make(client, (8, 8), BF16)])
    f([t], 1.0, outputs=[make(client, (4, 16))])
    f([t, t], 1.0, match="overlaps another")                              # one tensor twice would be scaled twice
    f([t, u], 1.0, outputs=[u, t], match="overlaps another")
    f([t, u], 1.0, outputs=[make(client, (8, 8)), t], match="overlaps another")
    buf = client.empty(8 * 8 * 4 + 4)
    f([make(client, (8, 8), handle=buf)], 1.0, outputs=[make(client, (8, 8), handle=buf.offset_start_by(4))], match="overlaps")
    assert log(client)["sums"] == 0 and log(client)["scale"] == 0
    # column ranges of one matrix do not share memory, although their rows are interleaved
    wide = client.empty(8 * 24 * 4)
    parts = [make(client, (8, 8), F32, (24, 1), wide.offset_start_by(32 * i)) for i in range(3)]
    ops.clip_by_global_norm(client, parts, 1.0)
    f(parts + [make(client, (8, 8), F32, (24, 1), wide.offset_start_by(16))], 1.0, match="overlaps")
    # the same values read twice are two tensors of the list as long as neither is written
    ops.clip_by_global_norm(client, [t, t], 1.0, outputs=[u, make(client, (8, 8))])
    ws = client.empty(64)
    assert client.lib.mi355_global_norm(client.ctx, None, ops.TensorList([t]).spans, 1, out.device_ptr(), ws.device_ptr(), 64) == N.E_INVALID_ARGUMENT
    assert client.lib.mi355_clip_by_global_norm(client.ctx, None, None, None, 1, 1.0, None, ws.device_ptr(), 64) == N.E_INVALID_ARGUMENT
