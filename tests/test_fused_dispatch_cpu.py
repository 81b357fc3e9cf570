"""Which kernels mi355_gemm_fused launches, without a device: the library's own objects with every launcher replaced by one that writes down its
name and whether it was given an epilogue.  The dispatcher (gemm.cpp) and the kernels' own `supports` checks are the product's."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from cubecl_amd import _native as N

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "cubecl_amd" / "csrc"
BF, F16, F32, E4 = N.DTYPE_BF16, N.DTYPE_F16, N.DTYPE_F32, N.DTYPE_F8E4M3
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

RECORDER = r"""
#include "CSRC/gemm_common.hpp"
#include "CSRC/linear_ops.hpp"
#include <string>
static std::string seen;
static void note(const char *name, bool ep) { seen += (seen.empty() ? "" : " ") + std::string(name) + (ep ? "+" : ""); }
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }
namespace mi355 {
#define D const mi355_gemm_desc &, const void *, const void *, void *
#define WITH(name) int32_t launch_gemm_##name(mi355_ctx *, hipStream_t, D, const epilogue_args *ep) { note(#name, ep); return MI355_OK; }
#define WITHOUT(name) int32_t launch_gemm_##name(mi355_ctx *, hipStream_t, D) { note(#name, false); return MI355_OK; }
WITH(generic) WITH(f32_mfma) WITH(lp128) WITH(lp256x128) WITH(lp256m16) WITH(skinny) WITH(nnrows) WITH(stream64)
WITHOUT(lp256p) WITHOUT(lp256q) WITHOUT(lp256qm)
int32_t launch_gemm_lp256w4(mi355_ctx *, hipStream_t, D, const void *, const epilogue_args *ep) { note("lp256w4", ep); return MI355_OK; }
int32_t launch_gemm_lp256x192(mi355_ctx *, hipStream_t, D, int rows, const epilogue_args *ep) { note(rows == 192 ? "lp192x192" : "lp256x192", ep); return MI355_OK; }
int32_t launch_gemm_edge(mi355_ctx *, hipStream_t, D, const epilogue_args &) { note("edge", true); return MI355_OK; }
void launch_transpose(hipStream_t, const void *, void *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int) { note("transpose", false); }
void launch_pad_copy(hipStream_t, const void *, void *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int) { note("pad_copy", false); }
void launch_zero_columns(hipStream_t, void *, int64_t, int64_t, int64_t) {}
void launch_splitk_fold(hipStream_t, const float *, uint32_t, int64_t, int64_t, int64_t, int64_t, void *, int32_t, int64_t, int64_t) { note("fold", false); }
void launch_epilogue(hipStream_t, const float *, uint32_t, int64_t, const epilogue_args &, void *, int64_t, int64_t, int64_t, int64_t, int64_t) { note("fold", true); }
int32_t splitk_scratch(mi355_ctx *, hipStream_t, size_t, float **out) { *out = (float *)4096; return MI355_OK; }
int32_t scratch_get(mi355_ctx *, hipStream_t, int, size_t, void **out) { *out = (void *)4096; return MI355_OK; }
bool gemm_nnrows_ready(mi355_ctx *, hipStream_t, const mi355_gemm_desc &) { return true; }
void check_launch(mi355_ctx *, const char *) {}
}
extern "C" __attribute__((visibility("default"))) const char *record(const mi355_gemm_desc *d, const mi355_gemm_epilogue *ep)
{
    static mi355_ctx ctx;
    ctx.props.num_streaming_multiprocessors = 256;
    seen.clear();
    const char *a = (const char *)(1ull << 40), *b = (const char *)(1ull << 41), *c = (const char *)(1ull << 42);
    const int32_t rc = ep ? mi355_gemm_fused(&ctx, nullptr, d, ep, a, b, (void *)c) : mi355_gemm(&ctx, nullptr, d, a, b, (void *)c);
    if (rc != MI355_OK) seen = "refused " + std::to_string(rc) + " " + ctx.last_error;
    return seen.c_str();
}
"""


@pytest.fixture(scope="module")
def record(tmp_path_factory):
    objs = sorted((CSRC / "build").glob("*.o"))
    if not objs or not Path(HIPCC).exists() or not shutil.which("objcopy"):
        pytest.skip("the library's objects are not built here")
    d = tmp_path_factory.mktemp("recorder")
    (d / "recorder.cpp").write_text(RECORDER.replace("CSRC", str(CSRC)))
    subprocess.run([HIPCC, "-std=c++17", "-O1", "-fPIC", "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-c", str(d / "recorder.cpp"), "-o", str(d / "recorder.o")],
                   check=True, capture_output=True)
    for o in objs:                                       # their own launchers give way to the recorder's
        subprocess.run(["objcopy", "-w", "--weaken-symbol=_ZN5mi355*", str(o), str(d / o.name)], check=True)
    so = d / "librecord.so"
    subprocess.run([HIPCC, "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", str(so), str(d / "recorder.o")] + [str(d / o.name) for o in objs] + ["-ldl", "-lpthread"], check=True)
    lib = C.CDLL(str(so))
    lib.record.argtypes, lib.record.restype = [C.POINTER(N.GemmDesc), C.POINTER(N.GemmEpilogue)], C.c_char_p

    def run(m, n, k, dt, dt_c=None, ta=0, tb=1, batch=1, ep=None, algo=0):
        desc = N.GemmDesc(m=m, n=n, k=k, batch=batch, lda=m if ta else k, ldb=k if tb else n, ldc=n, stride_a=m * k if batch > 1 else 0, stride_b=k * n if batch > 1 else 0,
                          stride_c=m * n if batch > 1 else 0, dtype_ab=dt, dtype_c=dt if dt_c is None else dt_c, trans_a=ta, trans_b=tb, algo=algo)
        return lib.record(C.byref(desc), C.byref(ep) if ep is not None else None).decode()
    return run


def bias():
    return N.GemmEpilogue(bias=1 << 43, dtype_bias=F32)


PRODUCTS = [(4096, 4096, 4096), (8192, 8192, 8192), (8192, 28672, 8192), (4096, 14336, 4096), (16384, 4096, 4096), (8192, 11008, 4096), (4608, 4096, 8192), (2048, 2048, 2048),
            (2048, 2048, 256), (1, 8192, 8192), (16, 4096, 1024), (64, 2048, 2048), (300, 4096, 1024), (128, 256, 8192), (5000, 4096, 448)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dt,dt_c", [(BF, BF), (F16, F16), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("ta,tb", [(0, 1), (0, 0), (1, 0)])
def test_an_epilogue_without_parts_is_the_plain_product(record, m, n, k, dt, dt_c, ta, tb):
    """The gradients' products: the kernels mi355_gemm takes, or the edge kernel where operands would be copied first or f32 tiles leave the chip idle."""
    plain, fused = record(m, n, k, dt, dt_c, ta, tb), record(m, n, k, dt, dt_c, ta, tb, ep=N.GemmEpilogue())
    assert fused == plain or (fused == "edge+" and any(w in plain for w in ("transpose", "pad_copy", "f32_mfma", "generic"))), (plain, fused)


def test_the_largest_gradients_run_on_the_persistent_kernel(record):
    for m, n, k in PRODUCTS[:6]:
        assert record(m, k, n, BF, tb=1, ep=N.GemmEpilogue()) == "lp256qm", (m, n, k)      # grad_lhs = grad_pre rhs^T, rhs stored [k][n]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dt,dt_c", [(BF, BF), (BF, F32), (F32, F32)])
def test_an_epilogue_with_parts_reaches_a_kernel_that_carries_it(record, m, n, k, dt, dt_c):
    """Once, in the last launch that writes the output -- or in each of the two where a strip goes by itself."""
    for tb in (0, 1):
        seen = record(m, n, k, dt, dt_c, tb=tb, ep=bias()).split()
        assert seen[-1].endswith("+") and not any(s.startswith(("lp256q", "lp256p")) for s in seen), seen


def test_8_bit_products_take_the_small_tile_for_the_epilogue_only(record):
    """Two co-resident 128 x 128 tiles a CU hide each other's epilogue; the plain product stays on the square tile."""
    assert record(1777, 4096, 4096, E4, BF) == record(1777, 4096, 4096, E4, BF, ep=N.GemmEpilogue()) == "lp256w4"
    assert record(1777, 4096, 4096, E4, BF, ep=bias()) == "lp128+" and record(2560, 4096, 4096, E4, BF, ep=bias()) == "lp256w4+"
