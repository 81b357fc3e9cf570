"""The operators around a linear layer on the MI355X -- matmul_fused, rms_norm, global_norm / clip_by_global_norm and their gradients -- against
their formulas in 64 bits.

Tolerances, from the arithmetic (u = half a step of the output's type, relative: f32 2^-24, bf16 2^-8 / 2, f16 2^-11 / 2 -- torch.finfo(t).eps / 2):
  * a rounded output: u |ref| (f16: plus 2^-25, half a subnormal step) plus what the f32 arithmetic before it may be off;
  * products: 1e-5 sum |a||b| (the bound the GEMM tests hold every kernel to; the f8f6f4 instruction's own truncation on top for 8-bit operands);
  * activations: their slope is at most 1.13 (gelu's is), v_exp_f32 and v_rcp_f32 are 1 ulp and the exponent's product rounds at |x| 2^-24, so
    z * sigmoid(u) is off by less than (|u| + 4) 2^-23 of itself; erf by Abramowitz & Stegun 7.1.26 is 1.5e-7 absolute: 1.5e-7 |z|;
  * sums of n terms in f32: n-term chains are at most a few hundred long before they meet in a tree: 2^-24 * 512 of the sum of magnitudes;
  * 8-bit outputs: half a step of the 8-bit type of the value (e4m3 2^-4, e5m2 2^-3) or of its subnormals."""
import ctypes as C

import numpy as np
import pytest
import torch

from cubecl_amd import ElemType, ServerError, TensorHandle, ops
from cubecl_amd import _native as N

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3, E5M2, UE8M0 = ElemType.F32, ElemType.BF16, ElemType.F16, ElemType.F8E4M3, ElemType.F8E5M2, ElemType.UE8M0
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16, E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
MAX = {E4M3: 448.0, E5M2: 57344.0}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
FLOATS = [F32, BF16, F16]


def unit(dt):
    return torch.finfo(TORCH[dt]).eps / 2


def least(dt):
    return 2.0 ** -25 if dt == F16 else 0.0


def rng(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dt=F32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(TORCH[dt])


BITS = {4: (torch.int32, np.uint32), 2: (torch.int16, np.uint16), 1: (torch.uint8, np.uint8)}


def up(client, t, dt=None):
    """A torch tensor on the host -> a contiguous TensorHandle."""
    dt = dt or next(k for k, v in TORCH.items() if v == t.dtype)
    raw = t.contiguous().view(BITS[dt.size()][0]).numpy() if t.numel() else np.zeros(0, np.uint8)
    return TensorHandle.new_contiguous(tuple(t.shape), client.create_from_slice(raw) if raw.nbytes else client.empty(16), dt)


def empty(client, shape, dt):
    return TensorHandle.new_contiguous(shape, client.empty(max(int(np.prod(shape)) * dt.size(), 16)), dt)


def raw_down(client, h):
    """The bytes from a TensorHandle's first element to its last."""
    if 0 in h.shape:
        return torch.zeros(0, dtype=torch.uint8)
    n = (sum((d - 1) * s for d, s in zip(h.shape, h.strides)) + 1) * h.dtype.size()
    return torch.from_numpy(client.read_one(h.handle).copy())[:n]


def down(client, h):
    """A TensorHandle of any (non-negative) strides -> its values in 64 bits (ue8m0: the scales)."""
    if 0 in h.shape:
        return torch.zeros(tuple(h.shape), dtype=torch.float64)
    raw = raw_down(client, h)
    if h.dtype == UE8M0:
        e = raw.double()
        return torch.where(raw == 255, torch.full_like(e, float("nan")), torch.exp2(e - 127)).as_strided(h.shape, h.strides)
    return raw.view(TORCH[h.dtype]).double().as_strided(h.shape, h.strides)


def close(got, ref, tol, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (what, "NaNs elsewhere")
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), (what, "infinities elsewhere")
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(ref)
    off = (got - ref).abs() - tol
    off = torch.where(fine, off, torch.full_like(off, -1.0))
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - ref)[fine].abs().max()), int((off > 0).sum()), off.numel())


def rounded(ref, tol, dt):
    """The tolerance of a value rounded to `dt` that was `tol` off before."""
    return tol + unit(dt) * (ref.abs() + tol) + least(dt)


def act64(name, z):
    """(activation, derivative) in 64 bits; the limits at the infinities."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), torch.where(torch.isnan(z), z, (z > 0).double())
    zc = torch.where(torch.isnan(z), z, z.clamp(-1e4, 1e4))
    if name == "gelu":
        phi = 0.5 * torch.erfc(-zc / np.sqrt(2.0))
        d = phi + zc * torch.exp(-zc * zc / 2) / np.sqrt(2 * np.pi)
    else:
        c0, c1 = np.sqrt(2 / np.pi), 0.044715
        u, du = (zc, 1.0) if name == "silu" else (2 * c0 * zc * (1 + c1 * zc ** 2), 2 * c0 * (1 + 3 * c1 * zc ** 2))
        phi = torch.sigmoid(u)
        d = phi + zc * phi * (1 - phi) * du
    y = zc * phi
    y = torch.where(z == float("inf"), z, torch.where(z == -float("inf"), torch.zeros_like(z), torch.where(z.abs() > 1e4, z * (z > 0), y)))
    return y, d


def act_tol(name, z, tol_z):
    """How far the kernel's activation of a z that is tol_z off may be from act64's of the exact one."""
    if name in ("none", "relu"):
        return tol_z
    y = act64(name, z)[0].abs()
    u = 2 * 0.8 * z.abs() * (1 + 0.0448 * z * z) if name == "gelu_tanh" else z.abs()
    return 1.13 * tol_z + (u.clamp(max=100.0) + 4) * 2.0 ** -22 * y + (1.5e-7 * z.abs() if name == "gelu" else 0.0) + 1e-30


# ---- matmul_fused -------------------------------------------------------------------------------------------------------------------
def run_fused(client, m, n, k, dt, out_dt, act, bias=None, residual=False, pre=False, scales="", rhs="kn", lhs="mk", batch=(), seed=0, algo=N.GEMM_ALGO_AUTO):
    g = rng(seed)
    a, b = rand(g, *batch, m, k, dt=dt), rand(g, *batch, k, n, dt=dt, scale=max(k, 1) ** -0.5)
    ta = up(client, a) if lhs == "mk" else up(client, a.transpose(-1, -2).contiguous()).permute(tuple(range(len(batch))) + (len(batch) + 1, len(batch)))
    tb = up(client, b) if rhs == "kn" else up(client, b.transpose(-1, -2).contiguous()).permute(tuple(range(len(batch))) + (len(batch) + 1, len(batch)))
    kw, A, B = {}, a.double(), b.double()
    z, tol = A @ B, 1e-5 * (A.abs() @ B.abs())
    if dt in (E4M3, E5M2):
        from test_gpu_gemm import fp8_mfma_truncation_bound
        extra = fp8_mfma_truncation_bound(A.reshape(-1, k).numpy(), B.numpy())
        tol = tol + torch.as_tensor(extra).reshape(tol.shape)
    if "r" in scales:
        s = rand(g, *batch, m).abs() + 0.1
        kw["lhs_scale"], z, tol = up(client, s), z * s.double()[..., None], tol * s.double()[..., None]
    if "c" in scales:
        s = rand(g, n).abs() + 0.1
        kw["rhs_scale"], z, tol = up(client, s), z * s.double(), tol * s.double()
    if "t" in scales:
        s = torch.tensor([0.37])
        kw["rhs_scale"], z, tol = up(client, s), z * s.double(), tol * s.double()
    tol = tol + 2.0 ** -22 * z.abs()
    if bias is not None:
        v = rand(g, n, dt=bias, scale=0.5)
        kw["bias"], z = up(client, v), z + v.double()
    tol = tol + 2.0 ** -23 * z.abs()
    y = act64(act, z)[0]
    tol_y = act_tol(act, z, tol)
    out = empty(client, batch + (m, n), out_dt)
    if residual:
        r = rand(g, *batch, m, n, dt=out_dt)
        kw["residual"], y = up(client, r), y + r.double()
        tol_y = tol_y + 2.0 ** -23 * y.abs()
    if pre:
        kw["pre_activation"] = empty(client, batch + (m, n), out_dt)
    ops.matmul_fused(client, ta, tb, out, activation=act, algo=algo, **kw)
    close(down(client, out), y, rounded(y, tol_y, out_dt), "out")
    if pre:
        close(down(client, kw["pre_activation"]), z, rounded(z, tol, out_dt), "pre_activation")


SHAPES = [(1, 7, 5), (1, 256, 512), (2, 8, 64), (3, 64, 64), (17, 33, 129), (16, 512, 1024), (40, 130, 256), (64, 256, 128), (100, 1000, 72), (128, 128, 64), (300, 260, 192),
          (513, 520, 96), (777, 264, 320)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("rhs", ["kn", "nk"])
def test_fused_shapes(client, m, n, k, dt, rhs):
    i = SHAPES.index((m, n, k))
    run_fused(client, m, n, k, dt, dt, ACTS[i % 5], bias=dt, residual=i % 2 == 0, pre=i % 3 == 0, rhs=rhs, seed=i)
    if dt != F32:
        run_fused(client, m, n, k, dt, F32, ACTS[(i + 2) % 5], bias=F32, residual=i % 2 == 1, pre=True, rhs=rhs, seed=i + 50)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("parts", ["", "b", "r", "p", "br", "bp", "rp", "brp"])
@pytest.mark.parametrize("size", [(5, 24, 64), (130, 264, 128), (512, 512, 192)])
def test_fused_parts(client, act, parts, size):
    run_fused(client, *size, BF16, BF16, act, bias=F32 if "b" in parts else None, residual="r" in parts, pre="p" in parts, rhs="nk", seed=len(parts))


# sizes that the dispatcher hands to its different tiles and streaming kernels, both layouts of the weight
@pytest.mark.parametrize("m,n,k,dt,rhs", [
    (1, 4096, 2048, BF16, "nk"), (1, 4096, 2048, BF16, "kn"), (4, 2048, 2048, F16, "nk"), (16, 4096, 1024, BF16, "kn"), (33, 4096, 2048, BF16, "nk"), (64, 4096, 1024, F16, "kn"),
    (48, 2048, 2048, F32, "nk"), (2048, 48, 1024, BF16, "nk"), (256, 512, 8192, BF16, "nk"), (128, 256, 8192, BF16, "kn"), (1024, 1024, 512, BF16, "nk"), (1024, 1536, 512, F16, "kn"),
    (2048, 2048, 1024, BF16, "nk"), (2049, 2056, 512, BF16, "kn"), (2048, 2304, 256, F32, "nk"), (1536, 2048, 256, F32, "kn"), (4096, 4096, 512, BF16, "nk"), (4096, 4352, 1024, BF16, "nk"),
    (4096, 4608, 512, F16, "kn"), (4608, 4096, 2048, BF16, "nk"), (5000, 4096, 448, BF16, "nk")])
def test_fused_on_every_kernel(client, m, n, k, dt, rhs):
    run_fused(client, m, n, k, dt, dt, "silu", bias=dt, residual=True, pre=True, rhs=rhs, seed=3)
    run_fused(client, m, n, k, dt, F32, "gelu", bias=F32, residual=True, rhs=rhs, seed=4)


ALGOS = {"generic": N.GEMM_ALGO_GENERIC, "lp128": N.GEMM_ALGO_LP_128, "lp256w4": N.GEMM_ALGO_LP_256W4, "lp256x128": N.GEMM_ALGO_LP_256X128, "lp256x192": N.GEMM_ALGO_LP_256X192,
         "lp192x192": N.GEMM_ALGO_LP_192X192, "lp256m16": N.GEMM_ALGO_LP_256M16, "lp256p": N.GEMM_ALGO_LP_256P, "lp256qm": N.GEMM_ALGO_LP_256QM, "edge": N.GEMM_ALGO_EDGE}


@pytest.mark.parametrize("algo", sorted(ALGOS))
def test_fused_on_a_named_kernel(client, algo):
    run_fused(client, 512, 768, 512, BF16, BF16, "gelu_tanh", bias=F32, residual=True, pre=True, rhs="nk", algo=ALGOS[algo], seed=8)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 2), (31, 33, 7), (64, 64, 64), (65, 129, 63), (70, 66, 65), (100, 200, 517), (257, 130, 1001), (2050, 2049, 99), (33, 40, 4001)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("layout", ["mk,kn", "mk,nk", "km,kn", "km,nk"])
def test_fused_on_the_edge_kernel(client, m, n, k, dt, layout):
    """Every layout at sizes and alignments that nothing else stages as they lie; long K in slices."""
    lhs, rhs = layout.split(",")
    run_fused(client, m, n, k, dt, dt, "gelu_tanh", bias=dt, residual=True, pre=True, lhs=lhs, rhs=rhs, seed=m + k, algo=N.GEMM_ALGO_EDGE)
    if dt != F32:
        run_fused(client, m, n, k, dt, F32, "none", lhs=lhs, rhs=rhs, seed=m, algo=N.GEMM_ALGO_EDGE)
    run_fused(client, min(m, 80), min(n, 80), min(k, 80), dt, dt, "silu", bias=dt, scales="rc", batch=(3,), lhs=lhs, rhs=rhs, seed=n, algo=N.GEMM_ALGO_EDGE)


@pytest.mark.parametrize("m,n,k", [(1, 64, 128), (5, 40, 33), (16, 256, 256), (100, 96, 384), (257, 300, 512), (1030, 1040, 256)])
@pytest.mark.parametrize("dt", [E4M3, E5M2], ids=lambda d: d.name)
@pytest.mark.parametrize("scales", ["rc", "r", "t", ""])
def test_fused_on_8_bit_operands(client, m, n, k, dt, scales):
    run_fused(client, m, n, k, dt, BF16, "silu", bias=BF16, residual=True, pre=True, scales=scales, rhs="nk", seed=m)
    run_fused(client, m, n, k, dt, F16, "none", scales=scales, rhs="kn", seed=m + 1)


def test_fused_layouts(client):
    run_fused(client, 96, 80, 64, BF16, BF16, "gelu", bias=BF16, residual=True, lhs="km")
    run_fused(client, 264, 256, 128, F16, F32, "silu", bias=F32, residual=True, lhs="km", rhs="kn")
    run_fused(client, 24, 40, 64, BF16, BF16, "silu", bias=BF16, residual=True, pre=True, batch=(3,))
    run_fused(client, 130, 264, 64, BF16, BF16, "silu", bias=F32, residual=True, scales="rc", batch=(2, 2), rhs="nk")


@pytest.mark.parametrize("dt,m,n,k", [(BF16, 37, 40, 64), (F32, 37, 41, 65), (F16, 300, 272, 128), (BF16, 1, 512, 512)])
def test_fused_strides(client, dt, m, n, k):
    """Output, residual and pre-activation as column ranges of wider rows, at odd columns; the residual broadcast over rows; what lies between the
    rows of the output stays as it was; and the residual as the output itself."""
    g = rng(5)
    a, b, r, v = rand(g, m, k, dt=dt), rand(g, k, n, dt=dt, scale=k ** -0.5), rand(g, m, n, dt=dt), rand(g, n, dt=dt)
    z = a.double() @ b.double() + v.double()
    tol = 1e-5 * (a.double().abs() @ b.double().abs()) + 2.0 ** -22 * z.abs()
    y, tol_y = act64("silu", z)[0], act_tol("silu", z, tol) + 2.0 ** -22 * (z.abs() + r.double().abs())
    ta, tb, tv = up(client, a), up(client, b), up(client, v)
    es, ld = dt.size(), 3 * n + 5
    mark = torch.full((m, ld), 7.0).to(TORCH[dt])
    wide = up(client, mark)
    at = lambda off: TensorHandle.new(wide.handle.offset_start_by(off * es), (m, n), (ld, 1), dt)
    mark[:, 2 * n + 3: 3 * n + 3] = r
    wide = up(client, mark)
    out, pre, res = at(1), at(n + 2), at(2 * n + 3)
    ops.matmul_fused(client, ta, tb, out, bias=tv, activation="silu", residual=res, pre_activation=pre)
    whole = down(client, wide)
    ref = y + r.double()
    close(whole[:, 1: n + 1], ref, rounded(ref, tol_y, dt), "out")
    close(whole[:, n + 2: 2 * n + 2], z, rounded(z, tol, dt), "pre")
    for cols in (slice(0, 1), slice(n + 1, n + 2), slice(2 * n + 2, 2 * n + 3), slice(3 * n + 3, ld)):
        assert bool((whole[:, cols] == 7).all())
    one = up(client, r[:1])
    out = empty(client, (m, n), dt)
    ops.matmul_fused(client, ta, tb, out, bias=tv, activation="silu", residual=TensorHandle.new(one.handle, (m, n), (0, 1), dt))
    ref = y + r[:1].double()
    close(down(client, out), ref, rounded(ref, tol_y + 2.0 ** -22 * ref.abs(), dt), "broadcast residual")
    both = up(client, r)
    ops.matmul_fused(client, ta, tb, both, bias=tv, activation="silu", residual=both)
    ref = y + r.double()
    close(down(client, both), ref, rounded(ref, tol_y, dt), "in place")


def test_fused_batch_broadcasts(client):
    g = rng(6)
    a, b, v, s = rand(g, 3, 20, 32), rand(g, 32, 24), rand(g, 3, 24), rand(g, 3, 20).abs()
    z = (a.double() @ b.double()) * s.double()[..., None] + v.double()[:, None]
    tol = 1e-5 * (a.double().abs() @ b.double().abs()) * s.double()[..., None] + 2.0 ** -22 * z.abs()
    out = empty(client, (3, 20, 24), F32)
    ops.matmul_fused(client, up(client, a), up(client, b), out, bias=up(client, v), lhs_scale=up(client, s))
    close(down(client, out), z, rounded(z, tol, F32))
    # a bias that is every other value of a vector, a scale that is a column of a matrix
    v2, s2 = rand(g, 48), rand(g, 32, 5)
    z = (a[0].double() @ b.double()) * s2[:20, 2].double()[:, None] + v2[::2].double()
    out = empty(client, (20, 24), F32)
    tv, ts = up(client, v2), up(client, s2)
    ops.matmul_fused(client, up(client, a[0]), up(client, b), out, bias=TensorHandle.new(tv.handle, (24,), (2,), F32),
                     lhs_scale=TensorHandle.new(ts.handle.offset_start_by(8), (20,), (5,), F32))
    close(down(client, out), z, rounded(z, 1e-5 * (a[0].double().abs() @ b.double().abs()) * s2[:20, 2].double().abs()[:, None] + 2.0 ** -22 * z.abs(), F32))


@pytest.mark.parametrize("act", ACTS)
def test_fused_without_a_product(client, act):
    """k = 0: act(bias) + residual; no rows, no columns: nothing."""
    v, r = rand(rng(7), 9, scale=3.0), rand(rng(8), 4, 9)
    out = empty(client, (4, 9), F32)
    ops.matmul_fused(client, empty(client, (4, 0), F32), empty(client, (0, 9), F32), out, bias=up(client, v), activation=act, residual=up(client, r))
    z = v.double().expand(4, 9)
    ref = act64(act, z)[0] + r.double()
    close(down(client, out), ref, rounded(ref, act_tol(act, z, torch.zeros(())) + 2.0 ** -22 * ref.abs(), F32))
    ops.matmul_fused(client, empty(client, (0, 4), F32), empty(client, (4, 9), F32), empty(client, (0, 9), F32), activation=act)
    ops.matmul_fused(client, empty(client, (4, 4), F32), empty(client, (4, 0), F32), empty(client, (4, 0), F32), activation=act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(4, 64), (256, 256)])
def test_fused_special_values(client, act, size):
    """z = a b with b the identity: infinities, NaN, the largest and smallest numbers come out as the formula's limits."""
    m, n = size
    a = torch.zeros(m, n)
    special = torch.tensor([float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 1e-38, -1e-38, 0.0, -0.0, 88.0, -88.0, -104.0, 200.0, -200.0, 5.0, -5.0])
    out, b = empty(client, (m, n), F32), torch.zeros(1, n)
    b[0, : len(special)] = special
    ops.matmul_fused(client, up(client, torch.zeros(m, 64)), up(client, torch.zeros(64, n)), out, bias=up(client, b[0]), activation=act)
    z = b.double().expand(m, n)
    ref = act64(act, z)[0]
    tol = torch.where(torch.isfinite(z), act_tol(act, torch.where(torch.isfinite(z), z, torch.zeros_like(z)), torch.zeros(())), torch.zeros(()).double())
    tol = torch.where((z.abs() > 80) & torch.isfinite(z), 2.0 ** -22 * ref.abs() + 1e-33, tol)
    close(down(client, out), ref, tol + 2.0 ** -22 * ref.abs())


# ---- its gradient -----------------------------------------------------------------------------------------------------------------------
def grad_tol(act, z, g, tol):
    """v_exp / v_rcp errors as in act_tol on a derivative of at most 1.13, times the incoming gradient."""
    if act in ("none", "relu"):
        return tol
    u = 2 * 0.8 * z.abs() * (1 + 0.0448 * z * z) if act == "gelu_tanh" else z.abs()
    return tol + g.abs() * ((u.clamp(max=100.0) + 8) * 2.0 ** -22 * (1 + z.abs().clamp(max=20.0)) * 0.6 + 3e-7)


@pytest.mark.parametrize("m,n", [(1, 1), (1, 8), (3, 7), (5, 513), (64, 512), (100, 1000), (333, 517), (1000, 40), (4099, 24)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("act", ACTS)
def test_fused_backward_of_the_epilogue(client, m, n, dt, act):
    g = rng(m + n)
    dy, z = rand(g, m, n, dt=dt), rand(g, m, n, dt=dt, scale=2.0)
    dz, db = empty(client, (m, n), dt), empty(client, (n,), F32)
    ops.matmul_fused_backward(client, up(client, dy), up(client, z), dz, activation=act, grad_bias=db)
    ref = dy.double() * act64(act, z.double())[1]
    tol = grad_tol(act, z.double(), dy.double(), 2.0 ** -23 * ref.abs())
    close(down(client, dz), ref, rounded(ref, tol, dt), "grad_pre")
    close(down(client, db), ref.sum(0), tol.sum(0) + 2.0 ** -24 * 512 * ref.abs().sum(0), "grad_bias")


@pytest.mark.parametrize("act", ACTS[1:])
def test_activation_gradients_against_differences(client, act):
    """The kernel's derivative against central differences of the kernel's own activation: h = 2^-6, so the difference is off by h^2 / 6 times a
    third derivative below 3, and by the forward's 4e-7 / h."""
    z = torch.linspace(-6, 6, 384) + 0.013
    h = 2.0 ** -6
    eye = torch.zeros(1, 64)
    def forward(v):
        out = empty(client, (1, 384), F32)
        ops.matmul_fused(client, up(client, eye), up(client, torch.zeros(64, 384)), out, bias=up(client, v), activation=act)
        return down(client, out)[0]
    numeric = (forward((z + h).float()) - forward((z - h).float())) / (2 * h)
    dz = empty(client, (1, 384), F32)
    ops.matmul_fused_backward(client, up(client, torch.ones(1, 384)), up(client, z[None].float()), dz, activation=act)
    away = (z.abs() > h) | torch.tensor(act != "relu")
    close(down(client, dz)[0][away], numeric[away], h * h / 6 * 3 + 4e-7 * 6 / h)


@pytest.mark.parametrize("dt,gdt", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("m,n,k", [(3, 8, 16), (64, 128, 64), (100, 72, 40), (33, 65, 17), (256, 512, 256)])
def test_fused_backward_with_products(client, dt, gdt, m, n, k):
    g = rng(m * n)
    dy, z, a, b = rand(g, m, n, dt=dt), rand(g, m, n, dt=dt), rand(g, m, k, dt=dt), rand(g, k, n, dt=dt, scale=k ** -0.5)
    dz, db, da, dB = empty(client, (m, n), dt), empty(client, (n,), dt), empty(client, (m, k), gdt), empty(client, (k, n), gdt)
    ops.matmul_fused_backward(client, up(client, dy), up(client, z), dz, activation="gelu_tanh", grad_bias=db, lhs=up(client, a), rhs=up(client, b), grad_lhs=da, grad_rhs=dB)
    ref = dy.double() * act64("gelu_tanh", z.double())[1]
    off = rounded(ref, grad_tol("gelu_tanh", z.double(), dy.double(), 2.0 ** -23 * ref.abs()), dt)     # what grad_pre may be off
    for got, r, t in ((da, ref @ b.double().t(), (off + 1e-5 * ref.abs()) @ b.double().abs().t()), (dB, a.double().t() @ ref, a.double().abs().t() @ (off + 1e-5 * ref.abs()))):
        close(down(client, got), r, rounded(r, t, gdt))
    close(down(client, db), ref.sum(0), rounded(ref.sum(0), off.sum(0), dt))


def test_fused_backward_of_broadcast_operands(client):
    """A weight (a left operand, a bias) that a batch shared gets the sum over the batch."""
    g = rng(11)
    dy, a, b = rand(g, 3, 8, 24), rand(g, 3, 8, 16), rand(g, 3, 16, 24)
    D, A, B = dy.double(), a.double(), b.double()
    def run(lhs, rhs, grad_bias):
        dz, da, dB, db = empty(client, (3, 8, 24), F32), empty(client, tuple(lhs.shape), F32), empty(client, tuple(rhs.shape), F32), empty(client, grad_bias, F32)
        ops.matmul_fused_backward(client, up(client, dy), None, dz, grad_bias=db, lhs=up(client, lhs), rhs=up(client, rhs), grad_lhs=da, grad_rhs=dB)
        return down(client, da), down(client, dB), down(client, db)
    tol = 1e-5 * 3 * 24 * 6
    da, dB, db = run(a, b, (24,))
    close(da, D @ B.transpose(1, 2), tol), close(dB, A.transpose(1, 2) @ D, tol), close(db, D.sum((0, 1)), 1e-5)
    da, dB, db = run(a, b[0], (3, 24))
    close(da, D @ B[0].t(), tol), close(dB, torch.einsum("bmk,bmn->kn", A, D), tol), close(db, D.sum(1), 1e-5)
    da, dB, db = run(a[0], b, (24,))
    close(da, torch.einsum("bmn,bkn->mk", D, B), tol), close(dB, A[0].t() @ D, tol)
    da, dB, db = run(a[0], b[0], (24,))
    close(da, torch.einsum("bmn,kn->mk", D, B[0]), tol), close(dB, torch.einsum("mk,bmn->kn", A[0], D), tol)


def test_fused_backward_in_place_strided_and_empty(client):
    g = rng(12)
    dy, z = rand(g, 40, 33, dt=BF16), rand(g, 40, 33, dt=BF16)
    ref = dy.double() * act64("silu", z.double())[1]
    tol = rounded(ref, grad_tol("silu", z.double(), dy.double(), 2.0 ** -23 * ref.abs()), BF16)
    for which in (0, 1):
        td, tz = up(client, dy), up(client, z)
        ops.matmul_fused_backward(client, td, tz, (td, tz)[which], activation="silu")
        close(down(client, (td, tz)[which]), ref, tol)
    turned = up(client, dy.t().contiguous()).permute((1, 0))                       # a transposed gradient is made contiguous first
    out, db = TensorHandle.new(client.empty(40 * 50 * 2), (40, 33), (50, 1), BF16), empty(client, (33,), F32)
    ops.matmul_fused_backward(client, turned, up(client, z), out, activation="silu", grad_bias=db)
    close(down(client, out), ref, tol)
    only = empty(client, (33,), F32)
    ops.matmul_fused_backward(client, up(client, dy), up(client, z), None, activation="silu", grad_bias=only)
    assert torch.equal(down(client, only), down(client, db))
    zero = up(client, torch.ones(33))
    ops.matmul_fused_backward(client, empty(client, (0, 33), BF16), empty(client, (0, 33), BF16), empty(client, (0, 33), BF16), activation="silu", grad_bias=zero)
    assert bool((down(client, zero) == 0).all())


# ---- rms_norm ---------------------------------------------------------------------------------------------------------------------------
COLS = [1, 7, 8, 31, 32, 100, 512, 513, 1000, 1024, 1025, 2048, 2056, 4096, 5000, 8192, 8200, 16384, 16385, 20000]


def norm64(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    rstd = (h.square().mean(-1) + eps) ** -0.5
    return h, rstd, h * rstd[..., None] * (w.double() if w is not None else 1.0)


def norm_tol(y):
    """Sum of squares: 2^-24 * 64 relative at most, half of it through the root; rsq, two products."""
    return 2.0 ** -18 * y.abs() + 1e-37


@pytest.mark.parametrize("rows,cols", [(r, c) for c in COLS for r in ((1, 3) if c > 4096 else (5, 600))] + [(9, 3000), (40000, 16)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
def test_rms_norm_shapes(client, rows, cols, dt):
    g = rng(rows + cols)
    x, r, w = rand(g, rows, cols, dt=dt), rand(g, rows, cols, dt=dt, scale=2.0), 1 + 0.2 * torch.randn(cols, generator=g)
    w = w.to(TORCH[dt if cols % 2 else F32])
    h, rstd, y = norm64(x, r, w, 1e-5)
    out, hid, rs = empty(client, (rows, cols), dt), empty(client, (rows, cols), dt), empty(client, (rows,), F32)
    ops.rms_norm(client, up(client, x), up(client, w), out, eps=1e-5, residual=up(client, r), residual_out=hid, rstd=rs)
    close(down(client, out), y, rounded(y, norm_tol(y) + 2.0 ** -23 * rstd[:, None] * (x.double().abs() + r.double().abs()) * w.double().abs(), dt), "out")
    close(down(client, hid), h, rounded(h, 2.0 ** -24 * h.abs(), dt), "residual_out")
    close(down(client, rs), rstd, 2.0 ** -18 * rstd, "rstd")
    _, rstd, y = norm64(x, None, None, 1e-5)
    f32 = empty(client, (rows, cols), F32)
    ops.rms_norm(client, up(client, x), None, f32, eps=1e-5)
    close(down(client, f32), y, norm_tol(y), "f32 output, no weight")


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (600, 500), (4, 8192), (700, 4096), (3, 20001), (2, 16000)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("out_dt", [E4M3, E5M2], ids=lambda d: d.name)
def test_rms_norm_to_8_bits_by_row(client, rows, cols, dt, out_dt):
    g = rng(rows * cols)
    x, r, w = rand(g, rows, cols, dt=dt), rand(g, rows, cols, dt=dt), rand(g, cols, dt=dt)
    _, _, y = norm64(x, r, w, 1e-6)
    q, s = empty(client, (rows, cols), out_dt), empty(client, (rows,), F32)
    ops.rms_norm(client, up(client, x), up(client, w), q, residual=up(client, r), scales=s)
    got_q, got_s = down(client, q), down(client, s)
    close(got_s, y.abs().amax(1) / MAX[out_dt], 2.0 ** -17 * got_s, "scales")
    assert float(got_q.abs().max()) <= MAX[out_dt]
    step = 2.0 ** -9 if out_dt == E4M3 else 2.0 ** -16
    close(got_q * got_s[:, None], y, (2.0 ** -4 if out_dt == E4M3 else 2.0 ** -3) * y.abs() * (1 + 2.0 ** -16) + (step / 2 + 1e-6) * got_s[:, None] + 2 * norm_tol(y) +
          2.0 ** -21 * got_s[:, None] * MAX[out_dt], "values")


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (600, 96), (2, 512), (700, 1024), (5, 2048), (4, 8192), (700, 4096), (3, 20000), (2, 16416)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("out_dt", [E4M3, E5M2], ids=lambda d: d.name)
def test_rms_norm_to_8_bits_by_block(client, rows, cols, dt, out_dt):
    g = rng(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-8, 8, (rows, cols // 32), generator=g).float()).repeat_interleave(32, 1)).to(TORCH[dt])
    x[:, :32] = 0
    w = rand(g, cols, dt=dt)
    _, _, y = norm64(x, None, w, 1e-6)
    q, s = empty(client, (rows, cols), out_dt), empty(client, (rows, cols // 32), UE8M0)
    ops.rms_norm(client, up(client, x), up(client, w), q, scales=s)
    got_q, got_s = down(client, q), down(client, s)
    top = y.view(rows, -1, 32).abs().amax(2)
    ratio = top / got_s / MAX[out_dt]                        # the least power of two with ratio <= 1
    assert bool((ratio <= 1 + 2.0 ** -17).all()) and bool(((ratio > 0.5 * (1 - 2.0 ** -17)) | (top == 0)).all())
    assert bool((got_s[:, 0] == 1).all())                    # a block of zeros
    assert float(got_q.abs().max()) <= MAX[out_dt]
    sc = got_s.repeat_interleave(32, 1)
    step = 2.0 ** -9 if out_dt == E4M3 else 2.0 ** -16
    close(got_q * sc, y, (2.0 ** -4 if out_dt == E4M3 else 2.0 ** -3) * y.abs() * (1 + 2.0 ** -16) + step / 2 * sc + 2 * norm_tol(y), "values")


def test_rms_norm_special_rows(client):
    """Zeros, the largest and smallest numbers, NaN and infinities; each row by itself."""
    cols = 96
    g = rng(21)
    for dt in (F32, BF16):
        x = rand(g, 7, cols, dt=dt)
        x[0] = 0
        x[1] = (x[1].float() * 1e37).to(TORCH[dt])
        x[2] = 3e38
        x[3] = (x[3].float() * 1e-30).to(TORCH[dt])
        x[4, 5] = float("nan")
        x[5, 6] = float("inf")
        _, rstd, y = norm64(x, None, None, 1e-6)
        out, rs = empty(client, (7, cols), dt), empty(client, (7,), F32)
        ops.rms_norm(client, up(client, x), None, out, rstd=rs)
        close(down(client, out)[:4], y[:4], rounded(y[:4], norm_tol(y[:4]), dt))
        got = down(client, out)
        assert bool(torch.isnan(got[4]).all()) and bool(torch.isnan(got[5, 6])) and bool((got[5][torch.arange(cols) != 6] == 0).all())
        close(got[6], y[6], rounded(y[6], norm_tol(y[6]), dt))
        close(down(client, rs)[[0, 1, 2, 3, 6]], rstd[[0, 1, 2, 3, 6]], 2.0 ** -18 * rstd[[0, 1, 2, 3, 6]] + 2.0 ** -140)
        for sdt, shape in ((F32, (7,)), (UE8M0, (7, 3))):
            q, s = empty(client, (7, cols), E4M3), empty(client, shape, sdt)
            ops.rms_norm(client, up(client, x), None, q, scales=s)
            sc = down(client, s)
            sc = sc[:, None].expand(7, cols) if sdt == F32 else sc.repeat_interleave(32, 1)
            v = down(client, q) * sc
            keep = [0, 1, 2, 3, 6]
            close(v[keep], y[keep], 2.0 ** -4 * y[keep].abs() * 1.0001 + 2.0 ** -10 * sc[keep] + 1e-3 * sc[keep])
            assert bool(torch.isnan(v[4]).all()) and bool(torch.isnan(v[5, 6]))


@pytest.mark.parametrize("cols", [40, 1000, 4100, 17000])
def test_rms_norm_strides_and_in_place(client, cols):
    """Rows of wider matrices at odd columns, what lies between the rows of the output untouched; residual_out as the residual; output as input."""
    g, rows = rng(cols), 5
    x, r, w = rand(g, rows, cols, dt=BF16), rand(g, rows, cols, dt=BF16), rand(g, cols)
    h, rstd, y = norm64(x, r, w, 1e-6)
    tol = rounded(y, norm_tol(y) + 2.0 ** -22 * y.abs() + 2.0 ** -23 * rstd[:, None] * (x.double().abs() + r.double().abs()) * w.double().abs(), BF16)
    ld = 2 * cols + 3
    wide = torch.full((rows, ld), 7.0).to(torch.bfloat16)
    wide[:, 1: cols + 1] = x
    tw, tr = up(client, wide), up(client, r)
    view = lambda at: TensorHandle.new(tw.handle.offset_start_by(2 * at), (rows, cols), (ld, 1), BF16)
    ops.rms_norm(client, view(1), up(client, w), view(cols + 2), residual=tr, residual_out=tr)
    whole = down(client, tw)
    close(whole[:, cols + 2: 2 * cols + 2], y, tol)
    assert torch.equal(whole[:, 1: cols + 1], x.double()) and bool((whole[:, [0, cols + 1, 2 * cols + 2]] == 7).all())
    close(down(client, tr), h, rounded(h, 2.0 ** -24 * h.abs(), BF16))
    tx = up(client, x)
    ops.rms_norm(client, tx, up(client, w), tx, residual=up(client, r))
    close(down(client, tx), y, tol)
    turned = up(client, x.t().contiguous()).permute((1, 0))
    out = empty(client, (rows, cols), BF16)
    ops.rms_norm(client, turned, up(client, w), out, residual=up(client, r))
    close(down(client, out), y, tol)


def test_rms_norm_of_more_axes_and_none(client):
    x = rand(rng(30), 2, 3, 4, 64)
    _, rstd, y = norm64(x, None, None, 1e-6)
    out, rs = empty(client, (2, 3, 4, 64), F32), empty(client, (2, 3, 4), F32)
    ops.rms_norm(client, up(client, x), None, out, rstd=rs)
    close(down(client, out), y, norm_tol(y)), close(down(client, rs), rstd, 2.0 ** -18 * rstd)
    part = TensorHandle.new(up(client, x).handle, (2, 4, 64), (3 * 4 * 64, 64, 1), F32)          # rows that do not collapse
    out = empty(client, (2, 4, 64), F32)
    ops.rms_norm(client, part, None, out)
    close(down(client, out), y[:, 0], norm_tol(y[:, 0]))
    one = empty(client, (64,), F32)
    ops.rms_norm(client, up(client, x[0, 0, 0]), None, one)
    close(down(client, one), y[0, 0, 0], norm_tol(y[0, 0, 0]))


# ---- its gradient -----------------------------------------------------------------------------------------------------------------------
def norm_grad64(g, h, w, rstd, s):
    g, h, w, rstd = g.double(), h.double(), (w.double() if w is not None else torch.ones(h.shape[-1], dtype=torch.float64)), rstd.double()[:, None]
    xh, wg = h * rstd, g * w
    dx = rstd * (wg - xh * (wg * xh).mean(-1, keepdim=True)) + (s.double() if s is not None else 0.0)
    terms = rstd * (wg.abs() + xh.abs() * (wg * xh).abs().mean(-1, keepdim=True))
    return dx, (g * xh).sum(0), 2.0 ** -17 * terms, 2.0 ** -24 * 600 * (g * xh).abs().sum(0)


@pytest.mark.parametrize("rows,cols", [(r, c) for c in COLS for r in ((1, 5) if c > 4096 else (3, 700))] + [(3000, 24), (2100, 1032), (600, 8192), (300, 16400)])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
def test_rms_norm_backward_shapes(client, rows, cols, dt):
    g = rng(rows * 3 + cols)
    dy, h, w, s = rand(g, rows, cols, dt=dt), rand(g, rows, cols, dt=dt, scale=2.0), rand(g, cols, dt=dt), rand(g, rows, cols, dt=dt)
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    dx, dw, tx, tw = norm_grad64(dy, h, w, rstd, s)
    gx, gw = empty(client, (rows, cols), dt), empty(client, (cols,), F32)
    ops.rms_norm_backward(client, up(client, dy), up(client, h), up(client, w), up(client, rstd), gx, grad_weight=gw, grad_hidden=up(client, s))
    close(down(client, gx), dx, rounded(dx, tx + 2.0 ** -23 * dx.abs(), dt), "grad_input")
    close(down(client, gw), dw, tw, "grad_weight")
    dx, dw, tx, tw = norm_grad64(dy, h, None, rstd, None)
    gx = empty(client, (rows, cols), dt)
    ops.rms_norm_backward(client, up(client, dy), up(client, h), None, up(client, rstd), gx)
    close(down(client, gx), dx, rounded(dx, tx, dt), "no weight")


def test_rms_norm_backward_against_differences(client):
    """The gradient of sum(y c) with respect to input and weight against central differences of the forward kernel, f32: h = 2^-7; the forward is
    4e-6 of its terms off (norm_tol), the difference by h^2 / 6 of a third derivative below 60."""
    g, cols, step = rng(40), 24, 2.0 ** -7
    x, w, c = rand(g, 1, cols), rand(g, cols), rand(g, 1, cols)
    def value(x, w):
        out = empty(client, tuple(x.shape), F32)
        ops.rms_norm(client, up(client, x), up(client, w), out)
        return (down(client, out) * c.double()).sum(1)
    rs, out = empty(client, (1,), F32), empty(client, (1, cols), F32)
    ops.rms_norm(client, up(client, x), up(client, w), out, rstd=rs)
    gx, gw = empty(client, (1, cols), F32), empty(client, (cols,), F32)
    ops.rms_norm_backward(client, up(client, c), up(client, x), up(client, w), rs, gx, grad_weight=gw)
    shift = torch.eye(cols) * step
    tol = 60 * step * step / 6 + 4e-6 * 24 / step
    close(down(client, gx)[0], (value(x + shift, w) - value(x - shift, w)) / (2 * step), tol)
    numeric = torch.stack([(value(x, w + shift[i]) - value(x, w - shift[i]))[0] / (2 * step) for i in range(cols)])
    close(down(client, gw), numeric, tol)


@pytest.mark.parametrize("cols", [48, 4104, 17000])
def test_rms_norm_backward_in_place_and_empty(client, cols):
    g, rows = rng(cols), 6
    dy, h, w, s = rand(g, rows, cols, dt=F16), rand(g, rows, cols, dt=F16), rand(g, cols, dt=F16), rand(g, rows, cols, dt=F16)
    rstd = (h.double().square().mean(1) + 1e-6).rsqrt().float()
    dx, dw, tx, tw = norm_grad64(dy, h, w, rstd, s)
    for which in range(3):
        t = [up(client, dy), up(client, h), up(client, s)]
        gw = empty(client, (cols,), F16)
        ops.rms_norm_backward(client, t[0], t[1], up(client, w), up(client, rstd), t[which], grad_weight=gw, grad_hidden=t[2])
        close(down(client, t[which]), dx, rounded(dx, tx + 2.0 ** -23 * dx.abs(), F16), which)
        close(down(client, gw), dw, rounded(dw, tw, F16), which)
    zero = up(client, torch.ones(cols))
    ops.rms_norm_backward(client, empty(client, (0, cols), F16), empty(client, (0, cols), F16), up(client, w), empty(client, (0,), F32), empty(client, (0, cols), F16), grad_weight=zero)
    assert bool((down(client, zero) == 0).all())


# ---- global_norm and clip_by_global_norm ------------------------------------------------------------------------------------------------
def norm_list(client, ts):
    return float(np.sqrt(sum(float(t.double().square().sum()) for t in ts)))


LISTS = {
    "one value": [((), F32)], "one": [((5,), BF16)], "odd": [((3, 7), F16), ((1,), F32), ((0, 9), F32), ((1001,), BF16), ((33, 33), F32)],
    "chunk borders": [((16384,), F32), ((16385,), BF16), ((16383,), F16), ((2, 16384), BF16), ((7,), F32)],
    "many": [((i % 13 + 1, 5), (F32, BF16, F16)[i % 3]) for i in range(260)], "long": [(((1 << 20) + 3,), BF16), ((700, 1025), F32)],
}


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("max_norm", [0.37, 1e6, float("inf")])
def test_clip(client, name, max_norm):
    g = rng(50)
    ts = [rand(g, *s, dt=dt, scale=1.0 + 0.01 * i) for i, (s, dt) in enumerate(LISTS[name])]
    handles = [up(client, t) for t in ts]
    outs = [empty(client, s, dt) for s, dt in LISTS[name]]
    norm, total = empty(client, (1,), F32), empty(client, (1,), F32)
    ops.global_norm(client, handles, norm)
    ops.clip_by_global_norm(client, handles, max_norm, outputs=outs, total_norm=total)
    ref = norm_list(client, ts)
    close(down(client, norm), torch.tensor([ref], dtype=torch.float64), 2.0 ** -23 * ref)
    assert torch.equal(raw_down(client, norm), raw_down(client, total))
    coef = min(1.0, max_norm / ref)
    for t, o, h in zip(ts, outs, handles):
        dt = o.dtype
        close(down(client, o), t.double() * coef, rounded(t.double() * coef, 2.0 ** -22 * t.double().abs() * coef, dt) if coef < 1 else 0.0)
        assert torch.equal(down(client, h), t.double())
    ops.clip_by_global_norm(client, ops.TensorList(handles), max_norm)               # in place
    for o, h in zip(outs, handles):
        assert torch.equal(down(client, o), down(client, h))


def test_clip_views(client):
    """Padded rows, column ranges of one matrix in place, odd offsets; what lies between the rows stays."""
    g = rng(51)
    for rows, cols, ld, dt in ((300, 33, 100, F32), (5, 20000, 61000, BF16), (40000, 3, 10, F16)):
        whole = rand(g, rows, ld, dt=dt)
        th = up(client, whole)
        view = lambda at: TensorHandle.new(th.handle.offset_start_by(at * dt.size()), (rows, cols), (ld, 1), dt)
        parts = [whole[:, 1: 1 + cols], whole[:, 2 + cols: 2 + 2 * cols]]
        ref = norm_list(client, parts)
        coef = 0.5
        ops.clip_by_global_norm(client, [view(1), view(2 + cols)], ref / 2)
        want = whole.double().clone()
        want[:, 1: 1 + cols] *= coef
        want[:, 2 + cols: 2 + 2 * cols] *= coef
        tol = rounded(want, 2.0 ** -21 * want.abs(), dt)
        got = down(client, th)
        close(got, want, tol)
        assert torch.equal(got[:, 0], whole.double()[:, 0]) and torch.equal(got[:, 1 + cols], whole.double()[:, 1 + cols])
        flat = empty(client, (rows, cols), dt)                                       # padded in, contiguous out
        src = TensorHandle.new(up(client, whole).handle.offset_start_by(dt.size()), (rows, cols), (ld, 1), dt)
        ops.clip_by_global_norm(client, [src], float("inf"), outputs=[flat])
        assert torch.equal(down(client, flat), parts[0].double())
    line = rand(g, 1000, dt=BF16)
    h = up(client, line)
    odd = TensorHandle.new_contiguous((997,), h.handle.offset_start_by(2), BF16)
    ops.clip_by_global_norm(client, [odd], norm_list(client, [line[1:998]]) / 4)
    got = down(client, h)
    close(got[1:998], line[1:998].double() / 4, rounded(line[1:998].double() / 4, 2.0 ** -21 * line[1:998].double().abs(), BF16))
    assert got[0] == line[0].double() and torch.equal(got[998:], line[998:].double())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_clip_in_place_below_the_norm_changes_nothing(client, dt):
    """Contiguous tensors and column ranges of wider ones, in place, with a norm below the limit: the same bits, and the norm all the same."""
    g = rng(77)
    a, b = rand(g, 5, 4099, dt=dt), rand(g, 130, 77, dt=dt)
    ta, wide = up(client, a), up(client, b)
    view = TensorHandle.new(wide.handle, (130, 40), (77, 1), dt)
    before, norm = (raw_down(client, ta), raw_down(client, wide)), empty(client, (1,), F32)
    ops.clip_by_global_norm(client, ops.TensorList([ta, view]), 1e6, total_norm=norm)
    assert torch.equal(raw_down(client, ta), before[0]) and torch.equal(raw_down(client, wide), before[1])
    want = float(torch.sqrt(a.double().pow(2).sum() + b[:, :40].double().pow(2).sum()))
    assert abs(float(down(client, norm)[0]) - want) <= want * 2.0 ** -22


def test_clip_special_values(client):
    """Squares beyond f32 on both sides; a NaN or an infinity anywhere makes every output NaN; zeros stay zeros."""
    out = empty(client, (1,), F32)
    for scale in (1e30, 1e-30):
        t = (rand(rng(52), 3000) * scale)
        h = up(client, t)
        ref = norm_list(client, [t])
        ops.clip_by_global_norm(client, [h], ref / 8, total_norm=out)
        close(down(client, out), torch.tensor([ref], dtype=torch.float64), 2.0 ** -23 * ref)
        close(down(client, h), t.double() / 8, 2.0 ** -21 * t.double().abs())
    h = up(client, torch.full((4096,), 3e38))                                        # a norm that f32 does not hold
    ops.clip_by_global_norm(client, [h], 64.0, total_norm=out)
    assert float(down(client, out)) == float("inf")
    close(down(client, h), torch.ones(4096, dtype=torch.float64), 2.0 ** -20)
    for bad in (float("nan"), float("inf"), -float("inf")):
        a, b = torch.ones(5000), torch.ones(33)
        b[7] = bad
        ha, hb = up(client, a), up(client, b.to(torch.bfloat16))
        ops.clip_by_global_norm(client, [ha, hb], 1.0, total_norm=out)
        assert bool(torch.isnan(down(client, ha)).all()) and bool(torch.isnan(down(client, hb)).all())
        assert not bool(torch.isfinite(down(client, out)).all())
    z = up(client, torch.zeros(100))
    ops.clip_by_global_norm(client, [z], 1.0, total_norm=out)
    assert float(down(client, out)) == 0.0 and bool((down(client, z) == 0).all())
    ops.clip_by_global_norm(client, [], 1.0, total_norm=out)
    assert float(down(client, out)) == 0.0


# ---- together, on streams and in graphs ---------------------------------------------------------------------------------------------------
def test_results_are_the_same_bits_from_run_to_run(client):
    g = rng(60)
    dy, h, w = up(client, rand(g, 900, 2048, dt=BF16)), up(client, rand(g, 900, 2048, dt=BF16)), up(client, rand(g, 2048, dt=BF16))
    rstd = up(client, torch.ones(900))
    seen = []
    for _ in range(3):
        gx, gw, dz, db, norm = empty(client, (900, 2048), BF16), empty(client, (2048,), F32), empty(client, (900, 2048), BF16), empty(client, (2048,), F32), empty(client, (1,), F32)
        ops.rms_norm_backward(client, dy, h, w, rstd, gx, grad_weight=gw)
        ops.matmul_fused_backward(client, dy, h, dz, activation="silu", grad_bias=db)
        ops.global_norm(client, [gx, gw, dz, db], norm)
        seen.append([raw_down(client, t) for t in (gx, gw, dz, db, norm)])
    assert all(torch.equal(a, b) for s in seen[1:] for a, b in zip(seen[0], s))


class Step:
    """norm -> 8-bit linear layer -> residual norm -> gelu layer with its gradient -> clipping, as one training / serving step would chain them."""

    def __init__(self, client, seed, rows=70, width=128, wide=256):
        g = rng(seed)
        self.x, self.r = rand(g, rows, width, dt=BF16), rand(g, rows, width, dt=BF16)
        self.nw, self.w8 = (1 + 0.1 * torch.randn(width, generator=g)).to(torch.bfloat16), rand(g, wide, width)
        self.sw = self.w8.abs().amax(1) / 448
        self.q8 = (self.w8 / self.sw[:, None]).to(torch.float8_e4m3fn)
        self.b, self.w2 = rand(g, wide, dt=BF16), rand(g, wide, width, dt=BF16, scale=wide ** -0.5)
        self.dy = rand(g, rows, width, dt=BF16)
        self.t = {k: up(client, getattr(self, k)) for k in ("x", "r", "nw", "sw", "q8", "b", "w2", "dy")}
        e = lambda *s, dt=BF16: empty(client, s, dt)
        self.o = dict(q=e(rows, width, dt=E4M3), s=e(rows, dt=F32), hid=e(rows, width), rstd=e(rows, dt=F32), pre=e(rows, wide), act=e(rows, wide), y=e(rows, width), z2=e(rows, width),
                      dz=e(rows, width), db=e(width, dt=F32), dact=e(rows, wide), dw2=e(wide, width), dz1=e(rows, wide), db1=e(wide, dt=F32), dh=e(rows, width), dnw=e(width, dt=F32),
                      c0=e(wide, width), c1=e(width, dt=F32), total=e(1, dt=F32))

    def run(self, client):
        t, o = self.t, self.o
        ops.rms_norm(client, t["x"], t["nw"], o["q"], residual=t["r"], residual_out=o["hid"], scales=o["s"], rstd=o["rstd"])
        ops.matmul_fused(client, o["q"], t["q8"].permute((1, 0)), o["act"], bias=t["b"], activation="silu", lhs_scale=o["s"], rhs_scale=t["sw"], pre_activation=o["pre"])
        ops.matmul_fused(client, o["act"], t["w2"], o["y"], residual=o["hid"], activation="gelu", pre_activation=o["z2"])
        ops.matmul_fused_backward(client, t["dy"], o["z2"], o["dz"], activation="gelu", grad_bias=o["db"], lhs=o["act"], rhs=t["w2"], grad_lhs=o["dact"], grad_rhs=o["dw2"])
        ops.matmul_fused_backward(client, o["dact"], o["pre"], o["dz1"], activation="silu", grad_bias=o["db1"])
        ops.rms_norm_backward(client, t["dy"], o["hid"], t["nw"], o["rstd"], o["dh"], grad_weight=o["dnw"], grad_hidden=t["dy"])
        ops.clip_by_global_norm(client, [o["dw2"], o["dnw"]], 0.5, outputs=[o["c0"], o["c1"]], total_norm=o["total"])

    def bits(self, client):
        return {k: raw_down(client, v) for k, v in self.o.items()}


def test_a_step_against_64_bits(client):
    """The chain's values against the formulas on the chain's own intermediate results, so each operator is held to its own bound."""
    st = Step(client, 70)
    st.run(client)
    o = {k: down(client, v) for k, v in st.o.items()}
    h, rstd, y = norm64(st.x, st.r, st.nw, 1e-6)
    close(o["hid"], h, rounded(h, 2.0 ** -24 * h.abs(), BF16))
    close(o["q"] * o["s"][:, None], y, 2.0 ** -4 * y.abs() * 1.001 + (2.0 ** -10 + 1e-3) * o["s"][:, None])
    W = st.q8.double() * st.sw.double()[:, None]
    a = o["q"] * o["s"][:, None]
    z = a @ W.t() + st.b.double()
    tol = (2.0 ** -12) * (a.abs() @ W.abs().t()) + 2.0 ** -22 * z.abs()
    close(o["pre"], z, rounded(z, tol, BF16))
    close(o["act"], act64("silu", z)[0], rounded(act64("silu", z)[0], act_tol("silu", z, tol), BF16))
    z2 = o["act"] @ st.w2.double()
    t2 = 1e-5 * (o["act"].abs() @ st.w2.double().abs())
    ref = act64("gelu", z2)[0] + o["hid"]
    close(o["y"], ref, rounded(ref, act_tol("gelu", z2, t2) + 2.0 ** -22 * ref.abs(), BF16))
    dz = st.dy.double() * act64("gelu", o["z2"])[1]
    close(o["dz"], dz, rounded(dz, grad_tol("gelu", o["z2"], st.dy.double(), 2.0 ** -23 * dz.abs()), BF16))
    for got, r, t in ((o["dact"], o["dz"] @ st.w2.double().t(), o["dz"].abs() @ st.w2.double().abs().t()), (o["dw2"], o["act"].t() @ o["dz"], o["act"].abs().t() @ o["dz"].abs())):
        close(got, r, rounded(r, 1e-5 * t, BF16))
    total = torch.sqrt(o["dw2"].square().sum() + o["dnw"].square().sum())
    close(o["total"], total.view(1), 2.0 ** -22 * total)
    close(o["c0"], o["dw2"] * 0.5 / total, rounded(o["dw2"] * 0.5 / total, 2.0 ** -21 * o["dw2"].abs(), BF16))


def test_a_block_scaled_step(client):
    """rms_norm's ue8m0 blocks are what matmul_scaled multiplies back."""
    g = rng(71)
    x, nw = rand(g, 40, 256, dt=BF16), rand(g, 256, dt=BF16)
    w = (torch.randn(96, 256, generator=g)).to(torch.float8_e4m3fn)
    sw = torch.full((96, 8), 127, dtype=torch.uint8)
    q, s = empty(client, (40, 256), E4M3), empty(client, (40, 8), UE8M0)
    ops.rms_norm(client, up(client, x), up(client, nw), q, scales=s)
    out = empty(client, (40, 96), F32)
    ops.matmul_scaled(client, q, s, up(client, w), up(client, sw, UE8M0), out)
    a = down(client, q) * down(client, s).repeat_interleave(32, 1)
    ref = a @ w.double().t()
    close(down(client, out), ref, 2.0 ** -10 * (a.abs() @ w.double().abs().t()))


def test_steps_on_two_streams(client):
    """Two programs on streams of their own at once, their operands made on the first: what they compute alone."""
    a, b = Step(client, 72), Step(client, 73, rows=33, wide=512)
    a.run(client), b.run(client)
    want = [a.bits(client), b.bits(client)]
    one, two = client.with_stream(1), client.with_stream(2)
    for _ in range(3):
        a.run(one), b.run(two)
    one.sync(), two.sync()
    for st, w in zip((a, b), want):
        assert all(torch.equal(v, w[k]) for k, v in st.bits(client).items())


def test_captured_steps(client):
    """Two graphs of the same operators live at once and are replayed in turn, eager work of the same kind between them."""
    steps = [Step(client, 74), Step(client, 75, rows=50)]
    want = []
    for st in steps:
        st.run(client)
        want.append(st.bits(client))
        st.run(client)
    client.sync()
    graphs = [client.capture(lambda st=st: st.run(client)) for st in steps]
    other = Step(client, 76, rows=20, wide=384)
    try:
        for i in range(4):
            for st in steps:
                for v in st.o.values():
                    client._s.check(client.lib.mi355_memset(client.ctx, client.on(v), C.c_void_p(v.device_ptr()), 0xFF, v.handle.size_in_used()))
            for g in graphs if i % 2 else graphs[::-1]:
                client.replay(g)
                other.run(client)
            client.sync()
            for st, w in zip(steps, want):
                assert all(torch.equal(v, w[k]) for k, v in st.bits(client).items()), i
    finally:
        for g in graphs:
            client.graph_destroy(g)


@pytest.mark.parametrize("m,n,k,layout", [(2101, 2103, 1003, "mk,kn"), (2101, 2103, 1003, "km,kn"), (301, 203, 99, "km,nk"), (1024, 512, 8192, "mk,nk")])
def test_captured_products_of_any_size(client, m, n, k, layout):
    """Operands that are copied and zero-padded first, the edge kernel and K slices, captured and replayed with eager work of the same kind between."""
    g = rng(m)
    lhs, rhs = layout.split(",")
    a, b, v = rand(g, m, k, dt=BF16), rand(g, k, n, dt=BF16, scale=k ** -0.5), rand(g, n, dt=BF16)
    ta = up(client, a) if lhs == "mk" else up(client, a.t().contiguous()).permute((1, 0))
    tb = up(client, b) if rhs == "kn" else up(client, b.t().contiguous()).permute((1, 0))
    tv, out, other = up(client, v), empty(client, (m, n), BF16), empty(client, (m, n), BF16)
    call = lambda o: ops.matmul_fused(client, ta, tb, o, bias=tv, activation="silu")
    call(out)
    z = a.double() @ b.double() + v.double()
    y = act64("silu", z)[0]
    close(down(client, out), y, rounded(y, act_tol("silu", z, 1e-5 * (a.double().abs() @ b.double().abs()) + 2.0 ** -22 * z.abs()), BF16))
    want = raw_down(client, out)
    graph = client.capture(lambda: call(out))
    try:
        for _ in range(3):
            client._s.check(client.lib.mi355_memset(client.ctx, client.on(out), C.c_void_p(out.device_ptr()), 0xFF, m * n * 2))
            client.replay(graph)
            call(other)
            client.sync()
            assert torch.equal(raw_down(client, out), want) and torch.equal(raw_down(client, other), want)
    finally:
        client.graph_destroy(graph)


def test_refusals_leave_the_output_alone(client):
    a, b = up(client, torch.ones(4, 8)), up(client, torch.ones(8, 8))
    c = up(client, torch.full((4, 8), 7.0))
    for kw in (dict(pre_activation=c), dict(bias=up(client, torch.ones(5))), dict(activation="nope"), dict(lhs_scale=up(client, torch.ones(3)))):
        with pytest.raises(ServerError):
            ops.matmul_fused(client, a, b, c, **kw)
    with pytest.raises(ServerError):
        ops.rms_norm(client, a, up(client, torch.ones(7)), c)
    with pytest.raises(ServerError):
        ops.clip_by_global_norm(client, [c, c], 1.0)
    assert bool((down(client, c) == 7).all())
