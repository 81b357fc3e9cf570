"""Calls of the operators around a linear layer that once gave a wrong result or read what was not theirs, on the MI355X, against their formulas in
64 bits.  Helpers and tolerances are tests/test_gpu_linear_ops.py's unless a test says otherwise."""
import ctypes as C

import pytest
import torch

from cubecl_amd import TensorHandle, ops
from cubecl_amd import _native as N
from test_gpu_linear_ops import BF16, E4M3, E5M2, F32, FLOATS, TORCH, Step, act64, act_tol, close, down, empty, grad_tol, rand, raw_down, rng, rounded, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strides", [(0, 0, 1), (0, 16, 1), (16, 0, 1), (64, 8, 1)])
@pytest.mark.parametrize("dt", [F32, BF16], ids=lambda d: d.name)
def test_backward_of_an_lhs_whose_rows_share_memory(client, dt, strides):
    """A weight that a batch shared, behind a left operand broadcast over the rows, over the batch, or with rows that overlap."""
    m, n, k, batch = 8, 24, 16, 3
    g = rng(80)
    dy, store, b = rand(g, batch, m, n, dt=dt), rand(g, (batch - 1) * strides[0] + (m - 1) * strides[1] + k, dt=dt), rand(g, k, n, dt=dt)
    lhs = TensorHandle.new(up(client, store).handle, (batch, m, k), strides, dt)
    a = store.double().as_strided((batch, m, k), strides)
    dz, dB = empty(client, (batch, m, n), dt), empty(client, (k, n), dt)
    ops.matmul_fused_backward(client, up(client, dy), None, dz, lhs=lhs, rhs=up(client, b), grad_rhs=dB)
    ref = a.reshape(-1, k).t() @ dy.double().reshape(-1, n)
    close(down(client, dB), ref, rounded(ref, 1e-5 * (a.reshape(-1, k).abs().t() @ dy.double().reshape(-1, n).abs()), dt))


@pytest.mark.parametrize("dt", [F32, BF16], ids=lambda d: d.name)
def test_gradients_of_shared_operands_over_an_empty_batch(client, dt):
    """Sums over no entries: zeros, for a weight, a left operand and a bias."""
    one = lambda *s: up(client, torch.ones(s).to(torch.float32 if dt == F32 else torch.bfloat16))
    for lhs_shape in ((4, 5), (0, 4, 5)):
        da, db, bias = one(*lhs_shape), one(5, 6), one(6)
        ops.matmul_fused_backward(client, empty(client, (0, 4, 6), dt), None, empty(client, (0, 4, 6), dt), grad_bias=bias,
                                  lhs=one(*lhs_shape) if lhs_shape[0] else empty(client, lhs_shape, dt), rhs=one(5, 6), grad_lhs=da, grad_rhs=db)
        assert all(bool((down(client, t) == 0).all()) for t in (da, db, bias))


@pytest.mark.parametrize("m,n,k,batch", [(4, 8, 16, 3), (70, 33, 20, 4), (130, 264, 64, 2), (1, 40, 64, 5)])
@pytest.mark.parametrize("dt", [F32, BF16], ids=lambda d: d.name)
def test_entries_that_take_turns_by_rows(client, m, n, k, batch, dt):
    """The kept argument, the residual and the gradients as [m][batch][n] parts of one [m][batch][4 n] tensor; the fourth part stays as it was."""
    g = rng(81)
    a, b, r, dy = rand(g, batch, m, k, dt=dt), rand(g, k, n, dt=dt, scale=k ** -0.5), rand(g, batch, m, n, dt=dt), rand(g, batch, m, n, dt=dt)
    host = torch.full((m, batch, 4 * n), 7.0).to(r.dtype)
    host[:, :, n: 2 * n], host[:, :, 2 * n: 3 * n] = r.transpose(0, 1), dy.transpose(0, 1)
    whole = up(client, host)
    part = lambda i: TensorHandle.new(whole.handle.offset_start_by(i * n * dt.size()), (batch, m, n), (4 * n, 4 * n * batch, 1), dt)
    out, db = empty(client, (batch, m, n), dt), empty(client, (n,), F32)
    ops.matmul_fused(client, up(client, a), up(client, b), out, activation="silu", residual=part(1), pre_activation=part(0))
    z = a.double() @ b.double()
    tol = 1e-5 * (a.double().abs() @ b.double().abs()) + 2.0 ** -22 * z.abs()
    y = act64("silu", z)[0] + r.double()
    close(down(client, out), y, rounded(y, act_tol("silu", z, tol) + 2.0 ** -22 * y.abs(), dt))
    kept = down(client, part(0))
    close(kept, z, rounded(z, tol, dt))
    ops.matmul_fused_backward(client, part(2), part(0), part(2), activation="silu", grad_bias=db)
    ref = dy.double() * act64("silu", kept)[1]
    off = grad_tol("silu", kept, dy.double(), 2.0 ** -23 * ref.abs())
    close(down(client, part(2)), ref, rounded(ref, off, dt))
    close(down(client, db), ref.sum((0, 1)), off.sum((0, 1)) + 2.0 ** -24 * 512 * ref.abs().sum((0, 1)))
    assert torch.equal(down(client, part(1)), r.double()) and bool((down(client, part(3)) == 7).all())


@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-20, 1e-38])
def test_clip_by_factors_at_the_end_of_the_range(client, max_norm):
    """Norms that f32 does not hold brought down to small ones: the factor is a subnormal f32, or none at all, the results are ordinary numbers.
    Two roundings in f32 (the factor, the product) and the output's own; half a subnormal step of the type at the very end."""
    g = rng(82)
    for dt, scale in ((F32, 3e37), (BF16, 3e37), (F32, 1e25)):
        parts = [rand(g, 5000, scale=scale).to(TORCH[dt]), rand(g, 33, 70, scale=scale * 1e-9).to(TORCH[dt])]
        handles, total = [up(client, t) for t in parts], empty(client, (1,), F32)
        ops.clip_by_global_norm(client, handles, max_norm, total_norm=total)
        limit = float(torch.tensor(max_norm, dtype=torch.float32))
        factor = limit / float(torch.sqrt(sum(t.double().square().sum() for t in parts)))
        for t, h in zip(parts, handles):
            ref = t.double() * factor
            close(down(client, h), ref, rounded(ref, 2.0 ** -23 * 1.01 * ref.abs() + (2.0 ** -149 if dt == F32 else 2.0 ** -134), dt))


@pytest.mark.parametrize("m,n,k", [(64, 128, 64), (40, 64, 16384), (128, 256, 8192), (100, 100, 5001)])
@pytest.mark.parametrize("dt", [BF16, F32], ids=lambda d: d.name)
@pytest.mark.parametrize("power", [100, -100])
def test_scales_whose_product_leaves_the_range(client, m, n, k, dt, power):
    """(A B) rs cs with both scales 2^100 (2^-100) and products near 2^-80 (2^80): the same on one tile's accumulators and in the fold of K slices.
    Powers of two, so the only error is the product's."""
    g = rng(83)
    side = 2.0 ** (-40 if power > 0 else 40)
    a, b = rand(g, m, k, dt=dt, scale=side), rand(g, k, n, dt=dt, scale=side * k ** -0.5)
    out, scale = empty(client, (m, n), F32), torch.full((max(m, n),), 2.0 ** power)
    ops.matmul_fused(client, up(client, a), up(client, b.t().contiguous()).permute((1, 0)), out, lhs_scale=up(client, scale[:m]), rhs_scale=up(client, scale[:n]))
    ref, whole = a.double() @ b.double(), 2.0 ** (2 * power)
    close(down(client, out), ref * whole, 1e-5 * (a.double().abs() @ b.double().abs()) * whole)


@pytest.mark.parametrize("rows,cols", [(4000, 1024), (1500, 4096), (400, 8192), (500, 16384), (300, 20000)])
@pytest.mark.parametrize("out_dt", [E4M3, E5M2], ids=lambda d: d.name)
def test_8_bit_rows_are_quotients(client, rows, cols, out_dt):
    """Every 8-bit value is the nearest to y / scale of the kernel's own y (its f32 output) and scale, ties to even: a quotient that is a rounding
    off falls on the other side of a tie in one of 2^19 values, and there are some 2^22."""
    g = rng(84)
    x, w = rand(g, rows, cols, dt=BF16), rand(g, cols, dt=F32, scale=2.0 ** -110)
    w[: cols // 2] *= 2.0 ** 108                                        # ordinary rows, and from the third on rows of values near 2^-110
    x[2::3, : cols // 2] = 0
    x, w = up(client, x), up(client, w)
    y, q, s = empty(client, (rows, cols), F32), empty(client, (rows, cols), out_dt), empty(client, (rows,), F32)
    ops.rms_norm(client, x, w, y)
    ops.rms_norm(client, x, w, q, scales=s)
    want = (down(client, y).float() / down(client, s).float()[:, None]).to(TORCH[out_dt])
    assert torch.equal(raw_down(client, q), want.view(torch.uint8).reshape(-1))


# ---- activations to their tails -----------------------------------------------------------------------------------------------------------
# f32: exp2 1 ulp, its exponent in two pieces, the fit 4.3e-8 (2.9e-7 with its terms' rounding, evaluated in f32 over the whole range), three products
# of half an ulp each: below 8e-7 < 2^-20 of the value; a subnormal exponential is 2^-149 off, times |z|.  16-bit outputs: the fit 5.2e-6, the
# exponent |u| 2^-23 with |u| <= 88: below 2.4e-5 < 2^-15, then half a step of the type; what the instruction flushes is below 2^-118.
def tails(dt):
    z = torch.cat([torch.linspace(-104.0, 20.0, 2000), torch.linspace(-14.0, 6.0, 2000), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-4, -1e-4])]).to(TORCH[dt])
    return z[: z.numel() // 8 * 8]


def tail_tol(z, terms, dt):
    return 2.0 ** -20 * terms + (z.abs() + 2) * 2.0 ** -148 if dt == F32 else 2.0 ** -15 * terms + 2.0 ** -118


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("m,k,algo", [(1, 64, N.GEMM_ALGO_AUTO), (4, 64, N.GEMM_ALGO_GENERIC), (130, 64, N.GEMM_ALGO_AUTO), (130, 64, N.GEMM_ALGO_EDGE), (16, 8192, N.GEMM_ALGO_EDGE)])
def test_activation_tails(client, act, dt, m, k, algo):
    """Relative to the value, wherever the type has a number for it: on the tiles, element by element and in the fold of K slices."""
    z = tails(dt)
    out = empty(client, (m, z.numel()), dt)
    ops.matmul_fused(client, up(client, torch.zeros(m, k).to(z.dtype)), up(client, torch.zeros(k, z.numel()).to(z.dtype)), out, bias=up(client, z), activation=act, algo=algo)
    z = z.double().expand(m, -1)
    ref = act64(act, z)[0]
    close(down(client, out), ref, rounded(ref, tail_tol(z, ref.abs(), dt), dt) if dt != F32 else tail_tol(z, ref.abs(), dt))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", FLOATS, ids=lambda d: d.name)
def test_activation_gradient_tails(client, act, dt):
    """The derivative is a sum of two terms that may cancel: its error relative to theirs, twice a value's (each is two factors).  An f32 sigmoid
    below the normal numbers is a step of 2^-149 off (exponential and product half of one each), and the second term multiplies it by z u'(z): u' is 1
    for silu and sqrt(8 / pi) (1 + 3 c z^2), c = 0.044715, up to 25 at z = -10.6, for gelu's tanh form."""
    z = tails(dt)[None]
    dz = empty(client, tuple(z.shape), dt)
    ops.matmul_fused_backward(client, up(client, torch.ones_like(z)), up(client, z), dz, activation=act)
    z = z.double()
    y, ref = act64(act, z)
    part = torch.where(z == 0, 0.5, y / torch.where(z == 0, 1.0, z))                # Phi(z), sigmoid(u)
    slope = (8 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z) if act == "gelu_tanh" else torch.ones_like(z)
    close(down(client, dz), ref, rounded(ref, 2 * tail_tol(z * slope, part.abs() + (ref - part).abs(), dt), dt))


# ---- streams ----------------------------------------------------------------------------------------------------------------------------
def test_steps_on_two_streams_write_what_they_should(client):
    """Two programs at once on streams of their own, their outputs filled with 0xFF before each pass: work that was dropped, ended early or mixed up
    with the other program's workspaces and scratch shows in every pass."""
    steps = [Step(client, 90), Step(client, 91, rows=33, wide=512)]
    want = []
    for st in steps:
        st.run(client)
        want.append(st.bits(client))
    lanes = [client.with_stream(1), client.with_stream(2)]
    for i in range(4):
        for st in steps:
            for v in st.o.values():
                client._s.check(client.lib.mi355_memset(client.ctx, client.on(v), C.c_void_p(v.device_ptr()), 0xFF, v.handle.size_in_used()))
        client.sync()
        for _ in range(2):
            for st, lane in (zip(steps, lanes) if i % 2 else zip(steps[::-1], lanes)):
                st.run(lane)
        for lane in lanes:
            lane.sync()
        for st, w in zip(steps, want):
            got = st.bits(client)
            assert all(torch.equal(got[k], w[k]) for k in w), (i, [k for k in w if not torch.equal(got[k], w[k])])


def test_a_graph_of_k_slices_replayed_on_another_stream_beside_eager_calls(client):
    """The slices' partial sums lie in scratch of the stream that the graph was captured on: replays on two other streams and that stream's own calls
    of other operands, all queued at once, give what each gives alone."""
    m, n, k = 1024, 512, 8192
    g = rng(92)
    w = up(client, rand(g, k, n, dt=BF16, scale=k ** -0.5))
    rows = [up(client, rand(g, m, k, dt=BF16)) for _ in range(3)]
    outs = [empty(client, (m, n), BF16) for _ in rows]
    call = lambda i: ops.matmul_fused(client, rows[i], w, outs[i], activation="silu")
    want = []
    for i in range(3):
        call(i)
        want.append(raw_down(client, outs[i]))
    lanes = [client.with_stream(1), client.with_stream(2)]
    graphs = [client.capture(lambda i=i: call(i)) for i in range(2)]
    try:
        for _ in range(4):
            for v in outs:
                client._s.check(client.lib.mi355_memset(client.ctx, client.on(v), C.c_void_p(v.device_ptr()), 0xFF, m * n * 2))
            client.sync()
            for _ in range(6):
                lanes[0].replay(graphs[0])
                call(2)
                lanes[1].replay(graphs[1])
            for lane in (*lanes, client):
                lane.sync()
            assert all(torch.equal(raw_down(client, v), x) for v, x in zip(outs, want))
    finally:
        for graph in graphs:
            client.graph_destroy(graph)
