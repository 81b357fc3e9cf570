"""Calls of the operators around a linear layer that once gave a wrong result or read what was not theirs, on the MI355X, against their formulas in
64 bits.  Helpers and tolerances are tests/test_gpu_linear_ops.py's unless a test says otherwise."""
import pytest
import torch

from cubecl_amd import TensorHandle, ops
from test_gpu_linear_ops import BF16, F32, close, down, empty, rand, rng, rounded, up

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
