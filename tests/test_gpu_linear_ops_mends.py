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
