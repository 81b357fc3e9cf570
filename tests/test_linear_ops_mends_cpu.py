"""Calls that the operators around a linear layer once answered wrongly, or accepted and should not have, without a device: the host side on
the fake HIP runtime, as in tests/test_linear_ops_cpu.py.  Their GPU side is tests/test_gpu_linear_ops_mends.py."""
import numpy as np
import pytest

from cubecl_amd import ElemType, ops
from test_linear_ops_cpu import client, lib, log, make, refused  # noqa: F401

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
