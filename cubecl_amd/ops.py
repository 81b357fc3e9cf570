"""Launch entry points of the hot path: tiled matmul and reductions over TensorHandles.

The reference keeps these launchers in the out-of-tree `cubek` crates (README.md:161-165); what
the snapshot pins is the operand contract -- TensorHandle {handle, shape, strides, dtype}
(crates/cubecl-std/src/tensor/handle.rs:13-23), strides in elements, transposition / broadcast
expressed through strides and classified by matrix_batch_layout
(crates/cubecl-std/src/tensor/matrix_batch_layout.rs:21-79) -- and the arithmetic
(runtime_tests/cmma.rs:695-722 for matmul; examples/sum_things/src/lib.rs:6-19 and the book's
reduce_matrix for sums).  These functions take exactly that contract and forward to the C ABI.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from . import _native as N
from .runtime import ComputeClient, ElemType, Handle, ServerError
from .tensor import TensorHandle, matrix_batch_layout


def _matrix_operand(t: TensorHandle, name: str):
    """-> (transposed, leading dimension, batch count, batch stride)."""
    if len(t.shape) == 2 and min(t.shape) > 1 and min(t.strides) == 1:     # one matrix, either way round: nothing to classify
        rs, cs = t.strides
        return (False, rs, 1, 0) if cs == 1 else (True, cs, 1, 0)
    if t.rank() < 2:
        raise ServerError(N.E_INVALID_ARGUMENT, f"matmul: {name} must have rank >= 2")
    if t.shape[-2] == 0 or t.shape[-1] == 0:   # empty operand (K == 0 or empty output): nothing is read
        batch = 1
        for d in t.shape[:-2]:
            batch *= d
        return False, max(t.shape[-1], 1), batch, 0
    layout = matrix_batch_layout(t.strides)
    if layout.kind == "HighlyPermuted":
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"matmul: {name} is HighlyPermuted; make it contiguous first")
    rows, cols = t.shape[-2], t.shape[-1]
    rs, cs = t.strides[-2], t.strides[-1]
    if cs == 1:
        transposed, ld = False, rs
    elif rs == 1:
        transposed, ld = True, cs
    else:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"matmul: {name} has no unit stride in its last two dims")
    if (rows == 1 or cols == 1) and ld < (rows if transposed else cols):
        ld = rows if transposed else cols
    batch_dims, batch_strides = t.shape[:-2], t.strides[:-2]
    batch = 1
    for d in batch_dims:
        batch *= d
    nontrivial = [(d, s) for d, s in zip(batch_dims, batch_strides) if d != 1]
    if not nontrivial:
        bstride = 0
    else:
        # collapsible iff each outer stride = inner stride * inner dim (or everything broadcast)
        bstride = nontrivial[-1][1]
        for (d_out, s_out), (d_in, s_in) in zip(nontrivial[:-1], nontrivial[1:]):
            if s_out != s_in * d_in:
                raise ServerError(N.E_UNSUPPORTED_STRIDES, f"matmul: {name} batch dims are not collapsible")
    return transposed, ld, batch, bstride


def _kernel_ready(client: ComputeClient, t: TensorHandle, name: str):
    """What the reference's matmul launchers do in front of the kernel: an operand whose strides the kernel cannot
    consume (matrix_batch_layout says HighlyPermuted, or the batch axes do not collapse) goes through
    into_contiguous first (crates/cubecl-std/src/tensor/matrix_batch_layout.rs:9-19, contiguous/launch.rs:5-20)."""
    try:
        return t, _matrix_operand(t, name)
    except ServerError as e:
        if e.code != N.E_UNSUPPORTED_STRIDES:
            raise
    t = into_contiguous(client, t)
    return t, _matrix_operand(t, name)


def matmul(client: ComputeClient, lhs: TensorHandle, rhs: TensorHandle, out: TensorHandle,
           algo: int = N.GEMM_ALGO_AUTO, acc: Optional[TensorHandle] = None) -> None:
    """out[.., m, n] = sum_k lhs[.., m, k] * rhs[.., k, n]   (f32 accumulate)   [+ acc[.., m, n]].

    `acc` is the C operand of cmma::execute(a, b, c, d) (frontend/cmma.rs:1066-1110): the product plus acc is formed
    in f32 and rounded once to out's dtype; acc has out's dtype and may be `out` itself (in-place accumulate).

    Layouts come from strides alone: a `rhs` of logical shape [k, n] with strides [1, k] is the
    reference tests' "ColMajor B" / Out = Lhs * Rhs^T form (cmma.rs:23) and takes the fast
    K-contiguous MFMA path; strides [n, 1] is row-major B.
    """
    m, k = lhs.shape[-2], lhs.shape[-1]
    k2, n = rhs.shape[-2], rhs.shape[-1]
    if k != k2 or out.shape[-2] != m or out.shape[-1] != n:
        raise ServerError(N.E_INVALID_ARGUMENT, f"matmul: shape mismatch {lhs.shape} x {rhs.shape} -> {out.shape}")
    if lhs.dtype != rhs.dtype:
        raise ServerError(N.E_INVALID_ARGUMENT, "matmul: lhs/rhs dtypes differ")
    lhs, (ta, lda, ba, sa) = _kernel_ready(client, lhs, "lhs")
    rhs, (tb, ldb, bb, sb) = _kernel_ready(client, rhs, "rhs")
    tc, ldc, bc, sc = _matrix_operand(out, "out")
    if tc:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, "matmul: out must be row-major")
    batch = bc
    for b, name in ((ba, "lhs"), (bb, "rhs")):
        if b not in (1, batch):
            raise ServerError(N.E_INVALID_ARGUMENT, f"matmul: {name} batch {b} does not broadcast to {batch}")
    desc = N.GemmDesc(m=m, n=n, k=k, batch=batch, lda=lda, ldb=ldb, ldc=ldc,
                      stride_a=sa if ba == batch else 0, stride_b=sb if bb == batch else 0, stride_c=sc,
                      dtype_ab=int(lhs.dtype), dtype_c=int(out.dtype), trans_a=int(ta), trans_b=int(tb), algo=algo)
    if acc is None:
        client._s.check(client.lib.mi355_gemm(client.ctx, client.on(lhs, rhs, out), C.byref(desc), C.c_void_p(lhs.device_ptr()),
                                              C.c_void_p(rhs.device_ptr()), C.c_void_p(out.device_ptr())))
        return
    if acc.dtype != out.dtype or tuple(acc.shape) != tuple(out.shape):
        raise ServerError(N.E_INVALID_ARGUMENT, "matmul: acc must have out's shape and dtype")
    if tuple(acc.strides) != tuple(out.strides):
        acc = _like(client, acc, out)                       # bring C into D's layout (copy_into)
    client._s.check(client.lib.mi355_gemm_add(client.ctx, client.on(lhs, rhs, acc, out), C.byref(desc), C.c_void_p(lhs.device_ptr()),
                                              C.c_void_p(rhs.device_ptr()), C.c_void_p(acc.device_ptr()),
                                              C.c_void_p(out.device_ptr())))


def _like(client: ComputeClient, t: TensorHandle, model: TensorHandle) -> TensorHandle:
    """A copy of `t` laid out with `model`'s strides."""
    span = sum((d - 1) * s for d, s in zip(model.shape, model.strides)) + 1 if model.num_elems() else 0
    out = TensorHandle.new(client.empty(span * t.dtype.size()), model.shape, model.strides, t.dtype)
    copy_into(client, t, out)
    return out


def matmul_scaled(client: ComputeClient, lhs: TensorHandle, lhs_scales: TensorHandle, rhs: TensorHandle,
                  rhs_scales: TensorHandle, out: TensorHandle, *, block: int = 32, algo: int = N.GEMM_ALGO_AUTO) -> None:
    """Block-scaled matmul, out[.., m, n] = sum_k lhs[.., m, k] s_l[.., m, k/block] rhs[.., n, k] s_r[.., n, k/block].

    The layouts are the reference test's (runtime_tests/cmma.rs:1549-1560): `lhs` [.., m, k] row-major, `rhs` stored
    [.., n, k], scales [.., rows, k / block] (ue8m0).  F4E2M1X2 handles have a BYTE shape: [.., rows, k / 2]."""
    packed = 2 if lhs.dtype == ElemType.F4E2M1X2 else 1
    m, k = lhs.shape[-2], lhs.shape[-1] * packed
    n, k2 = rhs.shape[-2], rhs.shape[-1] * packed
    if k != k2 or out.shape[-2] != m or out.shape[-1] != n or lhs_scales.shape[-2] != m or rhs_scales.shape[-2] != n:
        raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_scaled: shape mismatch {lhs.shape} x {rhs.shape} -> {out.shape}")
    if lhs_scales.shape[-1] * block != k or rhs_scales.shape[-1] * block != k:
        raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_scaled: {lhs_scales.shape[-1]} scales per row do not cover k = {k} in blocks of {block}")
    for t, name in ((lhs, "lhs"), (rhs, "rhs"), (out, "out"), (lhs_scales, "lhs_scales"), (rhs_scales, "rhs_scales")):
        if t.strides[-1] != 1:
            raise ServerError(N.E_UNSUPPORTED_STRIDES, f"matmul_scaled: {name} must be contiguous along its last axis")

    def bstride(t, name):
        if t.rank() == 2:
            return 1, 0
        if t.rank() != 3:
            raise ServerError(N.E_UNSUPPORTED_STRIDES, f"matmul_scaled: {name} must have rank 2 or 3")
        return t.shape[0], t.strides[0]
    (ba, sa), (bb, sb), (bc, sc) = bstride(lhs, "lhs"), bstride(rhs, "rhs"), bstride(out, "out")
    (bsa, ssa), (bsb, ssb) = bstride(lhs_scales, "lhs_scales"), bstride(rhs_scales, "rhs_scales")
    batch = bc
    for b_, name in ((ba, "lhs"), (bb, "rhs"), (bsa, "lhs_scales"), (bsb, "rhs_scales")):
        if b_ not in (1, batch):
            raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_scaled: {name} batch {b_} does not broadcast to {batch}")
    if (ba == batch) != (bsa == batch) or (bb == batch) != (bsb == batch):
        raise ServerError(N.E_INVALID_ARGUMENT, "matmul_scaled: an operand and its scales must be batched alike")
    desc = N.GemmScaledDesc(m=m, n=n, k=k, batch=batch, lda=lhs.strides[-2] * packed, ldb=rhs.strides[-2] * packed,
                            ldc=out.strides[-2], ld_sa=lhs_scales.strides[-2], ld_sb=rhs_scales.strides[-2],
                            stride_a=(sa if ba == batch else 0) * packed, stride_b=(sb if bb == batch else 0) * packed,
                            stride_c=sc, stride_sa=ssa if bsa == batch else 0, stride_sb=ssb if bsb == batch else 0,
                            dtype_a=int(lhs.dtype), dtype_b=int(rhs.dtype), dtype_c=int(out.dtype), block=block, algo=algo)
    client._s.check(client.lib.mi355_gemm_scaled(client.ctx, client.on(lhs, lhs_scales, rhs, rhs_scales, out), C.byref(desc), C.c_void_p(lhs.device_ptr()),
                                                 C.c_void_p(lhs_scales.device_ptr()), C.c_void_p(rhs.device_ptr()),
                                                 C.c_void_p(rhs_scales.device_ptr()), C.c_void_p(out.device_ptr())))


def gemm_scaled_select(client: ComputeClient, desc: N.GemmScaledDesc) -> int:
    algo = C.c_int32()
    client._s.check(client.lib.mi355_gemm_scaled_select(client.ctx, C.byref(desc), C.byref(algo)))
    return algo.value


def gemm_select(client: ComputeClient, desc: N.GemmDesc) -> int:
    algo = C.c_int32()
    client._s.check(client.lib.mi355_gemm_select(client.ctx, C.byref(desc), C.byref(algo)))
    return algo.value


def gemm_relayout_plan(client: ComputeClient, desc: N.GemmDesc):
    """(relayout_a, relayout_b): which operands mi355_gemm would copy into library scratch before the MFMA kernel."""
    ra, rb = C.c_int32(), C.c_int32()
    client._s.check(client.lib.mi355_gemm_relayout_plan(C.byref(desc), C.byref(ra), C.byref(rb)))
    return bool(ra.value), bool(rb.value)


def gemm_split_plan(client: ComputeClient, desc: N.GemmDesc) -> int:
    """K slices the 128x128 kernel's launcher cuts `desc` into on this device (1 = one plain launch)."""
    out = C.c_int32()
    client._s.check(client.lib.mi355_gemm_split_plan(C.byref(desc), int(client.properties().num_streaming_multiprocessors or 0), C.byref(out)))
    return out.value


_WORKSPACES: dict = {}


def _workspace(client: ComputeClient, n: int) -> Handle:
    key = (id(client._s), client.stream_id())      # one per logical stream: two lanes may reduce at the same time
    need = C.c_uint64()
    client._s.check(client.lib.mi355_reduce_workspace_bytes(client.ctx, n, C.byref(need)))
    ws = _WORKSPACES.get(key)
    if ws is None or ws.size < need.value or ws.memory.server is not client._s:
        ws = client.empty(need.value)
        _WORKSPACES[key] = ws
    return ws


def _require_flat_f32(t: TensorHandle, what: str) -> int:
    """Array-wide reductions take f32, bf16 or f16 input (16-bit elements are widened to f32 on load)."""
    if t.dtype not in (ElemType.F32, ElemType.BF16, ElemType.F16):
        raise ServerError(N.E_UNSUPPORTED, f"{what}: input must be f32, bf16 or f16")
    if not t.is_contiguous():
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: input must be contiguous")
    return t.num_elems()


def _consumable(client: ComputeClient, t: TensorHandle, view, what: str):
    """-> (tensor, view(tensor)): a permuted / sliced input the reduction kernels cannot walk goes through into_contiguous
    first, the same step the matmul launcher takes (contiguous/launch.rs:5-20)."""
    try:
        return t, view(t, what)
    except ServerError as e:
        if e.code != N.E_UNSUPPORTED_STRIDES:
            raise
    t = into_contiguous(client, t)
    return t, view(t, what)


def reduce_sum(client: ComputeClient, input: TensorHandle, output: TensorHandle) -> None:
    """Array-wide sum into output[0] (f32)."""
    input, n = _consumable(client, input, _require_flat_f32, "reduce_sum")
    ws = _workspace(client, n)
    client._s.check(client.lib.mi355_reduce_sum(client.ctx, client.on(input, output, ws), C.c_void_p(input.device_ptr()), int(input.dtype), n,
                                                C.c_void_p(output.device_ptr()), C.c_void_p(ws.device_ptr()), ws.size))


def argmax(client: ComputeClient, input: TensorHandle, out_index: TensorHandle,
           out_value: Optional[TensorHandle] = None) -> None:
    """Array-wide argmax: out_index[0] (u64) = lowest index of the maximum; NaN ranks highest."""
    input, n = _consumable(client, input, _require_flat_f32, "argmax")
    ws = _workspace(client, n)
    client._s.check(client.lib.mi355_argmax(
        client.ctx, client.on(input, out_value, out_index, ws), C.c_void_p(input.device_ptr()), int(input.dtype), n,
        C.c_void_p(out_value.device_ptr()) if out_value is not None else None,
        C.c_void_p(out_index.device_ptr()), C.c_void_p(ws.device_ptr()), ws.size))


def sum_argmax(client: ComputeClient, input: TensorHandle, out_sum: TensorHandle, out_index: TensorHandle,
               out_value: Optional[TensorHandle] = None) -> None:
    """Sum and argmax in one pass over the data."""
    input, n = _consumable(client, input, _require_flat_f32, "sum_argmax")
    ws = _workspace(client, n)
    client._s.check(client.lib.mi355_sum_argmax(
        client.ctx, client.on(input, out_sum, out_value, out_index, ws), C.c_void_p(input.device_ptr()), int(input.dtype), n, C.c_void_p(out_sum.device_ptr()),
        C.c_void_p(out_value.device_ptr()) if out_value is not None else None,
        C.c_void_p(out_index.device_ptr()), C.c_void_p(ws.device_ptr()), ws.size))


_VALUE_OPS = {"sum": N.REDUCE_SUM, "mean": N.REDUCE_MEAN, "max": N.REDUCE_MAX, "min": N.REDUCE_MIN, "prod": N.REDUCE_PROD}
_INDEX_OPS = {"argmax": N.REDUCE_ARGMAX, "argmin": N.REDUCE_ARGMIN}


def _op_code(op, table, what: str) -> int:
    if isinstance(op, str):
        if op not in table:
            raise ServerError(N.E_UNSUPPORTED, f"{what}: unknown operation '{op}' (one of {sorted(table)})")
        return table[op]
    return int(op)


def reduce(client: ComputeClient, input: TensorHandle, output: TensorHandle, op="sum") -> None:
    """Array-wide value reduction into output[0] (f32): op = "sum" | "mean" | "max" | "min" | "prod" (or a MI355_REDUCE_* code).
    max / min: NaN if any element is NaN, -0 < +0 (mi355_reduce, include/mi355cube.h)."""
    input, n = _consumable(client, input, _require_flat_f32, "reduce")
    ws = _workspace(client, n)
    client._s.check(client.lib.mi355_reduce(client.ctx, client.on(input, output, ws), C.c_void_p(input.device_ptr()), int(input.dtype), n,
                                            _op_code(op, _VALUE_OPS, "reduce"), C.c_void_p(output.device_ptr()), C.c_void_p(ws.device_ptr()), ws.size))


def argreduce(client: ComputeClient, input: TensorHandle, out_index: TensorHandle, out_value: Optional[TensorHandle] = None,
              op="argmax") -> None:
    """Array-wide index reduction: op = "argmax" | "argmin"; out_index[0] (u64) = lowest index of the extremum, NaN wins, -0 == +0."""
    input, n = _consumable(client, input, _require_flat_f32, "argreduce")
    ws = _workspace(client, n)
    client._s.check(client.lib.mi355_argreduce(
        client.ctx, client.on(input, out_value, out_index, ws), C.c_void_p(input.device_ptr()), int(input.dtype), n, _op_code(op, _INDEX_OPS, "argreduce"),
        C.c_void_p(out_value.device_ptr()) if out_value is not None else None,
        C.c_void_p(out_index.device_ptr()), C.c_void_p(ws.device_ptr()), ws.size))


def argmin(client: ComputeClient, input: TensorHandle, out_index: TensorHandle, out_value: Optional[TensorHandle] = None) -> None:
    argreduce(client, input, out_index, out_value, "argmin")


def argmax_combine(client: ComputeClient, records: Handle, count: int, index_base, out_value: Optional[Handle],
                   out_index: Optional[Handle]) -> None:
    """The combine step of the multi-GPU argmax on the device (mi355_argmax_combine_f32): folds `count` gathered records
    {f32 value, u32 unused, u64 local index} -- rank order, as all_gather delivers them -- into (value, GLOBAL index) with
    the single-GPU rule; `index_base[r]` is the first element of shard r.  Queued on the client's stream."""
    base = (C.c_uint64 * max(count, 1))(*[int(b) for b in (index_base or [0] * count)])
    client._s.check(client.lib.mi355_argmax_combine_f32(
        client.ctx, client.on(records, out_value, out_index), C.c_void_p(records.device_ptr()), count, base,
        C.c_void_p(out_value.device_ptr()) if out_value is not None else None,
        C.c_void_p(out_index.device_ptr()) if out_index is not None else None))


def sum_argmax_combine(client: ComputeClient, records: Handle, count: int, index_base, out_sum: Optional[Handle],
                       out_value: Optional[Handle], out_index: Optional[Handle]) -> None:
    """The whole combine step of the sharded sum + argmax on the device (mi355_sum_argmax_combine_f32): folds `count` gathered
    records {f32 value, f32 partial sum, u64 local index} -- rank order, as ONE all_gather delivers them -- into the global
    sum (partial sums added in rank order: the same bits on every rank) and (value, GLOBAL index) with the single-GPU rule."""
    base = (C.c_uint64 * max(count, 1))(*[int(b) for b in (index_base or [0] * count)])
    client._s.check(client.lib.mi355_sum_argmax_combine_f32(
        client.ctx, client.on(records, out_sum, out_value, out_index), C.c_void_p(records.device_ptr()), count, base,
        C.c_void_p(out_sum.device_ptr()) if out_sum is not None else None,
        C.c_void_p(out_value.device_ptr()) if out_value is not None else None,
        C.c_void_p(out_index.device_ptr()) if out_index is not None else None))


def _rows_view(t: TensorHandle, what: str):
    if t.dtype not in (ElemType.F32, ElemType.BF16, ElemType.F16):
        raise ServerError(N.E_UNSUPPORTED, f"{what}: input must be f32, bf16 or f16")
    if t.rank() == 0:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: rank-0 input")
    cols = t.shape[-1]
    rows = t.num_elems() // cols if cols else 0
    if t.strides[-1] != 1 and cols > 1:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: last axis must have unit stride")
    row_stride = t.strides[-2] if t.rank() >= 2 else cols
    # leading dims must collapse onto one row stride (pitched row-major is fine)
    acc = row_stride
    for i in range(t.rank() - 3, -1, -1):
        acc *= t.shape[i + 1]
        if t.strides[i] != acc and t.shape[i] != 1:
            raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: leading dims are not collapsible")
    return rows, cols, row_stride


def reduce_sum_last_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle) -> None:
    """The book's reduce_matrix (cubecl-book/src/getting-started/src/bin/v1-cpu.rs:7-15):
    output shape = input shape minus the last axis."""
    input, (rows, cols, stride) = _consumable(client, input, _rows_view, "reduce_sum_last_axis")
    client._s.check(client.lib.mi355_reduce_last_axis_sum(
        client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype), C.c_void_p(output.device_ptr()), rows, cols, stride))


def argmax_last_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle) -> None:
    input, (rows, cols, stride) = _consumable(client, input, _rows_view, "argmax_last_axis")
    client._s.check(client.lib.mi355_reduce_last_axis_argmax(
        client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype), C.c_void_p(output.device_ptr()), rows, cols, stride))


def _axis_view(t: TensorHandle, axis: int, what: str):
    if t.dtype not in (ElemType.F32, ElemType.BF16, ElemType.F16):
        raise ServerError(N.E_UNSUPPORTED, f"{what}: input must be f32, bf16 or f16")
    if not t.is_contiguous():
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: input must be contiguous")
    rank = t.rank()
    if not -rank <= axis < rank:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: axis {axis} out of range for rank {rank}")
    axis %= rank
    outer = inner = 1
    for d in t.shape[:axis]:
        outer *= d
    for d in t.shape[axis + 1:]:
        inner *= d
    return outer, t.shape[axis], inner


def reduce_sum_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle, axis: int) -> None:
    """Sum over one axis: output shape = input shape minus that axis (any axis; a strided view is made contiguous first)."""
    input, (outer, red, inner) = _consumable(client, input, lambda t, w: _axis_view(t, axis, w), "reduce_sum_axis")
    client._s.check(client.lib.mi355_reduce_axis_sum(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype),
                                                     C.c_void_p(output.device_ptr()), outer, red, inner))


def argmax_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle, axis: int) -> None:
    """Argmax over one axis (u32 indices along that axis; lowest index wins ties, NaN ranks highest)."""
    input, (outer, red, inner) = _consumable(client, input, lambda t, w: _axis_view(t, axis, w), "argmax_axis")
    client._s.check(client.lib.mi355_reduce_axis_argmax(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype),
                                                        C.c_void_p(output.device_ptr()), outer, red, inner))


def reduce_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle, axis: int, op="sum") -> None:
    """Value reduction over one axis (f32 out): op = "sum" | "mean" | "max" | "min" | "prod"; output shape = input shape minus that axis."""
    input, (outer, red, inner) = _consumable(client, input, lambda t, w: _axis_view(t, axis, w), "reduce_axis")
    client._s.check(client.lib.mi355_reduce_axis(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype),
                                                 _op_code(op, _VALUE_OPS, "reduce_axis"), C.c_void_p(output.device_ptr()), outer, red, inner))


def argreduce_axis(client: ComputeClient, input: TensorHandle, output: TensorHandle, axis: int, op="argmax") -> None:
    """Index reduction over one axis (u32 indices along it): op = "argmax" | "argmin"; lowest index wins ties, NaN wins."""
    input, (outer, red, inner) = _consumable(client, input, lambda t, w: _axis_view(t, axis, w), "argreduce_axis")
    client._s.check(client.lib.mi355_argreduce_axis(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), int(input.dtype),
                                                    _op_code(op, _INDEX_OPS, "argreduce_axis"), C.c_void_p(output.device_ptr()), outer, red, inner))


def plane_reduce(client: ComputeClient, input: TensorHandle, output: TensorHandle, op: int, active: int = 64) -> None:
    """plane_sum / plane_prod / plane_max / plane_min / inclusive / exclusive sum and product over 64-lane planes."""
    n = input.num_elems()
    client._s.check(client.lib.mi355_plane_reduce_f32(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()),
                                                      C.c_void_p(output.device_ptr()), n, active, op))


def plane_op(client: ComputeClient, input: TensorHandle, output: TensorHandle, op: int, plane: int = 64, arg: int = 0) -> None:
    """plane_all / plane_any / plane_elect / plane_broadcast / plane_shuffle / _xor / _up / _down / plane_ballot
    (crates/cubecl-core/src/frontend/plane.rs:62-216, :388-440) over planes of `plane` lanes (32 or 64).  `output` holds one f32
    per input, except for PLANE_BALLOT: 4 x u32 per plane."""
    n = input.num_elems()
    client._s.check(client.lib.mi355_plane_op_f32(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()),
                                                  C.c_void_p(output.device_ptr()), n, plane, op, arg))


def identity(client: ComputeClient, output: TensorHandle) -> None:
    """tensor::identity::launch (crates/cubecl-std/src/tensor/identity.rs:36-84): `output`, a square matrix (possibly with
    pitched rows), becomes the identity matrix of its dtype."""
    if output.rank() != 2:
        raise ServerError(N.E_INVALID_ARGUMENT, "identity: input should be a matrix")
    if output.shape[0] != output.shape[1]:
        raise ServerError(N.E_INVALID_ARGUMENT, "identity: input should be a square matrix")
    if output.strides[1] != 1 and output.shape[1] > 1:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, "identity: the matrix must be row-major")
    client._s.check(client.lib.mi355_fill_identity(client.ctx, client.on(output), C.c_void_p(output.device_ptr()), int(output.dtype),
                                                   output.shape[0], max(output.strides[0], output.shape[1])))


# ---- strided copies (crates/cubecl-std/src/tensor/contiguous/) -------------------------------------------------------
def copy_into(client: ComputeClient, input: TensorHandle, output: TensorHandle) -> None:
    """copy_into (contiguous/launch.rs:40-56): element q of `input`'s linear view goes to element q of `output`'s linear
    layout.  Both may be strided, and they may differ in rank as long as they hold the same number of elements."""
    if input.dtype.size() != output.dtype.size():
        raise ServerError(N.E_INVALID_ARGUMENT, "copy_into: element sizes differ")
    li, lo = N.TensorLayout.of(input.shape, input.strides), N.TensorLayout.of(output.shape, output.strides)
    client._s.check(client.lib.mi355_copy_strided(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), C.byref(li),
                                                  C.c_void_p(output.device_ptr()), C.byref(lo), input.dtype.size()))


def copy_plan(client: ComputeClient, input: TensorHandle, output: TensorHandle):
    """-> (path, bytes per access) copy_into takes for these two views (host-side only)."""
    li, lo = N.TensorLayout.of(input.shape, input.strides), N.TensorLayout.of(output.shape, output.strides)
    path, access = C.c_int32(), C.c_int32()
    rc = client.lib.mi355_copy_strided_plan(C.c_void_p(input.device_ptr()), C.byref(li), C.c_void_p(output.device_ptr()), C.byref(lo),
                                            input.dtype.size(), C.byref(path), C.byref(access))
    if rc != N.OK:
        raise ServerError(rc, "copy_plan: the two views cannot be copied into each other")
    return path.value, access.value


def into_contiguous(client: ComputeClient, input: TensorHandle) -> TensorHandle:
    """into_contiguous (contiguous/launch.rs:5-20): a new contiguous tensor with the view's elements."""
    handle = client.empty(input.num_elems() * input.dtype.size())
    output = TensorHandle.new_contiguous(input.shape, handle, input.dtype)
    copy_into(client, input, output)
    return output


def into_contiguous_pitched(client: ComputeClient, input: TensorHandle) -> TensorHandle:
    """into_contiguous_pitched (contiguous/launch.rs:22-37): like into_contiguous, rows padded to the pitch that
    ComputeClient::empty_tensor picks."""
    if input.rank() <= 1:
        return into_contiguous(client, input)
    output = TensorHandle.empty(client, input.shape, input.dtype)
    copy_into(client, input, output)
    return output


def into_contiguous_packed(client: ComputeClient, input: TensorHandle, packed_dim: int, shape, packing: int) -> TensorHandle:
    """into_contiguous_packed (contiguous/base.rs:254-293): `input` stores `packing` sub-word values per u32 / u8 word,
    packed along axis rank - 1 - packed_dim of the logical `shape`; the result stores the same values packed along the
    innermost axis."""
    rank = len(shape)
    if rank <= 1:
        return into_contiguous(client, input)
    out_shape = list(shape)
    out_shape[-1] = -(-out_shape[-1] // packing)
    output = TensorHandle.empty(client, out_shape, input.dtype)
    li, lo = N.TensorLayout.of(input.shape, input.strides), N.TensorLayout.of(output.shape, output.strides)
    logical = (C.c_int64 * rank)(*[int(d) for d in shape])
    client._s.check(client.lib.mi355_copy_packed(client.ctx, client.on(input, output), C.c_void_p(input.device_ptr()), C.byref(li),
                                                 C.c_void_p(output.device_ptr()), C.byref(lo), logical, packed_dim, packing,
                                                 input.dtype.size()))
    return output


# ---- a linear layer's epilogue, norms, clipping ------------------------------------------------------------------------
_ACTIVATIONS = {"none": N.ACT_NONE, "relu": N.ACT_RELU, "gelu": N.ACT_GELU, "gelu_tanh": N.ACT_GELU_TANH, "silu": N.ACT_SILU}


def _activation(name, what: str) -> int:
    if name not in _ACTIVATIONS:
        raise ServerError(N.E_UNSUPPORTED, f"{what}: unknown activation '{name}' (one of {sorted(_ACTIVATIONS)})")
    return _ACTIVATIONS[name]


def _ptr(t):
    return None if t is None else t.device_ptr()


def _batched(t: TensorHandle, tail: int, batch: int, what: str):
    """(elements between batch entries, 0 for one that all entries share) of a [.., tail] operand that goes with `batch` matrices."""
    if len(t.shape) == tail:
        return 0
    lead = math.prod(t.shape[:t.rank() - tail])
    if lead == 1:
        return 0
    if lead != batch:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: batch {lead} does not broadcast to {batch}")
    dims = [(d, s) for d, s in zip(t.shape[:t.rank() - tail], t.strides) if d != 1]
    for (_, s_out), (d_in, s_in) in zip(dims[:-1], dims[1:]):
        if s_out != s_in * d_in:
            raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: batch dims are not collapsible")
    return dims[-1][1]


def _vector(client: ComputeClient, t: TensorHandle, n: int, batch: int, what: str):
    """-> (tensor, element stride, batch stride) of a per-row or per-column operand: [n] or [batch.., n], or one value for all."""
    if t.shape == (n,) and n > 1 and t.strides[0] >= 0:
        return t, t.strides[0], 0
    if t.num_elems() == 1:
        return t, 0, 0
    if t.shape[-1] != n:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: shape {t.shape} does not give {n} values")
    if t.strides[-1] < 0:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: negative stride")
    try:
        return t, (t.strides[-1] if n > 1 else 0), _batched(t, 1, batch, what)
    except ServerError as e:
        if e.code != N.E_UNSUPPORTED_STRIDES:
            raise
    t = into_contiguous(client, t)
    return t, (1 if n > 1 else 0), _batched(t, 1, batch, what)


def _rows_of_matrix(t: TensorHandle, batch: int, what: str):
    """(leading dimension, batch stride) of a row-major [.., rows, cols] tensor."""
    rows, cols = t.shape[-2], t.shape[-1]
    if cols > 1 and t.strides[-1] != 1:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: rows must be contiguous")
    ld = t.strides[-2] if rows > 1 else max(cols, t.strides[-2])
    if ld < cols:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: rows overlap")
    return ld, _batched(t, 2, batch, what)


def matmul_fused(client: ComputeClient, lhs: TensorHandle, rhs: TensorHandle, out: TensorHandle, *, bias: Optional[TensorHandle] = None,
                 activation: str = "none", residual: Optional[TensorHandle] = None, lhs_scale: Optional[TensorHandle] = None,
                 rhs_scale: Optional[TensorHandle] = None, pre_activation: Optional[TensorHandle] = None, algo: int = N.GEMM_ALGO_AUTO) -> None:
    """out = act(lhs_scale[m] * rhs_scale[n] * (lhs @ rhs) + bias[n]) + residual: matmul with a linear layer's epilogue, formed in f32 and
    rounded once to out's dtype (mi355_gemm_fused).

    lhs, rhs and out as `matmul` takes them.  `activation`: "none" | "relu" | "gelu" | "gelu_tanh" | "silu".  `bias`: [n] or [batch.., n], f32 or
    out's dtype.  `residual`: out's shape and dtype (any strides; may be `out` itself).  `lhs_scale` / `rhs_scale`: f32, one value, [m] / [n] or
    [batch.., m] / [batch.., n] -- what quantising the rows of lhs and the columns of rhs to 8 bits left behind.  `pre_activation`: if given,
    receives the activation's argument in out's shape and dtype, for matmul_fused_backward."""
    m, k = lhs.shape[-2], lhs.shape[-1]
    k2, n = rhs.shape[-2], rhs.shape[-1]
    if k != k2 or out.rank() < 2 or out.shape[-2] != m or out.shape[-1] != n:
        raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_fused: shape mismatch {lhs.shape} x {rhs.shape} -> {out.shape}")
    if lhs.dtype != rhs.dtype:
        raise ServerError(N.E_INVALID_ARGUMENT, "matmul_fused: lhs/rhs dtypes differ")
    act = _activation(activation, "matmul_fused")
    for t, name in ((residual, "residual"), (pre_activation, "pre_activation")):
        if t is not None and (tuple(t.shape) != tuple(out.shape) or t.dtype != out.dtype):
            raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_fused: {name} must have out's shape and dtype")
    for t, name in ((lhs_scale, "lhs_scale"), (rhs_scale, "rhs_scale")):
        if t is not None and t.dtype != ElemType.F32:
            raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_fused: {name} must be f32")
    lhs, (ta, lda, ba, sa) = _kernel_ready(client, lhs, "lhs")
    rhs, (tb, ldb, bb, sb) = _kernel_ready(client, rhs, "rhs")
    batch = math.prod(out.shape[:-2])
    if out.num_elems() == 0:
        return
    ldc, sc = _rows_of_matrix(out, batch, "matmul_fused: out")
    for b, name in ((ba, "lhs"), (bb, "rhs")):
        if b not in (1, batch):
            raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_fused: {name} batch {b} does not broadcast to {batch}")
    ep = N.GemmEpilogue(activation=act)
    if bias is not None:
        bias, inc, ep.stride_bias = _vector(client, bias, n, batch, "matmul_fused: bias")
        if inc != 1 and n > 1:                      # the kernels read it in rows of n
            if bias.num_elems() == 1:
                raise ServerError(N.E_INVALID_ARGUMENT, f"matmul_fused: bias of shape {bias.shape} does not give {n} values")
            bias = into_contiguous(client, bias)
            ep.stride_bias = _batched(bias, 1, batch, "matmul_fused: bias")
        ep.bias, ep.dtype_bias = bias.device_ptr(), int(bias.dtype)
    if residual is not None:
        try:
            ep.ld_residual, ep.stride_residual = _rows_of_matrix(residual, batch, "matmul_fused: residual")
        except ServerError as e:
            if e.code != N.E_UNSUPPORTED_STRIDES:
                raise
            residual = into_contiguous(client, residual)
            ep.ld_residual, ep.stride_residual = _rows_of_matrix(residual, batch, "matmul_fused: residual")
        ep.residual = residual.device_ptr()
    if lhs_scale is not None:
        lhs_scale, ep.inc_row_scale, ep.stride_row_scale = _vector(client, lhs_scale, m, batch, "matmul_fused: lhs_scale")
        ep.row_scale = lhs_scale.device_ptr()
    if rhs_scale is not None:
        rhs_scale, ep.inc_col_scale, ep.stride_col_scale = _vector(client, rhs_scale, n, batch, "matmul_fused: rhs_scale")
        ep.col_scale = rhs_scale.device_ptr()
    if pre_activation is not None:
        ep.ld_pre, ep.stride_pre = _rows_of_matrix(pre_activation, batch, "matmul_fused: pre_activation")
        ep.pre = pre_activation.device_ptr()
    desc = N.GemmDesc(m=m, n=n, k=k, batch=batch, lda=lda, ldb=ldb, ldc=ldc, stride_a=sa if ba == batch else 0, stride_b=sb if bb == batch else 0,
                      stride_c=sc, dtype_ab=int(lhs.dtype), dtype_c=int(out.dtype), trans_a=int(ta), trans_b=int(tb), algo=algo)
    client._s.check(client.lib.mi355_gemm_fused(
        client.ctx, client.on(lhs, rhs, out, bias, residual, lhs_scale, rhs_scale, pre_activation), C.byref(desc), C.byref(ep),
        lhs.device_ptr(), rhs.device_ptr(), out.device_ptr()))


def _swap_last(t: TensorHandle) -> TensorHandle:
    return t.permute(tuple(range(t.rank() - 2)) + (t.rank() - 1, t.rank() - 2))


def _as_rows(client: ComputeClient, t: TensorHandle) -> TensorHandle:
    """[batch.., rows, cols] as one [batch * rows, cols] matrix, copied only where the batch does not follow on from the rows."""
    if t.rank() == 2:
        return t
    rows, cols = math.prod(t.shape[:-1]), t.shape[-1]
    dims = [(d, s) for d, s in zip(t.shape[:-1], t.strides[:-1]) if d != 1]
    ld = dims[-1][1] if dims else cols
    # (rows that overlap -- an operand broadcast along them -- have no leading dimension)
    if ld < cols or (cols > 1 and t.strides[-1] != 1) or any(s_out != s_in * d_in for (_, s_out), (d_in, s_in) in zip(dims[:-1], dims[1:])):
        t, ld = into_contiguous(client, t), cols
    return TensorHandle.new(t.handle, (rows, cols), (ld, 1), t.dtype)


def matmul_fused_backward(client: ComputeClient, grad_out: TensorHandle, pre_activation: Optional[TensorHandle], grad_pre: Optional[TensorHandle], *,
                          activation: str = "none", grad_bias: Optional[TensorHandle] = None, lhs: Optional[TensorHandle] = None,
                          rhs: Optional[TensorHandle] = None, grad_lhs: Optional[TensorHandle] = None, grad_rhs: Optional[TensorHandle] = None) -> None:
    """The gradient of matmul_fused (without scales):

        grad_pre = grad_out * act'(pre_activation)    grad_bias = sum of grad_pre over rows (and over a batch that shares the bias)
        grad_lhs = grad_pre @ rhs^T                   grad_rhs = lhs^T @ grad_pre

    and the residual's gradient is grad_out itself.  Outputs that are not given are not computed; grad_pre (grad_out's shape and dtype, f32, bf16
    or f16; may be grad_out or pre_activation itself) is needed for the products, which take it as it is stored: each of
    their terms carries half a step of its type (bf16 2^-8, f16 2^-11 relative), as the products of stored gradients do.  grad_bias sums it before
    its rounding.
    `pre_activation` may be None for activation "none".  grad_bias: [n] or [batch.., n], f32 or grad_out's dtype.  An operand that matmul_fused
    broadcast over the batch gets the sum over the batch."""
    what = "matmul_fused_backward"
    act = _activation(activation, what)
    if grad_out.rank() < 2:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_out must have rank >= 2")
    m, n = grad_out.shape[-2:]
    batch = math.prod(grad_out.shape[:-2])
    for t, name in ((pre_activation, "pre_activation"), (grad_pre, "grad_pre")):
        if t is not None and (tuple(t.shape) != tuple(grad_out.shape) or t.dtype != grad_out.dtype):
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: {name} must have grad_out's shape and dtype")
    if pre_activation is None and act != N.ACT_NONE:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: activation '{activation}' needs pre_activation")
    for t, of, grad, name in ((rhs, lhs, grad_lhs, "lhs"), (lhs, rhs, grad_rhs, "rhs")):
        if grad is None:
            continue
        if t is None or grad_pre is None:
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_{name} needs grad_pre and the other operand")
        if t.dtype != grad_out.dtype or grad.dtype not in (grad_out.dtype, ElemType.F32):
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: the operands must have grad_out's dtype, grad_{name} that or f32")
        if of is not None and tuple(of.shape) != tuple(grad.shape):
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_{name} must have {name}'s shape")
    if grad_lhs is not None and (grad_lhs.shape[-2] != m or rhs.shape[-1] != n or grad_lhs.shape[-1] != rhs.shape[-2]):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: shape mismatch {grad_lhs.shape} x {rhs.shape} -> {grad_out.shape}")
    if grad_rhs is not None and (lhs.shape[-2] != m or grad_rhs.shape[-1] != n or grad_rhs.shape[-2] != lhs.shape[-1]):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: shape mismatch {lhs.shape} x {grad_rhs.shape} -> {grad_out.shape}")
    for t, name in ((rhs if grad_lhs is not None else None, "rhs"), (lhs if grad_rhs is not None else None, "lhs"), (grad_lhs, "grad_lhs"), (grad_rhs, "grad_rhs")):
        if t is not None and t.num_elems() // max(t.shape[-2] * t.shape[-1], 1) not in (1, batch) and t.num_elems():
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: {name} does not broadcast to batch {batch}")

    # what one launch writes before another one reads (each launch checks its own operands)
    late = [(t, *_extent(t)) for t, wanted in ((rhs, grad_lhs), (lhs, grad_rhs)) if wanted is not None]
    outs = [(t, *_extent(t)) for t in (grad_pre, grad_bias, grad_lhs, grad_rhs) if t is not None] if late else []
    for i, (o, first, end) in enumerate(outs):
        for t, t_first, t_end in late + outs[:i]:
            if first < t_end and t_first < end and _meshed(o, t, t_first - first):
                raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: an output overlaps an operand or another output")

    def rows(t, name, writable=False):
        try:
            return t, _rows_of_matrix(t, batch, f"{what}: {name}")
        except ServerError as e:
            if writable or e.code != N.E_UNSUPPORTED_STRIDES:
                raise
        t = into_contiguous(client, t)
        return t, _rows_of_matrix(t, batch, f"{what}: {name}")

    desc = N.GemmFusedGradDesc(m=m, n=n, batch=batch, dtype=int(grad_out.dtype), activation=act)
    z = None
    if grad_out.num_elems():
        g, (desc.ld_out, desc.stride_out) = rows(grad_out, "grad_out")
        if act != N.ACT_NONE:
            z, (desc.ld_pre, desc.stride_pre) = rows(pre_activation, "pre_activation")
        if grad_pre is not None:
            _, (desc.ld_grad, desc.stride_grad) = rows(grad_pre, "grad_pre", writable=True)
    else:
        g = grad_out
    ws, need = None, C.c_uint64()
    if grad_bias is not None:
        if not grad_bias.is_contiguous() or grad_bias.rank() < 1 or grad_bias.shape[-1] != n:
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_bias must be contiguous, [n] or [batch.., n] (got {grad_bias.shape}, n = {n})")
        entries = grad_bias.num_elems() // n if n else 1
        if entries not in (1, batch):
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_bias has {entries} entries for batch {batch}")
        if grad_bias.num_elems() == 0:              # one bias an entry, and no entries: nothing to write
            grad_bias = None
    if grad_bias is not None:
        desc.dtype_bias, desc.batch_bias = int(grad_bias.dtype), int(entries == batch and batch > 1)
        client._s.check(client.lib.mi355_gemm_fused_grad_workspace_bytes(C.byref(desc), C.byref(need)))
        if need.value:
            ws = client.empty(need.value)
    client._s.check(client.lib.mi355_gemm_fused_grad(
        client.ctx, client.on(g, z, grad_pre, grad_bias, ws), C.byref(desc), g.device_ptr(), _ptr(z), _ptr(grad_pre), _ptr(grad_bias),
        _ptr(ws), need.value))
    if grad_lhs is not None:
        lead = grad_lhs.num_elems() // (m * grad_lhs.shape[-1]) if grad_lhs.num_elems() else batch
        if lead == batch or grad_lhs.num_elems() == 0:
            matmul_fused(client, grad_pre, _swap_last(rhs), _with_batch_of(grad_lhs, grad_out))
        else:                                       # one lhs for all entries: their sum, in f32 until the last
            _sum_of_products(client, [(_entry(grad_pre, b), _swap_last(_entry(rhs, b))) for b in range(batch)], grad_lhs)
    if grad_rhs is not None:
        lead = grad_rhs.num_elems() // (n * grad_rhs.shape[-2]) if grad_rhs.num_elems() else batch
        left_lead = lhs.num_elems() // (m * lhs.shape[-1]) if lhs.num_elems() else batch
        if lead == batch or grad_rhs.num_elems() == 0:
            matmul_fused(client, _swap_last(lhs), grad_pre, _with_batch_of(grad_rhs, grad_out))
        elif left_lead == batch:                    # one rhs for all entries: their rows under each other are one product
            matmul_fused(client, _swap_last(_as_rows(client, lhs)), _as_rows(client, grad_pre), _entry(grad_rhs, 0))
        else:
            _sum_of_products(client, [(_swap_last(_entry(lhs, b)), _entry(grad_pre, b)) for b in range(batch)], grad_rhs)


def _extent(t: TensorHandle):
    """(first byte, one past the last); empty for an empty tensor."""
    first, last = t.device_ptr(), 0
    for d, s in zip(t.shape, t.strides):
        if d == 0:
            return first, first
        last += (d - 1) * s
    return first, first + (last + 1) * t.dtype.size()


def _meshed(a: TensorHandle, b: TensorHandle, distance: int) -> bool:
    """Of two tensors whose extents meet, b `distance` bytes after a: do they share a byte?  False for column ranges of the same wider rows that
    lie beside each other; other views that mesh without touching are taken as sharing."""
    for t in (a, b):
        if t.rank() < 2 or t.strides[-1] != 1 or any(t.strides[i] != t.strides[i + 1] * t.shape[i + 1] for i in range(t.rank() - 2)):
            return True
    ld = a.strides[-2] * a.dtype.size()
    if ld == 0 or ld != b.strides[-2] * b.dtype.size():
        return True
    at = distance % ld
    return at < a.shape[-1] * a.dtype.size() or at + b.shape[-1] * b.dtype.size() > ld


def _with_batch_of(t: TensorHandle, model: TensorHandle) -> TensorHandle:
    """`t` with model's rank: axes of one in front where it has fewer."""
    extra = model.rank() - t.rank()
    if extra <= 0:
        return t
    return TensorHandle.new(t.handle, (1,) * extra + tuple(t.shape), (t.shape[-2] * t.strides[-2],) * extra + tuple(t.strides), t.dtype)


def _entry(t: TensorHandle, b: int) -> TensorHandle:
    """Matrix `b` of a batch (the only one of a tensor that the batch shares)."""
    offset, lead = 0, t.num_elems() // max(t.shape[-2] * t.shape[-1], 1)
    if lead > 1:
        for d, s in zip(reversed(t.shape[:-2]), reversed(t.strides[:-2])):
            offset += (b % d) * s
            b //= d
    return TensorHandle.new(t.handle.offset_start_by(offset * t.dtype.size()), t.shape[-2:], t.strides[-2:], t.dtype)


def _sum_of_products(client: ComputeClient, pairs, out: TensorHandle) -> None:
    """out = sum of the products, accumulated in f32 and rounded once; zeros where there are none (a batch of no entries)."""
    out = _entry(out, 0)
    rows, cols = out.shape
    pairs = pairs or [(TensorHandle.new_contiguous((rows, 0), client.empty(4), ElemType.F32), TensorHandle.new_contiguous((0, cols), client.empty(4), ElemType.F32))]
    total = TensorHandle.new_contiguous(out.shape, client.empty(out.num_elems() * 4), ElemType.F32)
    for i, (a, b) in enumerate(pairs):
        matmul(client, a, b, total, acc=total if i else None)
    if out.dtype != ElemType.F32:
        rounded = TensorHandle.new_contiguous(out.shape, client.empty(out.num_elems() * out.dtype.size()), out.dtype)
        client._s.check(client.lib.mi355_cast(client.ctx, client.on(total, rounded), total.device_ptr(), int(ElemType.F32),
                                              rounded.device_ptr(), int(out.dtype), out.num_elems()))
        total = rounded
    copy_into(client, total, out)


def _norm_rows(t: TensorHandle, what: str):
    """(rows, cols, row stride) of a tensor whose last axis is the norm's; E_UNSUPPORTED_STRIDES where the rows do not collapse."""
    if len(t.shape) == 2 and t.strides[1] == 1 and t.strides[0] >= t.shape[1] > 0:
        return t.shape[0], t.shape[1], t.strides[0]
    if t.rank() == 0:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: rank-0 tensor")
    cols, rows = t.shape[-1], math.prod(t.shape[:-1])
    if rows == 0 or cols == 0:
        return rows, cols, cols
    if cols > 1 and t.strides[-1] != 1:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: last axis must have unit stride")
    dims = [(d, s) for d, s in zip(t.shape[:-1], t.strides[:-1]) if d != 1]
    for (_, s_out), (d_in, s_in) in zip(dims[:-1], dims[1:]):
        if s_out != s_in * d_in:
            raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: leading dims are not collapsible")
    stride = dims[-1][1] if dims else cols
    if stride < cols:
        raise ServerError(N.E_UNSUPPORTED_STRIDES, f"{what}: rows overlap")
    return rows, cols, stride


def _norm_operand(client: ComputeClient, t: Optional[TensorHandle], shape, dtype, what: str):
    """-> (operand, row stride); a view the kernels cannot walk goes through into_contiguous first."""
    if t is None:
        return None, 0
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: expected {tuple(shape)} {dtype.name}, got {tuple(t.shape)} {t.dtype.name}")
    if len(shape) == 2 and t.strides[1] == 1 and t.strides[0] >= shape[1] > 0:
        return t, t.strides[0]
    t, (_, _, stride) = _consumable(client, t, _norm_rows, what)
    return t, stride


def _flat(t: Optional[TensorHandle], shape, dtypes, what: str):
    """A contiguous operand of this shape (axes of one aside) and one of these dtypes."""
    if t is None or (t.shape == shape and t.strides == (1,) and t.dtype in dtypes):
        return t
    if ([d for d in t.shape if d != 1] != [d for d in shape if d != 1] or t.dtype not in dtypes or not t.is_contiguous()):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: expected contiguous {tuple(shape)} {'/'.join(d.name for d in dtypes)}, got {tuple(t.shape)} {t.dtype.name}")
    return t


_FP8 = (ElemType.F8E4M3, ElemType.F8E5M2)


def rms_norm(client: ComputeClient, input: TensorHandle, weight: Optional[TensorHandle], output: TensorHandle, *, eps: float = 1e-6,
             residual: Optional[TensorHandle] = None, residual_out: Optional[TensorHandle] = None, scales: Optional[TensorHandle] = None,
             rstd: Optional[TensorHandle] = None) -> None:
    """output = h * rstd * weight over the last axis, h = input + residual, rstd = 1 / sqrt(mean(h^2) + eps) (mi355_rms_norm).

    input, residual, residual_out (receives h; may be input or residual itself): f32, bf16 or f16, one shape.  `weight`: [cols], f32 or input's
    dtype, or None for ones.  `rstd`: f32, input's shape without the last axis (what rms_norm_backward wants).  output: input's dtype or f32; or
    F8E4M3 / F8E5M2, and then `scales` receives one F32 per row (shape without the last axis; matmul_fused's lhs_scale) or one UE8M0 per
    32 columns (shape [.., cols / 32]; matmul_scaled's lhs_scales), by its dtype."""
    what = "rms_norm"
    if input.dtype not in (ElemType.F32, ElemType.BF16, ElemType.F16):
        raise ServerError(N.E_UNSUPPORTED, f"{what}: input must be f32, bf16 or f16")
    if input.rank() == 0:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: rank-0 tensor")
    shape, cols = tuple(input.shape), input.shape[-1]
    f8 = output.dtype in _FP8
    if tuple(output.shape) != shape:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: output has shape {tuple(output.shape)}, input {shape}")
    if f8 != (scales is not None):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: an 8-bit output comes with scales, and only that")
    if not (0.0 < eps < float("inf")):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: eps must be positive and finite")
    x, ld_in = _norm_operand(client, input, shape, input.dtype, f"{what}: input")
    res, ld_res = _norm_operand(client, residual, shape, input.dtype, f"{what}: residual")
    if residual_out is not None and (tuple(residual_out.shape) != shape or residual_out.dtype != input.dtype):
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: residual_out must have input's shape and dtype")
    _flat(weight, (cols,), (ElemType.F32, input.dtype), f"{what}: weight")
    _flat(rstd, shape[:-1], (ElemType.F32,), f"{what}: rstd")
    rows, _, ld_out = _norm_rows(output, f"{what}: output")
    ld_hidden = _norm_rows(residual_out, f"{what}: residual_out")[2] if residual_out is not None else 0
    block, ld_scales = 0, 0
    if f8 and scales.dtype == ElemType.UE8M0:
        block = 32
        if cols % 32 or tuple(scales.shape) != shape[:-1] + (cols // 32,):
            raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: ue8m0 scales of shape {tuple(scales.shape)} for {shape} in blocks of 32")
        ld_scales = _norm_rows(scales, f"{what}: scales")[2]
    elif f8:
        _flat(scales, shape[:-1], (ElemType.F32,), f"{what}: scales")
    desc = N.RmsNormDesc(rows=rows, cols=cols, ld_in=ld_in, ld_residual=ld_res, ld_hidden=ld_hidden, ld_out=ld_out, ld_scales=ld_scales, eps=eps,
                         dtype=int(input.dtype), dtype_weight=int(weight.dtype) if weight is not None else N.DTYPE_F32, dtype_out=int(output.dtype),
                         scale_block=block)
    client._s.check(client.lib.mi355_rms_norm(
        client.ctx, client.on(x, res, weight, residual_out, output, scales, rstd), C.byref(desc), x.device_ptr(), _ptr(res), _ptr(weight),
        _ptr(residual_out), output.device_ptr(), _ptr(scales), _ptr(rstd)))


def rms_norm_backward(client: ComputeClient, grad_output: TensorHandle, hidden: TensorHandle, weight: Optional[TensorHandle], rstd: TensorHandle,
                      grad_input: TensorHandle, *, grad_weight: Optional[TensorHandle] = None, grad_hidden: Optional[TensorHandle] = None) -> None:
    """The gradient of rms_norm (mi355_rms_norm_grad), x^ = hidden * rstd:

        grad_input = rstd * (w g - x^ mean(w g x^)) + grad_hidden       grad_weight = sum over rows of g x^

    `hidden`: what rms_norm left in residual_out (its input where nothing was added); `rstd` as it left it.  grad_hidden: the gradient that
    reaches hidden by the residual stream.  grad_input is the gradient of rms_norm's input and of its residual; it may be grad_output,
    hidden or grad_hidden itself.  grad_weight: [cols], f32 or grad_output's dtype."""
    what = "rms_norm_backward"
    dt = grad_output.dtype
    if dt not in (ElemType.F32, ElemType.BF16, ElemType.F16):
        raise ServerError(N.E_UNSUPPORTED, f"{what}: operands must be f32, bf16 or f16")
    if grad_output.rank() == 0:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: rank-0 tensor")
    shape, cols = tuple(grad_output.shape), grad_output.shape[-1]
    g, ld_out = _norm_operand(client, grad_output, shape, dt, f"{what}: grad_output")
    h, ld_hidden = _norm_operand(client, hidden, shape, dt, f"{what}: hidden")
    s, ld_stream = _norm_operand(client, grad_hidden, shape, dt, f"{what}: grad_hidden")
    if tuple(grad_input.shape) != shape or grad_input.dtype != dt:
        raise ServerError(N.E_INVALID_ARGUMENT, f"{what}: grad_input must have grad_output's shape and dtype")
    _flat(weight, (cols,), (ElemType.F32, dt), f"{what}: weight")
    _flat(rstd, shape[:-1], (ElemType.F32,), f"{what}: rstd")
    _flat(grad_weight, (cols,), (ElemType.F32, dt), f"{what}: grad_weight")
    rows, _, ld_in = _norm_rows(grad_input, f"{what}: grad_input")
    desc = N.RmsNormGradDesc(rows=rows, cols=cols, ld_out=ld_out, ld_hidden=ld_hidden, ld_in=ld_in, ld_stream=ld_stream, dtype=int(dt),
                             dtype_weight=int(weight.dtype) if weight is not None else N.DTYPE_F32,
                             dtype_grad_weight=int(grad_weight.dtype) if grad_weight is not None else N.DTYPE_F32)
    ws, need = None, C.c_uint64()
    if grad_weight is not None:
        client._s.check(client.lib.mi355_rms_norm_grad_workspace_bytes(C.byref(desc), C.byref(need)))
        if need.value:
            ws = client.empty(need.value)
    client._s.check(client.lib.mi355_rms_norm_grad(
        client.ctx, client.on(g, h, weight, rstd, s, grad_input, grad_weight, ws), C.byref(desc), g.device_ptr(), _ptr(h),
        _ptr(weight), _ptr(rstd), _ptr(s), grad_input.device_ptr(), _ptr(grad_weight), _ptr(ws), need.value))


class TensorList:
    """Tensors that are used together (a model's gradients): f32, bf16 or f16, each contiguous or with padded rows.  Keep it as long as the
    tensors' memory: global_norm and clip_by_global_norm then take it without going through the tensors again."""

    def __init__(self, tensors):
        self.tensors = list(tensors)
        self.memories = list({id(t.handle.memory): t.handle for t in self.tensors}.values())    # one handle per allocation, for stream order
        self.spans = (N.TensorSpan * max(len(self.tensors), 1))()
        self.kinds = [(tuple(t.shape), t.dtype, t.is_contiguous()) for t in self.tensors]
        for i, t in enumerate(self.tensors):
            if t.dtype not in (ElemType.F32, ElemType.BF16, ElemType.F16):
                raise ServerError(N.E_UNSUPPORTED, f"TensorList: tensor {i} must be f32, bf16 or f16")
            if self.kinds[i][2]:
                self.spans[i] = (t.device_ptr(), 1, t.num_elems(), t.num_elems(), int(t.dtype), 0)
            else:
                rows, cols, stride = _norm_rows(t, f"TensorList: tensor {i}")
                self.spans[i] = (t.device_ptr(), rows, cols, stride, int(t.dtype), 0)

    def __len__(self) -> int:
        return len(self.tensors)


def _tensor_list(tensors) -> TensorList:
    return tensors if isinstance(tensors, TensorList) else TensorList(tensors)


def _norm_workspace(client: ComputeClient) -> Handle:
    need = C.c_uint64()
    client._s.check(client.lib.mi355_global_norm_workspace_bytes(C.byref(need)))
    return client.empty(need.value)                 # the pool's: stream-ordered, and a captured graph keeps its own


def global_norm(client: ComputeClient, tensors, output: TensorHandle) -> None:
    """output[0] (f32) = sqrt(sum of x^2 over all elements of all tensors), summed in f64 in a fixed order (mi355_global_norm).  `tensors`: a
    TensorList or any sequence of tensors."""
    tensors = _tensor_list(tensors)
    _flat(output, (1,), (ElemType.F32,), "global_norm: output")
    ws = _norm_workspace(client)
    client._s.check(client.lib.mi355_global_norm(client.ctx, client.on(*tensors.memories, output, ws), tensors.spans, len(tensors),
                                                 _ptr(output), ws.device_ptr(), ws.size))


def clip_by_global_norm(client: ComputeClient, tensors, max_norm: float, *, outputs=None, total_norm: Optional[TensorHandle] = None) -> None:
    """Every tensor times min(1, max_norm / norm), norm as global_norm gives it, in place or into `outputs` (shapes and dtypes alike)
    (mi355_clip_by_global_norm).  total_norm (f32) receives the norm.  A NaN or infinite norm makes every output NaN.  `tensors` and
    `outputs`: TensorLists or any sequences of tensors; no two of them may share memory, in place aside."""
    tensors = _tensor_list(tensors)
    outputs = tensors if outputs is None else _tensor_list(outputs)
    if not max_norm > 0.0:
        raise ServerError(N.E_INVALID_ARGUMENT, "clip_by_global_norm: max_norm must be positive")
    _flat(total_norm, (1,), (ElemType.F32,), "clip_by_global_norm: total_norm")
    if len(outputs) != len(tensors):
        raise ServerError(N.E_INVALID_ARGUMENT, f"clip_by_global_norm: {len(outputs)} outputs for {len(tensors)} tensors")
    ins, outs = tensors.spans, outputs.spans
    if outs is not ins:
        ins, outs = _span_pairs(tensors, outputs)
    ws = _norm_workspace(client)
    handles = tensors.memories if outputs is tensors else tensors.memories + outputs.memories
    client._s.check(client.lib.mi355_clip_by_global_norm(client.ctx, client.on(*handles, total_norm, ws), ins, outs, len(tensors), max_norm,
                                                         _ptr(total_norm), ws.device_ptr(), ws.size))


def _span_pairs(tensors: TensorList, outputs: TensorList):
    """The spans of both sides, walked the same way: where one of a pair is contiguous and the other has padded rows, both go by rows."""
    if tensors.kinds == outputs.kinds:
        return tensors.spans, outputs.spans
    for a, b in zip(tensors.kinds, outputs.kinds):
        if a[:2] != b[:2]:
            raise ServerError(N.E_INVALID_ARGUMENT, f"clip_by_global_norm: output {b[0]} {b[1].name} for {a[0]} {a[1].name}")
    sides = []
    for side in (tensors, outputs):
        spans = (N.TensorSpan * max(len(side), 1))()
        for i, t in enumerate(side.tensors):
            rows, cols, stride = _norm_rows(t, f"clip_by_global_norm: tensor {i}") if t.rank() else (1, 1, 1)
            spans[i] = (t.device_ptr(), rows, cols, stride, int(t.dtype), 0)
        sides.append(spans)
    return sides
