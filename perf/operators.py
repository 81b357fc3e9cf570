"""The operators around a linear layer that are measured: the fused matrix product and its gradient, the root-mean-square norm (with the
residual's addition and 8-bit output) and its gradient, and clipping by the global norm.

`own` says which side `run` computes: False, elementary torch operations in 32 bits (64 where 32 lose what matters), rounded once at the
end; True, the calls a user makes of cubecl_amd.  Both work on what `prepare` laid out: device tensors, and on the framework's side the
TensorHandles over memory of its own pool that such a program keeps."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2,
         "ue8m0": torch.float8_e8m0fnu}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}     # largest finite value of the 8-bit type = 0.875 * 2^TOP_EXP
TOP_EXP = {"e4m3": 9, "e5m2": 16}
BLOCK = 32                                 # values per ue8m0 scale, what matmul_scaled takes
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------------------------------------------
def matmul(m, n, k, dtype, out, act, bias, residual, pre, rhs):
    return {"op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "out": out, "act": act, "bias": bias, "residual": residual, "pre": pre, "rhs": rhs}


def matmul_grad(m, n, k, dtype, act):
    return {"op": "matmul_grad", "m": m, "n": n, "k": k, "dtype": dtype, "act": act}


def norm(rows, cols, dtype, out, scales, residual):
    return {"op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "out": out, "scales": scales, "residual": residual}


def norm_grad(rows, cols, dtype, stream):
    return {"op": "norm_grad", "rows": rows, "cols": cols, "dtype": dtype, "stream": stream}


def clip(layers, width, vocab, dtype, max_norm):
    return {"op": "clip", "layers": layers, "width": width, "vocab": vocab, "dtype": dtype, "max_norm": max_norm}


def listed():
    return [
        # one token through a projection whose weight is stored [n, k]: reading the weight once is all there is to it
        dict(matmul(1, 8192, 4096, "bf16", "bf16", "silu", True, True, False, "nk"), name="linear 1 token"),
        # the up projection of a training step, row-major weight; the pre-activation is kept for the backward pass
        dict(matmul(4096, 8192, 2048, "bf16", "bf16", "gelu_tanh", True, False, True, "kn"), name="linear train gelu"),
        # the largest product of the repository's own benchmark with bias and residual: what the epilogue adds to a full chip
        dict(matmul(8192, 8192, 8192, "bf16", "bf16", "none", True, True, False, "nk"), name="linear 8192 residual"),
        # a prefill of odd length on 8-bit operands: one scale a row of activations, one a column of the weight
        dict(matmul(1777, 4096, 4096, "e4m3", "bf16", "silu", True, True, False, "nk"), name="linear fp8 prefill"),
        # the backward pass of the training step above
        dict(matmul_grad(4096, 8192, 2048, "bf16", "gelu_tanh"), name="linear grad train"),
        # odd sizes in 32 bits, rows that are not 16-byte aligned
        dict(matmul_grad(333, 517, 1001, "f32", "gelu"), name="linear grad odd f32"),
        # a few decoded tokens ahead of an 8-bit projection: latency
        dict(norm(4, 8192, "bf16", "e4m3", "row", True), name="norm decode fp8"),
        # a prefill ahead of a block-scaled projection: bandwidth
        dict(norm(16384, 4096, "bf16", "e4m3", "block", True), name="norm prefill mx"),
        # the training step's norm, the residual stream's gradient added on the way
        dict(norm_grad(16384, 4096, "bf16", True), name="norm grad train"),
        # odd sizes
        dict(norm_grad(777, 1001, "f16", False), name="norm grad odd f16"),
        # a model of 24 layers and 0.29 billion parameters, weights in bf16 and norms in f32
        dict(clip(24, 1024, 32768, "bf16", 1.0), name="clip 24 layers"),
        # an adapter's worth of small tensors: launches and latency
        dict(clip(4, 96, 1000, "f32", 1.0), name="clip small"),
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v if rng.random() < 0.5 else (v + 31) // 32 * 32))

    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    op = rng.choice(["matmul", "matmul", "matmul_grad", "norm", "norm_grad", "clip"])
    if op == "matmul":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "e4m3"])
        out = rng.choice(["bf16", "f16"]) if dtype == "e4m3" else rng.choice([dtype, dtype, "f32"])
        m, n, k = size(1, 8192), size(16, 8192), size(16, 8192)
        return matmul(m, n, k, dtype, out, act, rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.3, "nk" if dtype == "e4m3" else rng.choice(["nk", "kn"]))
    if op == "matmul_grad":
        return matmul_grad(size(1, 4096), size(16, 8192), size(16, 4096), rng.choice(["bf16", "f16", "f32"]), act)
    if op == "norm":
        rows, cols = size(1, 16384), size(8, 8192)
        dtype, scales = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["", "row", "block"])
        if scales == "block":
            cols = (cols + BLOCK - 1) // BLOCK * BLOCK
        if rows * cols > 1 << 26:
            rows = max(1, (1 << 26) // cols)
        return norm(rows, cols, dtype, rng.choice(["e4m3", "e4m3", "e5m2"]) if scales else dtype, scales, rng.random() < 0.6)
    if op == "norm_grad":
        rows, cols = size(1, 16384), size(8, 8192)
        if rows * cols > 1 << 26:
            rows = max(1, (1 << 26) // cols)
        return norm_grad(rows, cols, rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5)
    layers, width = size(1, 24), size(16, 1024)
    return clip(layers, width, size(16, 16384), rng.choice(["bf16", "f16", "f32"]) if width < 700 else "bf16", rng.choice([0.1, 1.0, 1e4]))


def shapes(case):
    """The parameters of `case`'s model: (shape, type) each; matrices in the case's type, norm weights in f32."""
    w, t = case["width"], case["dtype"]
    layer = [((w, w), t), ((w // 4 + 1, w), t), ((w // 4 + 1, w), t), ((w, w), t), ((4 * w, w), t), ((w, 4 * w), t), ((w,), "f32"), ((w,), "f32")]
    return [((case["vocab"], w), t)] + layer * case["layers"] + [((w,), "f32")]


def size_of(t):
    return {"f32": 4, "bf16": 2, "f16": 2}.get(t, 1)


def work(case):
    op = case["op"]
    if op in ("matmul", "matmul_grad"):
        m, n, k, s = case["m"], case["n"], case["k"], size_of(case["dtype"])
        if op == "matmul":
            c = size_of(case["out"])
            return {"bytes": (m * k + k * n) * s + m * n * c * (1 + case["residual"] + case["pre"]) + (n * c if case["bias"] else 0) + (4 * (m + n) if s == 1 else 0),
                    "flops": 2 * m * n * k}
        return {"bytes": (3 * m * n + 2 * m * k + 2 * k * n) * s + 4 * n, "flops": 4 * m * n * k}
    if op == "norm":
        e, s = case["rows"] * case["cols"], size_of(case["dtype"])
        scale = {"": 0, "row": 4 * case["rows"], "block": e // BLOCK}[case["scales"]]
        return {"bytes": e * (s * (1 + 2 * case["residual"]) + size_of(case["out"])) + s * case["cols"] + 4 * case["rows"] + scale, "flops": 4 * e}
    if op == "norm_grad":
        e, s = case["rows"] * case["cols"], size_of(case["dtype"])
        return {"bytes": e * s * (3 + case["stream"]) + case["cols"] * (s + 4) + 4 * case["rows"], "flops": 10 * e}
    elements = [(math.prod(shape), size_of(t)) for shape, t in shapes(case)]
    return {"bytes": sum(2 * n * s for n, s in elements), "flops": sum(3 * n for n, _ in elements)}


# ---- what a program has in hand --------------------------------------------------------------------------------------------------
class _Span:
    """Device memory at an address, in the form torch takes views of."""

    def __init__(self, ptr, nbytes):
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (ptr, False), "version": 3}


def _view(handle, shape, dtype):
    n = math.prod(shape) * TYPES[dtype].itemsize
    if n == 0:
        return torch.empty(shape, dtype=TYPES[dtype], device="cuda")
    return torch.as_tensor(_Span(handle.device_ptr(), n), device="cuda")[:n].view(TYPES[dtype]).view(shape)


def _elem(dtype):
    from cubecl_amd import ElemType
    return {"f32": ElemType.F32, "bf16": ElemType.BF16, "f16": ElemType.F16, "e4m3": ElemType.F8E4M3, "e5m2": ElemType.F8E5M2, "ue8m0": ElemType.UE8M0}[dtype]


def _name(t):
    return next(k for k, v in TYPES.items() if v == t.dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, t="f32", scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(TYPES[t])

    op, x, empty = case["op"], {}, {}
    if op == "matmul":
        m, n, k, t, o = case["m"], case["n"], case["k"], case["dtype"], case["out"]
        lhs, rhs = rand(m, k), rand(*((n, k) if case["rhs"] == "nk" else (k, n)), scale=k ** -0.5)
        if t == "e4m3":                      # quantised beforehand: a scale for each row of both operands
            x["lhs_scale"], x["rhs_scale"] = lhs.abs().amax(1) / TOP[t], rhs.abs().amax(1) / TOP[t]
            lhs, rhs = lhs / x["lhs_scale"][:, None], rhs / x["rhs_scale"][:, None]
        x["lhs"], x["rhs"] = lhs.to(TYPES[t]), rhs.to(TYPES[t])
        if case["bias"]:
            x["bias"] = rand(n, t=o, scale=0.5)
        if case["residual"]:
            x["residual"] = rand(m, n, t=o)
        empty["out"] = ((m, n), o)
        if case["pre"]:
            empty["pre_activation"] = ((m, n), o)
    elif op == "matmul_grad":
        m, n, k, t = case["m"], case["n"], case["k"], case["dtype"]
        x["grad_out"], x["pre_activation"] = rand(m, n, t=t), rand(m, n, t=t, scale=1.5)
        x["lhs"], x["rhs"] = rand(m, k, t=t), rand(k, n, t=t, scale=k ** -0.5)
        empty.update(grad_pre=((m, n), t), grad_bias=((n,), "f32"), grad_lhs=((m, k), t), grad_rhs=((k, n), t))
    elif op == "norm":
        r, c, t = case["rows"], case["cols"], case["dtype"]
        x["input"], x["weight"] = rand(r, c, t=t), (1 + 0.2 * rand(c)).to(TYPES[t])
        if case["residual"]:
            x["residual"] = rand(r, c, t=t, scale=2.0)
            empty["residual_out"] = ((r, c), t)
        empty["output"] = ((r, c), case["out"])
        empty["rstd"] = ((r,), "f32")
        if case["scales"]:
            empty["scales"] = ((r,), "f32") if case["scales"] == "row" else ((r, c // BLOCK), "ue8m0")
    elif op == "norm_grad":
        r, c, t = case["rows"], case["cols"], case["dtype"]
        x["grad_output"], x["hidden"], x["weight"] = rand(r, c, t=t), rand(r, c, t=t, scale=2.0), (1 + 0.2 * rand(c)).to(TYPES[t])
        x["rstd"] = torch.rsqrt(x["hidden"].float().square().mean(1) + EPS)
        if case["stream"]:
            x["grad_hidden"] = rand(r, c, t=t)
        empty.update(grad_input=((r, c), t), grad_weight=((c,), "f32"))
    else:
        return _prepare_clip(case, rand)
    state = {"case": case, "x": x}
    if not own:
        return state
    from cubecl_amd import Mi355Runtime, TensorHandle
    client = Mi355Runtime.client()

    def place(shape, dtype):
        h = client.empty(math.prod(shape) * TYPES[dtype].itemsize)
        return TensorHandle.new_contiguous(shape, h, _elem(dtype)), _view(h, shape, dtype)

    torch.cuda.synchronize()
    placed = {k: place(tuple(v.shape), _name(v)) for k, v in x.items()}
    [placed[k][1].copy_(v) for k, v in x.items()]
    outs = {k: place(*v) for k, v in empty.items()}
    state.update(client=client, h={k: v[0] for k, v in {**placed, **outs}.items()}, out={k: v[1] for k, v in outs.items()}, x={})
    return state


def _prepare_clip(case, rand):
    """Gradients as slices of one flat buffer for each type, as training programs keep them, and buffers like them for the result."""
    what = shapes(case)
    kinds = sorted({t for _, t in what})
    ends = {t: 0 for t in kinds}
    slots = []

    def slot(shape, t):
        at = ends[t]
        ends[t] = at + (math.prod(shape) + 63) // 64 * 64
        slots.append((shape, t, at))

    [slot(shape, t) for shape, t in what]
    flat = {t: torch.zeros(ends[t], dtype=TYPES[t], device="cuda") for t in kinds}

    def cut(buffers):
        return [buffers[t][at:at + math.prod(shape)].view(shape) for shape, t, at in slots]

    [v.copy_(rand(*v.shape, t=_name(v), scale=0.02 / (1 + i % 5))) for i, v in enumerate(cut(flat))]
    state = {"case": case}
    if not own:
        out = {t: torch.zeros_like(flat[t]) for t in kinds}
        return dict(state, grads=cut(flat), cuts=cut(out), out=out)
    from cubecl_amd import ElemType, Mi355Runtime, TensorHandle, ops
    client = Mi355Runtime.client()
    torch.cuda.synchronize()
    h = {t: (client.empty(ends[t] * size_of(t)), client.empty(ends[t] * size_of(t))) for t in kinds}
    views = {t: [_view(b, (ends[t],), t) for b in h[t]] for t in kinds}
    [(views[t][0].copy_(flat[t]), views[t][1].zero_()) for t in kinds]
    handles = [[TensorHandle.new_contiguous(shape, h[t][side].offset_start_by(at * size_of(t)), _elem(t)) for shape, t, at in slots] for side in (0, 1)]
    total = client.empty(4)
    return dict(state, client=client, grads=ops.TensorList(handles[0]), cuts=ops.TensorList(handles[1]), out={t: views[t][1] for t in kinds},
                total=TensorHandle.new_contiguous((1,), total, ElemType.F32), total_view=_view(total, (1,), "f32"))


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"matmul": _plain_matmul, "matmul_grad": _plain_matmul_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad, "clip": _plain_clip}[op](case, state)
    from cubecl_amd import ops
    client = state["client"]
    if op == "clip":
        ops.clip_by_global_norm(client, state["grads"], case["max_norm"], outputs=state["cuts"], total_norm=state["total"])
        return {"total_norm": state["total_view"], "out": state["out"]}
    h = state["h"]
    if op == "matmul":
        rhs = h["rhs"].permute((1, 0)) if case["rhs"] == "nk" else h["rhs"]
        ops.matmul_fused(client, h["lhs"], rhs, h["out"], bias=h.get("bias"), activation=case["act"], residual=h.get("residual"),
                         lhs_scale=h.get("lhs_scale"), rhs_scale=h.get("rhs_scale"), pre_activation=h.get("pre_activation"))
    elif op == "matmul_grad":
        ops.matmul_fused_backward(client, h["grad_out"], h["pre_activation"], h["grad_pre"], activation=case["act"], grad_bias=h["grad_bias"],
                                  lhs=h["lhs"], rhs=h["rhs"], grad_lhs=h["grad_lhs"], grad_rhs=h["grad_rhs"])
    elif op == "norm":
        ops.rms_norm(client, h["input"], h["weight"], h["output"], eps=EPS, residual=h.get("residual"), residual_out=h.get("residual_out"),
                     scales=h.get("scales"), rstd=h["rstd"])
    else:
        ops.rms_norm_backward(client, h["grad_output"], h["hidden"], h["weight"], h["rstd"], h["grad_input"], grad_weight=h["grad_weight"],
                              grad_hidden=h.get("grad_hidden"))
    return state["out"]


# ---- plain forms, in 32 bits ---------------------------------------------------------------------------------------------------------
C0, C1 = math.sqrt(2 / math.pi), 0.044715      # tanh's form of gelu


def _act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(C0 * (z + C1 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        t = torch.tanh(C0 * (z + C1 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * C0 * (1 + 3 * C1 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_matmul(case, state):
    x, o = state["x"], TYPES[case["out"]]
    rhs = x["rhs"].float()
    z = x["lhs"].float() @ (rhs.t() if case["rhs"] == "nk" else rhs)
    if "lhs_scale" in x:
        z = z * x["lhs_scale"][:, None] * x["rhs_scale"]
    if case["bias"]:
        z = z + x["bias"].float()
    y = _act(case["act"], z)
    if case["residual"]:
        y = y + x["residual"].float()
    out = {"out": y.to(o)}
    if case["pre"]:
        out["pre_activation"] = z.to(o)
    return out


def _plain_matmul_grad(case, state):
    x, t = state["x"], TYPES[case["dtype"]]
    dz = x["grad_out"].float() * _act_grad(case["act"], x["pre_activation"].float())
    return {"grad_pre": dz.to(t), "grad_bias": dz.sum(0), "grad_lhs": (dz @ x["rhs"].float().t()).to(t), "grad_rhs": (x["lhs"].float().t() @ dz).to(t)}


def _power(amax, t):
    """The least power of two s with amax / s <= the type's largest value (2^0 for zeros)."""
    mant, e = torch.frexp(amax)
    e = (e - TOP_EXP[t] + (mant > 0.875)).clamp(-127, 127)
    return torch.where(amax > 0, torch.exp2(e.to(amax.dtype)), torch.ones_like(amax))


def _plain_norm(case, state):
    x, t = state["x"], TYPES[case["dtype"]]
    h, out = x["input"].float(), {}
    if case["residual"]:
        h = h + x["residual"].float()
        out["residual_out"] = h.to(t)
    rstd = torch.rsqrt((h * h).mean(1) + EPS)
    y = h * rstd[:, None] * x["weight"].float()
    out["rstd"] = rstd
    if not case["scales"]:
        return dict(out, output=y.to(t))
    o = case["out"]
    if case["scales"] == "row":
        amax = y.abs().amax(1)
        s = torch.where(amax > 0, amax / TOP[o], torch.ones_like(amax))
        q = y / s[:, None]
    else:
        y = y.view(y.shape[0], -1, BLOCK)
        s = _power(y.abs().amax(2), o)
        q = (y / s[:, :, None]).flatten(1)
        s = s.to(torch.float8_e8m0fnu)
    return dict(out, output=q.clamp(-TOP[o], TOP[o]).to(TYPES[o]), scales=s)


def _plain_norm_grad(case, state):
    x, t = state["x"], TYPES[case["dtype"]]
    dy, rstd = x["grad_output"].float(), x["rstd"][:, None]
    xhat = x["hidden"].float() * rstd
    wdy = dy * x["weight"].float()
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(1, keepdim=True))
    if case["stream"]:
        dx = dx + x["grad_hidden"].float()
    return {"grad_input": dx.to(t), "grad_weight": (dy * xhat).sum(0)}


def _plain_clip(case, state):
    total = torch.sqrt(sum(g.double().square().sum() for g in state["grads"]))
    coef = torch.clamp(case["max_norm"] / total, max=1.0).float()
    [out.copy_(g.float() * coef) for g, out in zip(state["grads"], state["cuts"])]
    return {"total_norm": total.float().view(1), "out": state["out"]}


# ---- 64 bits, from the definitions ---------------------------------------------------------------------------------------------------
def _f64(name, z):
    """(activation, its derivative) of z in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).double()
        return z * on, on
    if name == "gelu":
        cdf, pdf = 0.5 * torch.erfc(-z / math.sqrt(2.0)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf
    # silu and tanh's gelu are both z * sigmoid(u(z))
    u, du = (z, 1.0) if name == "silu" else (2 * C0 * z * (1 + C1 * z ** 2), 2 * C0 * (1 + 3 * C1 * z ** 2))
    s = torch.sigmoid(u)
    return z * s, s + z * s * (1 - s) * du


def exact(case, seed):
    global own
    side, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = side
    op = case["op"]
    if op == "clip":
        g = {t: torch.zeros_like(v, dtype=torch.float64) for t, v in state["out"].items()}
        whole = torch.cat([v.double().reshape(-1) for v in state["grads"]])
        total = torch.linalg.vector_norm(whole)
        coef = min(1.0, case["max_norm"] / float(total))
        [c.copy_(v) for v, c in zip(state["grads"], state["cuts"])]          # the same slots, scaled in 64 bits below
        return {"total_norm": total.view(1), "out": {t: g[t] + state["out"][t].double() * coef for t in g}}
    x = {k: v.double() for k, v in state["x"].items()}
    if op == "matmul":
        z = torch.matmul(x["lhs"], x["rhs"].t() if case["rhs"] == "nk" else x["rhs"])
        if case["dtype"] == "e4m3":
            z = torch.outer(x["lhs_scale"], x["rhs_scale"]) * z
        z = z + x.get("bias", 0.0)
        out = {"out": _f64(case["act"], z)[0] + x.get("residual", 0.0)}
        return dict(out, pre_activation=z) if case["pre"] else out
    if op == "matmul_grad":
        dz = x["grad_out"] * _f64(case["act"], x["pre_activation"])[1]
        return {"grad_pre": dz, "grad_bias": dz.sum(0), "grad_lhs": torch.matmul(dz, x["rhs"].t()), "grad_rhs": torch.matmul(x["lhs"].t(), dz)}
    if op == "norm":
        h = x["input"] + x.get("residual", 0.0)
        rstd = ((h ** 2).sum(1) / case["cols"] + EPS) ** -0.5
        y = x["weight"] * (h * rstd.view(-1, 1))
        out = {"rstd": rstd, "residual_out": h} if case["residual"] else {"rstd": rstd}
        if not case["scales"]:
            return dict(out, output=y)
        o = case["out"]
        parts = y.view(case["rows"], -1, case["cols"] if case["scales"] == "row" else BLOCK)
        top = parts.abs().amax(2)
        s = top / TOP[o] if case["scales"] == "row" else torch.exp2(torch.ceil(torch.log2(top / TOP[o])))
        # the quotient before its rounding to 8 bits; three bits of e5m2 tell nothing about the computation's exactness
        q = (parts / s.unsqueeze(2)).reshape(case["rows"], case["cols"]) if o == "e4m3" else None
        return dict(out, output=q, scales=s.view(-1) if case["scales"] == "row" else s)
    rstd, xhat = x["rstd"].view(-1, 1), x["hidden"] * x["rstd"].view(-1, 1)
    wdy = x["grad_output"] * x["weight"]
    mean = (wdy * xhat).sum(1, keepdim=True) / case["cols"]
    return {"grad_input": (wdy - mean * xhat) * rstd + x.get("grad_hidden", 0.0), "grad_weight": (x["grad_output"] * xhat).sum(0)}
