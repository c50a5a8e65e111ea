"""The operators of a trained linear layer, as cases that can be timed and checked.

  fwd   Y = act(X W^T + b) [+ R], with the activation's argument Z kept for training
  bwd   the gradients of that product: dZ = dY * act'(Z), dX = dZ W, dW = dZ^T X, db = sum dZ
  dact  the step between two layers: dZ = (dY W) * act'(Z) and its column sums, in one product
  orth  Newton-Schulz iterations that orthogonalise a weight's update

Each in plain torch operations in 32 bits (`own` false) and through rtatblas_amd (`own` true).
Tensors are row-major as torch has them; to the column-major library a row-major (r x c) tensor
is the c x r matrix with leading dimension its row stride, which is how the calls below name
their operands.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
# The quintic of the Newton-Schulz step: singular values in (0, 1] end near 1 after five steps.
QUINTIC = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # One new token through an up-projection: the whole weight is read for one column.
        {"name": "fwd one token", "op": "fwd", "tokens": 1, "inp": 2048, "out": 8192, "dtype": "bf16", "act": "silu", "wt": "nk", "residual": False, "aux": False, "pad": 0},
        # A few sequences decoded together through a down-projection with the residual's addition.
        {"name": "fwd 13 tokens", "op": "fwd", "tokens": 13, "inp": 8192, "out": 2048, "dtype": "f16", "act": "none", "wt": "nk", "residual": True, "aux": False, "pad": 0},
        # A prompt of odd length in a model of odd width, rows padded to an odd stride, weight stored in x out.
        {"name": "fwd ragged", "op": "fwd", "tokens": 1531, "inp": 1001, "out": 2051, "dtype": "bf16", "act": "gelu", "wt": "kn", "residual": True, "aux": False, "pad": 3},
        # A training batch through an up-projection, the activation's argument kept.
        {"name": "fwd training batch", "op": "fwd", "tokens": 8192, "inp": 4096, "out": 8192, "dtype": "bf16", "act": "gelu_tanh", "wt": "nk", "residual": False, "aux": True, "pad": 0},
        # A small layer's backward pass.
        {"name": "bwd small", "op": "bwd", "tokens": 256, "inp": 1024, "out": 1024, "dtype": "f16", "act": "relu", "wt": "nk", "grads": "f16", "pad": 0},
        # Odd sizes; no activation and the weight's gradient in 32 bits, as an optimiser keeps it.
        {"name": "bwd ragged", "op": "bwd", "tokens": 4099, "inp": 1001, "out": 1531, "dtype": "bf16", "act": "none", "wt": "nk", "grads": "f32", "pad": 1},
        # The backward pass of the training batch.
        {"name": "bwd training batch", "op": "bwd", "tokens": 8192, "inp": 4096, "out": 8192, "dtype": "bf16", "act": "gelu_tanh", "wt": "nk", "grads": "bf16", "pad": 0},
        # Between a block's two products, odd sizes, and a training batch.
        {"name": "dact ragged", "op": "dact", "tokens": 777, "inp": 2050, "out": 511, "dtype": "f16", "act": "gelu", "pad": 0},
        {"name": "dact training batch", "op": "dact", "tokens": 4096, "inp": 8192, "out": 2048, "dtype": "bf16", "act": "silu", "pad": 0},
        # A small square weight's update; several ragged ones of one shape; a large projection's.
        {"name": "orth small", "op": "orth", "rows": 128, "cols": 128, "batch": 1, "dtype": "bf16", "steps": 5, "pad": 0},
        {"name": "orth ragged batch", "op": "orth", "rows": 1000, "cols": 333, "batch": 6, "dtype": "f32", "steps": 5, "pad": 3},
        {"name": "orth large", "op": "orth", "rows": 8192, "cols": 2048, "batch": 1, "dtype": "bf16", "steps": 5, "pad": 0},
    ]


def _size(rng, lo, hi):
    """Spread over the logarithm; every other one is rounded to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v if rng.random() < 0.5 else (v + 7) // 8 * 8))


def draw(rng):
    op = rng.choice(("fwd", "bwd", "dact", "orth"))
    if op == "orth":
        rows, cols = _size(rng, 32, 8192), _size(rng, 32, 2048)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        batch = rng.randint(1, 6) if rows * cols <= 1 << 20 else 1
        return {"op": op, "rows": rows, "cols": cols, "batch": batch, "dtype": rng.choice(("bf16", "f16", "f32")), "steps": rng.randint(3, 5), "pad": rng.choice((0, 0, 1, 8))}
    case = {"op": op, "tokens": _size(rng, 1, 8192), "inp": _size(rng, 64, 4096), "out": _size(rng, 64, 8192), "dtype": rng.choice(("bf16", "f16")), "act": rng.choice(ACTS), "pad": rng.choice((0, 0, 1, 8))}
    if op == "fwd":
        case |= {"wt": rng.choice(("nk", "nk", "kn")), "residual": rng.random() < 0.5, "aux": rng.random() < 0.3}
    elif op == "bwd":
        case |= {"wt": rng.choice(("nk", "nk", "kn")), "grads": "f32" if case["act"] == "none" else case["dtype"]}
    return case


def _rows(gen, shape, dtype, pad, scale=1.0):
    """Normal values in a tensor whose rows are `pad` elements further apart than they are long."""
    full = torch.randn(*shape[:-1], shape[-1] + pad, generator=gen, device="cuda") * scale
    return full.to(dtype)[..., : shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, pad = TYPES[case["dtype"]], case["pad"]
    s = {"case": dict(case)}
    if case["op"] == "orth":
        b, r, c = case["batch"], case["rows"], case["cols"]
        # An update's shape: a few strong directions over a floor of noise.
        u = torch.randn(b, r, 16, generator=gen, device="cuda")
        v = torch.randn(b, 16, c, generator=gen, device="cuda")
        g = torch.bmm(u, v).mul_(0.25) + torch.randn(b, r, c, generator=gen, device="cuda").mul_(0.3)
        s["G"] = torch.zeros(b, r, c + pad, device="cuda", dtype=dt)[..., :c]
        s["G"].copy_(g.mul_(1e-3))
        return s
    t, k, n = case["tokens"], case["inp"], case["out"]
    if case["op"] == "dact":
        s["dY"] = _rows(gen, (t, n), dt, pad)
        s["W"] = _rows(gen, (n, k), dt, 0, n ** -0.5)
        s["Z"] = _rows(gen, (t, k), dt, pad)
        return s
    s["X"] = _rows(gen, (t, k), dt, pad)
    s["W"] = _rows(gen, (n, k) if case["wt"] == "nk" else (k, n), dt, 0, k ** -0.5)
    s["b"] = _rows(gen, (n,), dt, 0, 0.5)
    if case["op"] == "fwd":
        s["R"] = _rows(gen, (t, n), dt, pad) if case["residual"] else None
    else:
        s["dY"] = _rows(gen, (t, n), dt, pad)
        s["Z"] = _rows(gen, (t, n), dt, pad) if case["act"] != "none" else None
    return s


# ---- plain forms -------------------------------------------------------------------------


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_fwd(s, case, dt):
    w = s["W"].float()
    z = s["X"].float() @ (w.t() if case["wt"] == "nk" else w) + s["b"].float()
    y = _act(z, case["act"])
    if s["R"] is not None:
        y = y + s["R"].float()
    return {"Y": y.to(dt), "Z": z.to(dt) if case["aux"] else None}


def _plain_bwd(s, case, dt):
    x, w, dz = s["X"].float(), s["W"].float(), s["dY"].float()
    if case["act"] != "none":
        dz = dz * _act_slope(s["Z"].float(), case["act"])
    dx = dz @ (w if case["wt"] == "nk" else w.t())
    dw = dz.t() @ x if case["wt"] == "nk" else x.t() @ dz
    return {"dX": dx.to(dt), "dW": dw.to(TYPES[case["grads"]]), "db": dz.sum(0)}


def _plain_dact(s, case, dt):
    dz = (s["dY"].float() @ s["W"].float()) * _act_slope(s["Z"].float(), case["act"])
    return {"dZ": dz.to(dt), "db": dz.sum(0)}


def _plain_orth(s, case):
    g = s["G"]
    x = (g.double() / (g.double().square().sum((1, 2), keepdim=True).sqrt() + 1e-7)).float()
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2).contiguous()
    a, b, c = QUINTIC
    for _ in range(case["steps"]):
        m = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * m + c * torch.bmm(m, m), x)
    return {"O": (x.transpose(1, 2).contiguous() if tall else x).to(torch.bfloat16)}


# ---- the same through the library --------------------------------------------------------

_lib = {}
_handles = {}


def _handle():
    """The program's handle on torch's current stream.  A handle works on one stream, its scratch with it, so every stream has
    one of its own; a stream that is to be captured runs a pass first, which creates it."""
    if not _lib:
        from rtatblas_amd import native
        _lib["native"] = native
        _lib["type"] = {torch.bfloat16: native.TYPE_BF16, torch.float16: native.TYPE_F16, torch.float32: native.TYPE_F32}
        _lib["act"] = {a: getattr(native, "ACT_" + a.upper()) for a in ACTS}
    # Not torch.cuda.current_stream(), which takes 2.6 us to build an object around this number (0.3).
    device = torch.cuda.current_device()
    on = (device, torch._C._cuda_getCurrentRawStream(device))
    if on not in _handles:
        _handles[on] = _lib["native"].Handle(on[1])
    return _lib["native"], _handles[on]


def _own_fwd(s, case, dt):
    nat, h = _handle()
    x, w, r = s["X"], s["W"], s["R"]
    t, k, n = case["tokens"], case["inp"], case["out"]
    y = torch.empty(t, n, dtype=dt, device="cuda")
    z = torch.empty(t, n, dtype=dt, device="cuda") if case["aux"] else None
    h.gemm_ep(_lib["type"][dt], nat.OP_T if case["wt"] == "nk" else nat.OP_N, nat.OP_N, n, t, k, 1.0, w, w.stride(0), x, x.stride(0), y, n, act=_lib["act"][case["act"]], bias=s["b"],
              aux=z, ldaux=n, beta=0.0 if r is None else 1.0, C=r, ldc=0 if r is None else r.stride(0))
    return {"Y": y, "Z": z}


def _own_bwd(s, case, dt):
    nat, h = _handle()
    x, w, dy, z = s["X"], s["W"], s["dY"], s["Z"]
    t, k, n = case["tokens"], case["inp"], case["out"]
    grads = TYPES[case["grads"]]
    dx = torch.empty(t, k, dtype=dt, device="cuda")
    dw = torch.empty(w.shape, dtype=grads, device="cuda")
    db = torch.empty(n, dtype=torch.float32, device="cuda")
    dz = torch.empty(t, n, dtype=dt, device="cuda") if z is not None else None
    h.gemm_ep_backward(_lib["type"][dt], nat.OP_T if case["wt"] == "nk" else nat.OP_N, nat.OP_N, n, t, k, 1.0, w, w.stride(0), x, x.stride(0), dy, dy.stride(0), act=_lib["act"][case["act"]],
                       aux=z, ldaux=0 if z is None else z.stride(0), dZ=dz, lddz=n, dA=dw, ldda=dw.stride(0), da_type=_lib["type"][grads], dB=dx, lddb=k, dbias=db)
    return {"dX": dx, "dW": dw, "db": db}


def _own_dact(s, case, dt):
    nat, h = _handle()
    dy, w, z = s["dY"], s["W"], s["Z"]
    t, k, n = case["tokens"], case["inp"], case["out"]
    dz = torch.empty(t, k, dtype=dt, device="cuda")
    db = torch.empty(k, dtype=torch.float32, device="cuda")
    h.gemm_dact(_lib["type"][dt], nat.OP_N, nat.OP_N, k, t, n, 1.0, w, w.stride(0), dy, dy.stride(0), _lib["act"][case["act"]], z, z.stride(0), dz, k, dbias=db)
    return {"dZ": dz, "db": db}


def _own_orth(s, case, dt):
    nat, h = _handle()
    g = s["G"]
    b, r, c = g.shape
    o = torch.empty(b, r, c, dtype=torch.bfloat16, device="cuda")
    h.newton_schulz(_lib["type"][dt], c, r, g, g.stride(1), o, c, [QUINTIC] * case["steps"], eps=1e-7, batch=b, strideg=g.stride(0), strideo=o.stride(0))
    return {"O": o}


def run(state):
    case = state["case"]
    dt, op = TYPES[case["dtype"]], case["op"]
    if own:
        if op == "fwd":
            return _own_fwd(state, case, dt)
        if op == "bwd":
            return _own_bwd(state, case, dt)
        return _own_dact(state, case, dt) if op == "dact" else _own_orth(state, case, dt)
    if op == "fwd":
        return _plain_fwd(state, case, dt)
    if op == "bwd":
        return _plain_bwd(state, case, dt)
    return _plain_dact(state, case, dt) if op == "dact" else _plain_orth(state, case)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "orth":
        lo, hi = sorted((case["rows"], case["cols"]))
        # Per step: the symmetric Gram product, its symmetric square, and the product with X.
        flops = case["steps"] * (lo * (lo + 1) * hi + lo * (lo + 1) * lo + 2 * lo * lo * hi)
        return {"bytes": case["batch"] * lo * hi * (size + 2), "flops": case["batch"] * flops}
    t, k, n = case["tokens"], case["inp"], case["out"]
    if case["op"] == "fwd":
        outs = 1 + int(case["residual"]) + int(case["aux"])
        return {"bytes": 2 * (t * k + k * n + n + outs * t * n), "flops": 2 * t * k * n}
    if case["op"] == "bwd":
        ins = 1 + int(case["act"] != "none")
        return {"bytes": 2 * (2 * t * k + k * n + ins * t * n) + k * n * (4 if case["grads"] == "f32" else 2) + 4 * n, "flops": 4 * t * k * n}
    return {"bytes": 2 * (t * n + n * k + 2 * t * k) + 4 * k, "flops": 2 * t * k * n}


# ---- the definition in 64 bits -----------------------------------------------------------


def _act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "orth":
        g = s["G"].double()
        a, b, c = QUINTIC
        outs = []
        for x in g:
            x = x / (torch.linalg.matrix_norm(x) + 1e-7)
            for _ in range(case["steps"]):
                if case["rows"] > case["cols"]:
                    p = x.t() @ x
                    x = a * x + b * (x @ p) + c * ((x @ p) @ p)
                else:
                    p = x @ x.t()
                    x = a * x + b * (p @ x) + c * (p @ (p @ x))
            outs.append(x)
        return {"O": torch.stack(outs)}
    w = s["W"].double()
    if op == "dact":
        z = s["Z"].double().requires_grad_(True)
        dz, = torch.autograd.grad(_act64(z, case["act"]), z, s["dY"].double() @ w)
        return {"dZ": dz, "db": dz.sum(0)}
    x = s["X"].double()
    if case["wt"] == "nk":
        w = w.t()
    if op == "fwd":
        z = torch.addmm(s["b"].double(), x, w)
        y = _act64(z, case["act"])
        return {"Y": y if s["R"] is None else y + s["R"].double(), "Z": z if case["aux"] else None}
    dz = s["dY"].double()
    if s["Z"] is not None:
        z = s["Z"].double().requires_grad_(True)
        dz, = torch.autograd.grad(_act64(z, case["act"]), z, dz)
    dw = torch.mm(x.t(), dz)
    return {"dX": torch.mm(dz, w.t()), "dW": dw.t().contiguous() if case["wt"] == "nk" else dw, "db": dz.sum(0)}
