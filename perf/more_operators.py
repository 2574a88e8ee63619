"""Cases of the operators around a linear layer in 8-bit integers: the RMS norm in
front of it with the residual's addition and its gradients, rows in 8 bits with a
scale each (of a norm, or of any matrix), and the product of two such matrices.

``listed()`` and ``draw(rng)`` give cases, ``prepare`` a case's inputs on the GPU,
``run`` one pass (plain torch operations, or the package's operators where
``own`` is true), ``work`` the bytes and operations that a pass cannot do without,
``exact`` the outputs in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decoding step of 16 sequences through a block's norm, the block before it added: latency
        {"name": "norm_step", "op": "norm", "type": "bf16", "rows": 16, "columns": 3840, "weight": True, "residual": True, "grad": False},
        # an image's and its caption's tokens through a block's norm
        {"name": "norm_block", "op": "norm", "type": "bf16", "rows": 4352, "columns": 3840, "weight": True, "residual": True, "grad": False},
        # training through the norm and the residual, ragged length
        {"name": "norm_train", "op": "norm", "type": "bf16", "rows": 4099, "columns": 4096, "weight": True, "residual": True, "grad": True},
        # training a small encoder in float32, without a residual
        {"name": "norm_train_f32", "op": "norm", "type": "f32", "rows": 1234, "columns": 768, "weight": True, "residual": False, "grad": True},
        # one decoding step of 4 sequences, rows in 8 bits for the linear layer behind the norm: latency
        {"name": "rows_step", "op": "rows", "type": "bf16", "rows": 4, "columns": 3840, "norm": True, "weight": True, "residual": True},
        # the tokens of an image, in 8 bits for the linear layers behind the norm
        {"name": "rows_block", "op": "rows", "type": "bf16", "rows": 4352, "columns": 3840, "norm": True, "weight": True, "residual": True},
        # a layer's weight, once when a model is loaded
        {"name": "rows_weight", "op": "rows", "type": "bf16", "rows": 10240, "columns": 3840, "norm": False, "weight": False,
         "residual": False},
        # a single token through a feed-forward's first product: bound by the weight's bytes
        {"name": "matmul_token", "op": "matmul", "type": "bf16", "rows": 1, "inner": 3840, "columns": 10240, "bias": False},
        # single tokens of 24 sequences through its second product
        {"name": "matmul_tokens", "op": "matmul", "type": "bf16", "rows": 24, "inner": 10240, "columns": 3840, "bias": False},
        # a prompt through a stacked q/k/v product, ragged length
        {"name": "matmul_prompt", "op": "matmul", "type": "f16", "rows": 333, "inner": 3840, "columns": 11520, "bias": True},
        # an image's tokens through a block's gate and up projections, stacked
        {"name": "matmul_block", "op": "matmul", "type": "bf16", "rows": 4352, "inner": 3840, "columns": 20480, "bias": False},
        # a long prompt, or a batch of them
        {"name": "matmul_long", "op": "matmul", "type": "bf16", "rows": 16384, "inner": 12288, "columns": 4096, "bias": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A row's length: mostly whole 16s, as models have it, sometimes anything."""
    n = _log(rng, low, high)
    return n if rng.random() < 0.2 else max(16, (n + 8) // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "norm", "rows", "rows", "matmul", "matmul", "matmul"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "matmul":
        inner, columns = _size(rng, 64, 16384), _size(rng, 64, 24576)
        return {"op": op, "type": kind, "rows": _log(rng, 1, max(2, min(16384, 400_000_000_000 // (inner * columns)))), "inner": inner,
                "columns": columns, "bias": rng.random() < 0.5}
    columns = _size(rng, 64, 16384)
    case = {"op": op, "type": kind, "rows": _log(rng, 1, max(2, min(16384, 30_000_000 // columns))), "columns": columns,
            "weight": rng.random() < 0.8, "residual": rng.random() < 0.6}
    if op == "norm":
        case["grad"] = rng.random() < 0.5
    else:
        case["norm"] = rng.random() < 0.6
        if not case["norm"]:
            case["weight"] = case["residual"] = False
    return case


def work(case):
    size, rows, columns = _BYTES[case["type"]], case["rows"], case["columns"]
    if case["op"] == "matmul":
        inner = case["inner"]
        return {"bytes": (rows + columns) * (inner + 4) + size * columns * (rows + (1 if case["bias"] else 0)),
                "flops": 2 * rows * columns * inner}
    values, weight = rows * columns, columns * size if case["weight"] else 0
    if case["op"] == "rows":  # the result as it is held: a byte for a value and a scale for a row
        moved = size * values * (1 + (2 if case["residual"] else 0)) + values + 4 * rows + weight
        return {"bytes": moved, "flops": values * (8 if case["norm"] else 4)}
    moved = size * values * (2 + (2 if case["residual"] else 0)) + weight
    if case["grad"]:  # the gradients of the results read, that of what is normalised written
        moved += size * values * (2 + (1 if case["residual"] else 0)) + weight
    return {"bytes": moved, "flops": values * (5 + (12 if case["grad"] else 0))}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    dtype, rows, columns = _TYPES[case["type"]], case["rows"], case["columns"]
    state = {"case": case}
    if case["op"] == "matmul":
        inner = case["inner"]

        def codes(n):  # rows of a normal distribution, the largest at 127
            x = normal(n, inner)
            return torch.round(x * (127.0 / x.abs().amax(dim=1, keepdim=True))).to(torch.int8)

        state.update(x=codes(rows), w=codes(columns), x_scales=torch.rand(rows, generator=g, device="cuda") * 0.03 + 0.01,
                     w_scales=torch.rand(columns, generator=g, device="cuda") * 0.0005 + 0.0002,
                     bias=normal(columns, std=0.1, dtype=dtype) if case["bias"] else None, dtype=dtype)
        return state
    # a few channels much larger than the others, as in the residual stream of a deep model
    if case["op"] == "rows" and not case["norm"]:
        state["x"] = normal(rows, columns, std=0.02, dtype=dtype)
        return state
    channels = torch.exp(normal(columns, std=0.7))
    state["x"] = (normal(rows, columns, std=0.6) * channels).to(dtype)
    state["residual"] = (normal(rows, columns, std=1.2) * channels).to(dtype) if case["residual"] else None
    state["weight"] = normal(columns, std=0.2).add(1.0).to(dtype) if case["weight"] else None
    if case["op"] == "norm" and case["grad"]:
        state["dy"] = normal(rows, columns, dtype=dtype)
        state["dsum"] = normal(rows, columns, dtype=dtype) if case["residual"] else None
        state["leaves"] = [state[n].requires_grad_() for n in ("x", "residual", "weight") if state[n] is not None]
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if not own:
        return _plain_matmul(state) if case["op"] == "matmul" else _plain_rows(state) if case["op"] == "rows" else _plain_norm(state)
    import mflux_amd

    if case["op"] == "matmul":
        return mflux_amd.int8_matmul(state["x"], state["x_scales"], state["w"], state["w_scales"], bias=state["bias"], dtype=state["dtype"])
    if case["op"] == "rows":
        if not case["norm"]:
            return mflux_amd.int8_dequantize(*mflux_amd.int8_quantize(state["x"]), dtype=state["x"].dtype)
        codes, scales, *rest = mflux_amd.rms_norm_int8(state["x"], state["weight"], residual=state["residual"])
        return [mflux_amd.int8_dequantize(codes, scales, dtype=state["x"].dtype)] + rest
    outputs = mflux_amd.rms_norm(state["x"], state["weight"], residual=state["residual"])
    if not case["grad"]:
        return outputs
    outputs = outputs if case["residual"] else (outputs,)
    gradients = (state["dy"], state["dsum"])[:len(outputs)]
    return [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, state["leaves"], gradients))


# ---- the plain forms -------------------------------------------------------------------------------------------------------------

_EPS = 1e-6


def _plain_sum(state):
    """What is normalised: the sum with the residual as it is stored."""
    x, residual = state["x"].detach(), state["residual"]
    return x if residual is None else (x.float() + residual.detach().float()).to(x.dtype)


def _plain_norm(state):
    case, s = state["case"], _plain_sum(state)
    h, weight = s.float(), state["weight"]
    rstd = torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + _EPS)
    n = h * rstd
    y = (n if weight is None else n * weight.detach().float()).to(s.dtype)
    outputs = [y, s] if case["residual"] else [y]
    if not case["grad"]:
        return outputs if case["residual"] else y
    dy = state["dy"].float()
    dn = dy if weight is None else dy * weight.detach().float()
    dx = rstd * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
    if case["residual"]:
        dx = dx + state["dsum"].float()
    dx = dx.to(s.dtype)
    outputs += [dx, dx] if case["residual"] else [dx]
    if weight is not None:
        outputs.append((dy * n).sum(dim=0).to(s.dtype))
    return outputs


def _plain_rows(state):
    case = state["case"]
    if not case["norm"]:
        s, factor = state["x"], 1.0
        p = s.double()
    else:
        s, weight = _plain_sum(state), state["weight"]
        h = s.float()
        factor = torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + _EPS)
        # in 64 bits: a code is decided by values next to a border
        p = s.double() if weight is None else s.double() * weight.double()
    top = p.abs().amax(dim=-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(p * 127 / top), 0.0)
    y = (codes.float() * (top.float() * factor / 127)).to(s.dtype)
    if not case["norm"]:
        return y
    return [y, s] if case["residual"] else [y]


def _plain_matmul(state):
    y = state["x"].float() @ state["w"].float().t()
    y = y * state["x_scales"][:, None] * state["w_scales"]
    return (y if state["bias"] is None else y + state["bias"].float()).to(state["dtype"])


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "matmul":
        y = torch.mm(state["x"].double(), state["w"].double().t().contiguous())
        y *= torch.outer(state["x_scales"].double(), state["w_scales"].double())
        return y if state["bias"] is None else y + state["bias"].double()
    s = state["x"].detach().double()
    residual, weight = state.get("residual"), state.get("weight")
    if residual is not None:  # the norm is of the sum as it is stored
        s = (s + residual.detach().double()).to(state["x"].dtype).double()
    gain = torch.ones(case["columns"], device="cuda", dtype=torch.float64) if weight is None else weight.detach().double()
    if case["op"] == "rows":
        size = 1.0
        if case["norm"]:
            size = (s.square().sum(dim=1, keepdim=True) / case["columns"] + _EPS).sqrt()
        largest = (s * gain).abs().max(dim=1, keepdim=True).values
        steps = (s * gain * 127 / largest.clamp(min=1e-300)).round()
        y = steps * (largest / size) / 127
        return y if not case["norm"] else [y] if residual is None else [y, s]
    size = (s.square().sum(dim=1, keepdim=True) / case["columns"] + _EPS).sqrt()
    outputs = [s / size * gain] + ([] if residual is None else [s])
    if not case["grad"]:
        return outputs if residual is not None else outputs[0]
    up = state["dy"].double()
    inner = (up * gain * s).sum(dim=1, keepdim=True)
    down = up * gain / size - s * inner / (case["columns"] * size ** 3)
    if residual is not None:
        down = down + state["dsum"].double()
    outputs += [down] if residual is None else [down, down]
    if weight is not None:
        outputs.append((up * s / size).sum(dim=0))
    return outputs
