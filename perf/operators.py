"""Cases of the operators between an attention block's q/k/v product and its
output projection: rotary tables, RMS norm of the heads with rotary positions,
and attention, each with its gradients where it has any.

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
        # the position table of one image's tokens and its text: three axes of ids side by side in a head of 128
        {"name": "tables_axes", "op": "tables", "positions": 4608, "dims": "16,56,56", "base": 10000.0, "scaling": "none", "factor": 1.0},
        # a text model's whole table, stretched for a long context
        {"name": "tables_long", "op": "tables", "positions": 131072, "dims": "128", "base": 1000000.0, "scaling": "yarn", "factor": 4.0},
        # one decoding step of 16 sequences: latency
        {"name": "rotary_step", "op": "rotary", "type": "bf16", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotated": 128, "layout": "half", "norm": False, "gather": True, "grad": False, "packed": False},
        # a diffusion block: q and k of the stacked product, normalised and rotated
        {"name": "rotary_block", "op": "rotary", "type": "bf16", "batch": 1, "tokens": 4608, "heads": 24, "kv_heads": 24, "dim": 128,
         "rotated": 128, "layout": "interleaved", "norm": True, "gather": False, "grad": False, "packed": True},
        # training through the norm and a rotation of half the head, ragged length
        {"name": "rotary_train", "op": "rotary", "type": "f16", "batch": 2, "tokens": 2055, "heads": 16, "kv_heads": 4, "dim": 128,
         "rotated": 64, "layout": "half", "norm": True, "gather": False, "grad": True, "packed": False},
        # a diffusion block's attention over image and text tokens
        {"name": "attention_block", "op": "attention", "form": "batched", "type": "bf16", "batch": 1, "queries": 4608, "keys": 4608,
         "heads": 24, "kv_heads": 24, "dim": 128, "causal": False, "ragged": False, "grad": False, "spread": 0},
        # a text encoder on a batch of padded prompts: small heads, latency
        {"name": "attention_encoder", "op": "attention", "form": "batched", "type": "f16", "batch": 8, "queries": 77, "keys": 77,
         "heads": 12, "kv_heads": 12, "dim": 64, "causal": True, "ragged": True, "grad": False, "spread": 1},
        # prompts of very different lengths packed behind each other, grouped heads
        {"name": "attention_packed", "op": "attention", "form": "packed", "type": "bf16", "batch": 11, "queries": 9001, "keys": 9001,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "ragged": True, "grad": False, "spread": 2},
        # one long prompt
        {"name": "attention_long", "op": "attention", "form": "batched", "type": "bf16", "batch": 1, "queries": 16384, "keys": 16384,
         "heads": 28, "kv_heads": 4, "dim": 128, "causal": True, "ragged": False, "grad": False, "spread": 0},
        # a training step on packed sequences
        {"name": "attention_train", "op": "attention", "form": "packed", "type": "bf16", "batch": 3, "queries": 4099, "keys": 4099,
         "heads": 24, "kv_heads": 8, "dim": 128, "causal": True, "ragged": True, "grad": True, "spread": 3},
        # single tokens of 32 sequences over caches of different lengths
        {"name": "attention_decode", "op": "attention", "form": "batched", "type": "bf16", "batch": 32, "queries": 1, "keys": 8192,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "ragged": True, "grad": False, "spread": 4},
        # one token over a long cache: few rows, a long axis
        {"name": "attention_decode_long", "op": "attention", "form": "batched", "type": "bf16", "batch": 1, "queries": 1, "keys": 100003,
         "heads": 28, "kv_heads": 4, "dim": 128, "causal": True, "ragged": False, "grad": False, "spread": 0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "rotary", "attention", "attention", "attention", "attention"])
    if op == "tables":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": op, "positions": _log(rng, 64, 131072), "dims": rng.choice(["64", "128", "16,56,56", "32,48,48"]),
                "base": rng.choice([10000.0, 256.0, 1000000.0]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0])}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7])
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "rotary":
        dim = rng.choice([64, 72, 128, 128, 256])
        batch = _log(rng, 1, 8)
        grad = rng.random() < 0.4
        return {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "batch": batch, "tokens": _log(rng, 1, 16384 // batch),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2]),
                "layout": rng.choice(["interleaved", "half"]), "norm": rng.random() < 0.5, "gather": rng.random() < 0.3, "grad": grad,
                "packed": rng.random() < 0.3}
    form = rng.choice(["batched", "packed"])
    dim = rng.choice([64, 80, 128, 128])
    if rng.random() < 0.3:  # single tokens, or a few
        batch = _log(rng, 1, 64)
        return {"op": op, "form": form, "type": kind, "batch": batch, "queries": batch if form == "packed" else rng.choice([1, 1, 1, 4]),
                "keys": (_log(rng, 64, 8192) if form == "batched" else _log(rng, 64 * batch, 8192 * batch)), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "causal": True, "ragged": True, "grad": False, "spread": rng.randrange(1000)}
    batch = _log(rng, 1, 8)
    total = _log(rng, 64, 8192)
    tokens = total if form == "packed" else max(1, total // batch)
    return {"op": op, "form": form, "type": kind, "batch": batch, "queries": tokens, "keys": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "causal": rng.random() < 0.6, "ragged": rng.random() < 0.7, "grad": rng.random() < 0.4 and total <= 4096,
            "spread": rng.randrange(1000)}


# ---- lengths -----------------------------------------------------------------------------------------------------------------

def _split(total, parts, spread):
    """`parts` lengths of unequal size whose sum is `total`."""
    weights = [math.exp(1.5 * math.sin(1.0 + 12.9898 * (i + 1) * (spread + 1))) for i in range(parts)]
    scale = total / sum(weights)
    lengths = [int(w * scale) for w in weights]
    lengths[0] += total - sum(lengths)
    return lengths


def _lengths(case):
    """(queries, keys) of every sequence of an attention case."""
    batch, queries, keys = case["batch"], case["queries"], case["keys"]
    if case["form"] == "packed":
        if not case["ragged"]:
            q = [queries // batch + (i < queries % batch) for i in range(batch)]
            return q, q if keys == queries else [keys // batch + (i < keys % batch) for i in range(batch)]
        k = _split(keys, batch, case["spread"])
        return (k if queries == keys else [1] * batch), k
    if not case["ragged"]:
        return [queries] * batch, [keys] * batch
    low = max(1, min(keys, keys // 8))
    k = [low + int((keys - low) * (0.5 + 0.5 * math.sin(2.0 + 78.233 * (i + 1) * (case["spread"] + 1)))) for i in range(batch)]
    return (k if queries == keys else [queries] * batch), k


def _pairs(nq, nk, causal):
    if not causal:
        return nq * nk
    first = nk - nq + 1  # keys that the first query sees
    skipped = max(0, -first + 1)
    return (nq - skipped) * (max(first, 1) + nk) // 2 if nq > skipped else 0


def work(case):
    if case["op"] == "tables":
        dims = [int(d) for d in case["dims"].split(",")]
        n = case["positions"]
        return {"bytes": n * (4 * len(dims) + 4 * sum(dims)), "flops": n * sum(dims) * 10}
    size = _BYTES[case["type"]]
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"]
        values = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 + (3 if case["grad"] and case["norm"] else 2 if case["grad"] else 0)
        if case["grad"] and case["norm"]:
            passes -= 1  # x is read by the pass once
        return {"bytes": passes * values * size + 4 * case["rotated"] * (rows if case["gather"] else case["tokens"]),
                "flops": values * (10 if not case["grad"] else 25)}
    q, k = _lengths(case)
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    pairs = sum(_pairs(a, b, case["causal"]) for a, b in zip(q, k))
    q_values, k_values = sum(q) * heads * dim, sum(k) * kv_heads * dim
    # forward: q, k, v read, the result written; backward: its gradient read, three written
    values = 2 * q_values + 2 * k_values + (2 * q_values + 2 * k_values if case["grad"] else 0)
    return {"bytes": size * values, "flops": pairs * heads * dim * (14 if case["grad"] else 4)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------

_YARN = {"original_length": 32768, "beta_fast": 32.0, "beta_slow": 1.0}


def _scaling(case):
    if case["scaling"] == "none":
        return None
    scaling = {"type": case["scaling"], "factor": case["factor"]}
    if case["scaling"] == "yarn":
        scaling.update(_YARN)
    return scaling


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    state = {"case": case}
    if case["op"] == "tables":
        dims = tuple(int(d) for d in case["dims"].split(","))
        n = case["positions"]
        if len(dims) == 1:  # a run of positions behind a prefix
            start = int(torch.randint(0, 4096, (1,), generator=g, device="cuda"))
            positions = torch.arange(start, start + n, device="cuda", dtype=torch.int32)
        else:  # text tokens at the origin, image tokens on a centred grid
            positions = torch.randint(-96, 97, (n, len(dims)), generator=g, device="cuda", dtype=torch.int32)
        state.update(positions=positions, dims=dims[0] if len(dims) == 1 else dims, scaling=_scaling(case))
        return state
    dtype = _TYPES[case["type"]]
    if case["op"] == "rotary":
        batch, tokens, heads, kv_heads, dim, rotated = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim", "rotated"))
        if case["packed"]:  # q, k and v side by side, as one stacked product leaves them
            stacked = normal(batch, tokens, heads + 2 * kv_heads, dim, std=1.5, dtype=dtype)
            q, k = stacked[:, :, :heads], stacked[:, :, heads:heads + kv_heads]
        else:
            q = normal(batch, tokens, heads, dim, std=1.5, dtype=dtype)
            k = normal(batch, tokens, kv_heads, dim, std=1.5, dtype=dtype)
        rows = 4 * tokens + 7 if case["gather"] else tokens
        angles = torch.rand(rows, rotated // 2, generator=g, device="cuda") * 6.283
        state.update(q=q, k=k, cos=angles.cos(), sin=angles.sin(), positions=None, q_weight=None, k_weight=None)
        if case["gather"]:
            state["positions"] = torch.randint(0, rows, (batch, tokens), generator=g, device="cuda", dtype=torch.int32)
        if case["norm"]:
            state["q_weight"] = normal(dim, std=0.1, dtype=torch.float32).add(1.0).to(dtype)
            state["k_weight"] = normal(dim, std=0.1, dtype=torch.float32).add(1.0).to(dtype)
        if case["grad"]:
            state["dq"] = normal(batch, tokens, heads, dim, dtype=dtype)
            state["dk"] = normal(batch, tokens, kv_heads, dim, dtype=dtype)
            state["leaves"] = [t.requires_grad_() for t in (q, k, state["q_weight"], state["k_weight"]) if t is not None]
            if case["packed"]:
                state["q"], state["k"] = state["leaves"][:2]
        return state
    q_lengths, k_lengths = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    lead_q, lead_k = (case["queries"],), (case["keys"],)
    if case["form"] == "batched":
        lead_q, lead_k = (case["batch"],) + lead_q, (case["batch"],) + lead_k
    # heads as the norm in front leaves them; scores of a few units, so that some keys matter more than others
    q = normal(*lead_q, heads, dim, std=1.5, dtype=dtype)
    k = normal(*lead_k, kv_heads, dim, std=1.0, dtype=dtype)
    v = normal(*lead_k, kv_heads, dim, std=1.0, dtype=dtype)
    state.update(q=q, k=k, v=v, lengths=(q_lengths, k_lengths), keywords={})

    def ints(values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)

    if case["form"] == "packed":
        def offsets(lengths):
            out = [0]
            for n in lengths:
                out.append(out[-1] + n)
            return ints(out)
        state["keywords"] = {"q_offsets": offsets(q_lengths), "k_offsets": offsets(k_lengths)}
    elif case["ragged"]:
        state["keywords"] = {"k_lengths": ints(k_lengths)}
        if q_lengths == k_lengths:
            state["keywords"]["q_lengths"] = ints(q_lengths)
    if case["grad"]:
        state["dy"] = normal(*lead_q, heads, dim, dtype=dtype)
        for t in (q, k, v):
            t.requires_grad_()
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "tables":
        if own:
            import mflux_amd

            return mflux_amd.rotary_tables(state["positions"], state["dims"], base=case["base"], scaling=state["scaling"])
        return _plain_tables(state)
    if case["op"] == "rotary":
        if not own:
            return _plain_rotary(state)
        import mflux_amd

        outputs = mflux_amd.rotary(state["q"], state["k"], state["cos"], state["sin"], layout=case["layout"],
                                   positions=state["positions"], q_weight=state["q_weight"], k_weight=state["k_weight"])
        if not case["grad"]:
            return outputs
        return [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, state["leaves"], (state["dq"], state["dk"])))
    if not own:
        return _plain_attention(state)
    import mflux_amd

    y = mflux_amd.attention(state["q"], state["k"], state["v"], causal=case["causal"], **state["keywords"])
    if not case["grad"]:
        return y
    return [y.detach()] + list(torch.autograd.grad(y, (state["q"], state["k"], state["v"]), state["dy"]))


# ---- the plain forms -------------------------------------------------------------------------------------------------------------

def _frequencies(dim, base, scaling):
    """(inverse frequencies in 64 bits, factor of the tables)."""
    i = torch.arange(0, dim, 2, device="cuda", dtype=torch.float64)
    if scaling is None:
        return base ** (-i / dim), 1.0
    factor = scaling["factor"]
    if scaling["type"] == "linear":
        return base ** (-i / dim) / factor, 1.0
    if scaling["type"] == "ntk":
        return (base * factor ** (dim / (dim - 2))) ** (-i / dim), 1.0
    plain = base ** (-i / dim)

    def index_of(turns):  # of the frequency that makes so many turns over the original length
        return dim * math.log(scaling["original_length"] / (turns * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(index_of(scaling["beta_fast"])), 0)
    high = min(math.ceil(index_of(scaling["beta_slow"])), dim - 1)
    ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    return plain / factor * ramp + plain * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _plain_tables(state):
    case, positions, dims = state["case"], state["positions"], state["dims"]
    if isinstance(dims, int):
        positions, dims = positions[:, None], (dims,)
    cos, sin = [], []
    for axis, dim in enumerate(dims):
        frequencies, factor = _frequencies(dim, case["base"], state["scaling"])
        angles = positions[:, axis, None].double() * frequencies
        cos.append((angles.cos() * factor).float())
        sin.append((angles.sin() * factor).float())
    return torch.cat(cos, dim=1), torch.cat(sin, dim=1)


def _tables_of(state, dtype):
    cos, sin = state["cos"].to(dtype), state["sin"].to(dtype)
    if state["positions"] is not None:
        index = state["positions"].long()
        return cos[index][:, :, None], sin[index][:, :, None]
    return cos[None, :, None], sin[None, :, None]


def _rotate(x, cos, sin, layout, rotated):
    head, rest = x[..., :rotated], x[..., rotated:]
    if layout == "half":
        a, b = head[..., :rotated // 2], head[..., rotated // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)


def _plain_rotary(state):
    case = state["case"]
    cos, sin = _tables_of(state, torch.float32)
    results, gradients, weight_gradients = [], [], []
    for name in ("q", "k"):
        raw, weight = state[name].detach(), state[name + "_weight"]
        x = raw.float()
        if weight is not None:
            w = weight.detach().float()
            rstd = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6)
            n = x * rstd
            results.append(_rotate(n * w, cos, sin, case["layout"], case["rotated"]).to(raw.dtype))
        else:
            results.append(_rotate(x, cos, sin, case["layout"], case["rotated"]).to(raw.dtype))
        if case["grad"]:
            dn = _rotate(state["d" + name].float(), cos, -sin, case["layout"], case["rotated"])
            if weight is not None:
                weight_gradients.append((dn * n).flatten(0, -2).sum(dim=0).to(weight.dtype))
                dn = dn * w
                dn = rstd * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
            gradients.append(dn.to(raw.dtype))
    return results + gradients + weight_gradients


def _visible(nq, nk):
    """[nq, nk], true where a query sees a key; aligned to the end."""
    rows = torch.arange(nq, device="cuda")[:, None] + (nk - nq)
    return torch.arange(nk, device="cuda")[None, :] <= rows


def _plain_sequence(q, k, v, causal, dy):
    """One sequence: q [nq, H, D], k and v [nk, Hkv, D] -> outputs in 32 bits."""
    nq, heads, dim = q.shape
    nk, kv_heads = k.shape[:2]
    group = heads // kv_heads
    y = torch.zeros(nq, heads, dim, device="cuda")
    dq = torch.zeros_like(y) if dy is not None else None
    dk = torch.zeros(nk, kv_heads, dim, device="cuda") if dy is not None else None
    dv = torch.zeros_like(dk) if dy is not None else None
    if nq == 0 or nk == 0:
        return y, dq, dk, dv
    scale = 1.0 / math.sqrt(dim)
    visible = _visible(nq, nk) if causal else None
    step = max(1, min(kv_heads, (1 << 29) // max(1, nq * nk * group)))
    for h in range(0, kv_heads, step):
        n = min(step, kv_heads - h)
        qs = q[:, h * group:(h + n) * group].float().reshape(nq, n, group, dim).permute(1, 2, 0, 3).reshape(n, group * nq, dim)
        ks = k[:, h:h + n].float().transpose(0, 1).contiguous()
        vs = v[:, h:h + n].float().transpose(0, 1).contiguous()
        s = torch.bmm(qs, ks.transpose(1, 2).contiguous()).mul_(scale).view(n, group, nq, nk)
        if visible is not None:
            s.masked_fill_(~visible, float("-inf"))
        top = s.amax(dim=-1, keepdim=True)
        p = s.sub_(top.clamp(min=-1e30)).exp_()
        p.div_(p.sum(dim=-1, keepdim=True).clamp(min=1e-30))
        p = p.view(n, group * nq, nk)
        o = torch.bmm(p, vs)

        def back(t):
            return t.view(n, group, nq, dim).permute(2, 0, 1, 3).reshape(nq, n * group, dim)

        y[:, h * group:(h + n) * group] = back(o)
        if dy is not None:
            ds = dy[:, h * group:(h + n) * group].float().reshape(nq, n, group, dim).permute(1, 2, 0, 3).reshape(n, group * nq, dim)
            dv[:, h:h + n] = torch.bmm(p.transpose(1, 2).contiguous(), ds).transpose(0, 1)
            dp = torch.bmm(ds, vs.transpose(1, 2).contiguous())
            dp = p * (dp - (ds * o).sum(dim=-1, keepdim=True)) * scale
            dq[:, h * group:(h + n) * group] = back(torch.bmm(dp, ks))
            dk[:, h:h + n] = torch.bmm(dp.transpose(1, 2).contiguous(), qs).transpose(0, 1)
    return y, dq, dk, dv


def _plain_tokens(state):
    """A few queries of every sequence against padded keys, all sequences at once."""
    q, k, v = state["q"], state["k"], state["v"]
    batch, nq, heads, dim = q.shape
    nk, kv_heads = k.shape[1:3]
    group = heads // kv_heads
    qs = q.float().view(batch, nq, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch * kv_heads, group * nq, dim)
    ks = k.float().transpose(1, 2).reshape(batch * kv_heads, nk, dim)
    s = torch.bmm(qs, ks.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(dim)).view(batch, kv_heads, group, nq, nk)
    lengths = torch.full((batch,), nk, device="cuda") if "k_lengths" not in state["keywords"] else state["keywords"]["k_lengths"]
    rows = torch.arange(nq, device="cuda")[None, :, None] + (lengths[:, None, None] - nq)
    if not state["case"]["causal"]:
        rows = (lengths - 1)[:, None, None].expand(batch, nq, 1)
    hidden = torch.arange(nk, device="cuda")[None, None, :] > rows
    s.masked_fill_(hidden[:, None, None], float("-inf"))
    p = s.sub_(s.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    p.div_(p.sum(dim=-1, keepdim=True).clamp(min=1e-30))
    o = torch.bmm(p.view(batch * kv_heads, group * nq, nk), v.float().transpose(1, 2).reshape(batch * kv_heads, nk, dim))
    return o.view(batch, kv_heads, group, nq, dim).permute(0, 3, 1, 2, 4).reshape(batch, nq, heads, dim).to(q.dtype)


def _sequences(state):
    """For every sequence, the places of its queries and of its keys."""
    q_lengths, k_lengths = state["lengths"]
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(zip(q_lengths, k_lengths)):
        if state["case"]["form"] == "packed":
            yield slice(q0, q0 + nq), slice(k0, k0 + nk)
            q0, k0 = q0 + nq, k0 + nk
        else:
            yield (b, slice(0, nq)), (b, slice(0, nk))


def _plain_attention(state):
    case = state["case"]
    q, k, v = state["q"].detach(), state["k"].detach(), state["v"].detach()
    if case["form"] == "batched" and case["queries"] <= 4 < case["keys"] and not case["grad"]:
        return _plain_tokens(state)
    dy = state.get("dy")
    y = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if dy is not None else (None, None, None)
    for qi, ki in _sequences(state):
        parts = _plain_sequence(q[qi], k[ki], v[ki], case["causal"], None if dy is None else dy[qi])
        y[qi] = parts[0].to(y.dtype)
        if dy is not None:
            dq[qi], dk[ki], dv[ki] = (t.to(y.dtype) for t in parts[1:])
    return y if dy is None else [y, dq, dk, dv]


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(case, state)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    if work(case)["flops"] > 1.6e13:
        return None
    return _exact_attention(case, state)


def _exact_tables(case, state):
    dims = [int(d) for d in case["dims"].split(",")]
    positions = state["positions"].reshape(case["positions"], len(dims)).double()
    columns, factor, table_factor = [], case["factor"], 1.0
    for axis, dim in enumerate(dims):
        for j in range(dim // 2):
            base = case["base"]
            if case["scaling"] == "ntk":
                base *= factor ** (dim / (dim - 2))
            frequency = base ** (-2.0 * j / dim)
            if case["scaling"] == "linear":
                frequency /= factor
            elif case["scaling"] == "yarn":
                table_factor = 1.0 + 0.1 * math.log(factor)
                length = _YARN["original_length"]
                ends = [dim * math.log(length / (2 * math.pi * beta)) / (2 * math.log(base))
                        for beta in (_YARN["beta_fast"], _YARN["beta_slow"])]
                first, last = max(0, math.floor(ends[0])), min(dim - 1, math.ceil(ends[1]))
                slow = min(1.0, max(0.0, (j - first) / max(last - first, 0.001)))
                frequency *= (1.0 - slow) + slow / factor
            columns.append(positions[:, axis] * frequency)
    angles = torch.stack(columns, dim=1)
    return angles.cos() * table_factor, angles.sin() * table_factor


def _exact_rotary(case, state):
    rotated, dim, tokens, batch = case["rotated"], case["dim"], case["tokens"], case["batch"]
    half = rotated // 2
    # the rotation as a complex product
    turn = torch.complex(state["cos"].double(), state["sin"].double())
    turn = turn[state["positions"].long()] if case["gather"] else turn.expand(batch, tokens, half)
    turn = turn[:, :, None]
    pairs = torch.arange(rotated, device="cuda").view(2, half) if case["layout"] == "half" else \
        torch.arange(rotated, device="cuda").view(half, 2).t()

    def rotate(x, by):
        z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * by
        out = x.clone()
        out[..., pairs[0]], out[..., pairs[1]] = z.real, z.imag
        return out

    first, second, third = [], [], []
    for x, w, dy in ((state["q"], state["q_weight"], state.get("dq")), (state["k"], state["k_weight"], state.get("dk"))):
        x = x.detach().double()
        size = ((x ** 2).sum(-1, keepdim=True) / dim + 1e-6).sqrt()
        w = None if w is None else w.detach().double()
        first.append(rotate(x if w is None else x / size * w, turn))
        if dy is None:
            continue
        d = rotate(dy.double(), turn.conj())
        if w is None:
            second.append(d)
            continue
        third.append((d * x / size).sum(dim=(0, 1, 2)))
        d = d * w
        second.append(d / size - x * (d * x).sum(-1, keepdim=True) / (dim * size ** 3))
    return first + second + third


def _exact_attention(case, state):
    q, k, v, dy = state["q"].detach(), state["k"].detach(), state["v"].detach(), state.get("dy")
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    outputs = [torch.zeros(q.shape, device="cuda", dtype=torch.float64)]
    if dy is not None:
        outputs += [torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (q, k, v)]
    for qi, ki in _sequences(state):
        nq, nk = q[qi].shape[0], k[ki].shape[0]
        if nq == 0 or nk == 0:
            continue
        for h in range(heads):
            one, two, three = q[qi][:, h].double(), k[ki][:, h * kv_heads // heads].double(), v[ki][:, h * kv_heads // heads].double()
            weights = one @ two.t().contiguous() / math.sqrt(dim)
            if case["causal"]:
                ahead = torch.ones(nq, nk, device="cuda", dtype=torch.bool).triu(nk - nq + 1)
                weights[ahead] = -math.inf
            total = torch.logsumexp(weights, dim=1, keepdim=True)
            weights = torch.where(torch.isinf(total), 0.0, (weights - total).exp())
            value = weights @ three
            outputs[0][qi][:, h] = value
            if dy is not None:
                up = dy[qi][:, h].double()
                outputs[3][ki][:, h * kv_heads // heads] += weights.t().contiguous() @ up
                change = weights * (up @ three.t().contiguous() - (up * value).sum(1, keepdim=True)) / math.sqrt(dim)
                outputs[1][qi][:, h] = change @ two
                outputs[2][ki][:, h * kv_heads // heads] += change.t().contiguous() @ one
    return outputs[0] if dy is None else outputs
