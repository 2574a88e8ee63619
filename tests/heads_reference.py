"""The heads' operators in float64, with how far a kernel's results may be off.

Bounds, with u half a step of the 16-bit type and e = 2^-24 of float32:

attention   A probability p is rounded once (u p), its score is a float32 sum of dim products (off by dim e
            sum |q k|, which is the same relative error of p after the exponential; the exponential and the factors add a few e more),
            and the sums over keys are float32 (at most one e an addition).  float16 also loses 2^-25 of a probability that is not
            normal there, times |v|.  The probabilities are divided by the sum of the rounded ones, so that they add up to 1: a sum
            that is off by u at most, which is u |y| of the result and u of every probability that the backward pass makes from the
            saved log-sum-exp.  Then y is rounded.
gradients   p as above from the saved float32 log-sum-exp; dS = p (dP - delta) is rounded once, and delta = sum dy y is as far off as
            y is.  Then the sums and the rounding of the result.  float16 rounds multiples of its gradients: 2^13 p, so less than 2^-33 of a
            probability is lost (and of the forward pass's, multiples as well, less than 2^-25), and dS times a power of two that has a column's largest at 2^4 or above, so at most 2^-28 of that.
"""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 0.0}
# what may be lost below the smallest normal number
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0, torch.float64: 0.0}
E = 2.0 ** -24


def rotary_frequencies(dim, base, scaling):
    """The angle a position adds to each pair, and the factor of the tables.  yarn: a pair that makes more than beta_fast turns over
    the original length keeps its angle, one that makes less than beta_slow has it divided, with whole pairs as the ends of the ramp."""
    kind, factor = (None, 1.0) if scaling is None else (scaling["type"], scaling["factor"])
    if kind == "ntk":
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind != "yarn":
        return f, 1.0
    length = scaling["original_length"]

    def pair(turns):  # turns = length * base^(-2 i / dim) / (2 pi), for i
        return dim / 2 * math.log(length / (2 * math.pi * turns)) / math.log(base)

    low, high = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0), min(math.ceil(pair(scaling.get("beta_slow", 1.0))), dim - 1)
    share = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(dim // 2)]
    tables = scaling.get("attention_factor")
    return [x * (1 - t) + x / factor * t for x, t in zip(f, share)], 1 + 0.1 * math.log(factor) if tables is None else tables


def visible(nq, nk, causal, device):
    if not causal:
        return torch.ones(nq, nk, dtype=torch.bool, device=device)
    return torch.arange(nk, device=device)[None] <= torch.arange(nq, device=device)[:, None] + (nk - nq)


def attention_sequence(q, k, v, causal, scale, dy=None, lost_p=None):
    """q [nq, H, D], k and v [nk, Hkv, D] of one sequence: {"y": (value, bound), and with dy "dq", "dk", "dv"}, float64.
    lost_p: what float16 may lose of a probability, in the result and in dv (default: as derived above)."""
    nq, H, D = q.shape
    nk, Hkv = k.shape[:2]
    g = H // Hkv
    u, tiny = HALF[q.dtype], TINY[q.dtype]
    lost_y, lost_dv = (tiny, tiny * 2.0 ** -8) if lost_p is None else lost_p
    q, k, v = q.double(), k.double(), v.double()
    names = ["y"] if dy is None else ["y", "dq", "dk", "dv"]
    shapes = {"y": q, "dq": q, "dk": k, "dv": v}
    out = {n: (torch.zeros_like(shapes[n]), torch.zeros_like(shapes[n])) for n in names}
    if nq == 0 or nk == 0:
        return out
    see = visible(nq, nk, causal, q.device)
    some = see.any(1, keepdim=True)
    for h in range(H):
        qh, kh, vh = q[:, h], k[:, h // g], v[:, h // g]
        s = scale * (qh @ kh.t().contiguous())
        top = s.masked_fill(~see, -math.inf).amax(1, keepdim=True)
        p = torch.where(see, (s - torch.where(some, top, 0.0)).exp(), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        p = torch.where(some & see, p, 0.0)
        y = p @ vh
        # relative error of a probability before its rounding
        size = torch.where(see, scale * (qh.abs() @ kh.abs().t().contiguous()), 0.0).amax()
        c = E * (2 * (D + 8) * size + 8 * top[some].abs().amax().clamp(min=1.0) + nk + 32) if some.any() else torch.tensor(0.0).to(q)
        av = p @ vh.abs()
        lost = lost_y * (see.double() @ vh.abs())
        out["y"][0][:, h] = y
        bound = ((u + c) * av + u * y.abs()) * 1.01 + lost
        out["y"][1][:, h] = bound + u * (y.abs() + bound) + tiny
        if dy is None:
            continue
        dyh = dy[:, h].double()
        dp = dyh @ vh.t().contiguous()
        delta = (dyh * y).sum(1, keepdim=True)
        ds = torch.where(see, p * (dp - delta), 0.0)
        adp = dyh.abs() @ vh.abs().t().contiguous()
        adelta = (dyh.abs() * (y.abs() + out["y"][1][:, h])).sum(1, keepdim=True)
        # dS before its rounding: p's relative error, dP's and delta's float32 sums, delta's rounded y
        eds = (u + c) * ds.abs() + torch.where(see, p * (E * (D + 4) * (adp + adelta) + (dyh.abs() * out["y"][1][:, h]).sum(1, keepdim=True)), 0.0)
        eds = (eds + u * (ds.abs() + eds) + (tiny > 0) * 2.0 ** -28 * ds.abs().amax() * see) * 1.01
        ep = torch.where(see, (2 * u + c) * p * 1.01 + lost_dv, 0.0)
        n = nq * g
        for name, value, error, first in (
                ("dq", scale * (ds @ kh), scale * (eds @ kh.abs() + E * (nk + 4) * (ds.abs() @ kh.abs())), True),
                ("dk", scale * (ds.t().contiguous() @ qh), scale * (eds.t().contiguous() @ qh.abs() + E * (n + 4) * (ds.abs().t().contiguous() @ qh.abs())), h % g == 0),
                ("dv", p.t().contiguous() @ dyh, ep.t().contiguous() @ dyh.abs() + E * (n + 4) * (p.t().contiguous() @ dyh.abs()), h % g == 0)):
            i = h if name == "dq" else h // g
            out[name][0][:, i] += value
            out[name][1][:, i] += error
    if dy is not None:
        for name in ("dq", "dk", "dv"):
            value, error = out[name]
            out[name] = value, error + u * (value.abs() + error) + tiny
    return out


def rms_norm_rotary(x, cos, sin, layout, weight, eps, dy=None):
    """x [B, S, H, D] with the tables' rows of every token [B, S, R / 2]: (y, bound), and with dy (dx, bound), (dw, bound)."""
    u, tiny, D = HALF[x.dtype], TINY[x.dtype], x.shape[-1]
    R = 2 * cos.shape[-1]
    x, cos, sin = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    w = None if weight is None else weight.double()
    if layout == "half":
        first, second = torch.arange(R // 2, device=x.device), torch.arange(R // 2, device=x.device) + R // 2
    else:
        first, second = 2 * torch.arange(R // 2, device=x.device), 2 * torch.arange(R // 2, device=x.device) + 1

    def turn(t, sin, cos=cos):
        out = t.clone()
        out[..., first] = t[..., first] * cos - t[..., second] * sin
        out[..., second] = t[..., second] * cos + t[..., first] * sin
        return out

    def turn_sizes(t):  # of both products of every value
        a, c, n = t.abs(), cos.abs(), sin.abs()
        out = a.clone()
        out[..., first] = a[..., first] * c + a[..., second] * n
        out[..., second] = a[..., second] * c + a[..., first] * n
        return out

    r = None if w is None else 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x if w is None else x * r * w
    y = turn(n, sin)
    # float32 steps: the mean's sum of D terms, a root, a quotient, two products, the turn's two products and sum
    steps = E * (8 + (0 if w is None else D / 2 + 8))
    size = turn_sizes(n)
    results = [(y, steps * size + u * y.abs() * (1 + 2 * steps) + u * steps * size + tiny)]
    if dy is None:
        return results
    dy = dy.double()
    d, dsize = turn(dy, -sin), turn_sizes(dy)
    if w is None:
        results.append((d, E * 8 * dsize + u * d.abs() * (1 + E * 8) + tiny))
        return results
    nx = x * r
    count = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (d * nx).sum((0, 1, 2))
    # a sum in several float32 stages: far below one e an addition
    dwsize = (dsize * nx.abs()).sum((0, 1, 2))
    results_w = (dw, E * (D / 2 + 32 + min(count, 4096)) * dwsize + u * dw.abs() * 1.01 + tiny)
    dn, dnsize = d * w, dsize * w.abs()
    mean, meansize = (dn * nx).mean(-1, keepdim=True), (dnsize * nx.abs()).mean(-1, keepdim=True)
    dx = r * (dn - nx * mean)
    dxsize = r * (dnsize + nx.abs() * meansize)
    results.append((dx, E * (2 * D + 64) * dxsize + u * dx.abs() * 1.01 + tiny))
    results.append(results_w)
    return results


def check(name, got, value, bound):
    got = got.detach().double()
    assert got.shape == value.shape, f"{name}: {tuple(got.shape)} instead of {tuple(value.shape)}"
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = tuple(int(j) for j in bad.nonzero()[0])
        worst = (off / bound.clamp(min=1e-300)).nan_to_num(math.inf).amax()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values out of bounds, first at {i}: {float(got[i])} instead of "
                             f"{float(value[i])} +- {float(bound[i])}; worst {float(worst):.3g} times its bound")
