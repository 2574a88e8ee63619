"""The norm, the codes and the product of codes in float64, with how far a kernel's results may be off.

Bounds, with u half a step of the result's type and e = 2^-24 of float32:

norm        sum(s^2) has positive terms: each is rounded once, and it passes at most n = K / 64 + 16 additions (a lane's own, the
            tree's), so it is off by (n + 1) e of itself; the mean, eps, the root and its inverse add 4 e, and the root halves what was
            before it.  y = s r w: two products more, and its rounding.
gradients   dot = sum(dy w s) is off by (n + 2) e sum |dy w s|.  dx = r (dy w - m n) + ds with m = r dot / K and n = s r: each factor
            r and n as off as above; the products and sums add 6 e of their terms.  dw adds up rows: at most rows + n additions.
scales      max|p| is exact for the 16-bit types (a product is 16 or 22 bits long) and rounded once for float32; then r, one
            product and one division.  Without a norm it is one division.
codes       equal to those of the exact quotient.
product     the sum is exact, its conversion, the two scales and the bias are a rounding each, then the result's.
"""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half of what lies between the smallest numbers
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
E = 2.0 ** -24


def total(x, residual):
    """What is normalised: the sum as it is stored.  Two numbers of a 16-bit type add up in float32 to what rounds like their sum."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def rms_norm(s, weight, eps, dy=None, dsum=None):
    """s: what is normalised.  {"y": (value, bound), and with dy "dx", "dw"}, float64."""
    u, tiny, K = HALF[s.dtype], TINY[s.dtype], s.shape[-1]
    v = s.detach().double()
    w = torch.ones(K, device=s.device, dtype=torch.float64) if weight is None else weight.detach().double()
    n = K // 64 + 16
    root = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    off = ((n + 1) / 2 + 4) * E  # of the root
    y = v * root * w
    out = {"y": (y, y.abs() * (u + off + 2 * E) * (1 + u) + tiny)}
    if dy is None:
        return out
    a, nv = dy.detach().double() * w, v * root
    mean = (a * nv).mean(-1, keepdim=True)
    spread = (a * nv).abs().mean(-1, keepdim=True)
    dx = root * (a - nv * mean)
    bound = root * (a.abs() * (off + 6 * E) + nv.abs() * (spread * ((n + 2) * E + 2 * off + 4 * E) + mean.abs() * (2 * off + 6 * E)))
    if dsum is not None:
        dx = dx + dsum.detach().double()
        bound = bound + dsum.detach().double().abs() * E
    bound = bound + dx.abs() * E
    out["dx"] = (dx, bound * (1 + u) + dx.abs() * u + tiny)
    terms = (dy.detach().double() * nv).reshape(-1, K)
    dw = terms.sum(0)
    out["dw"] = (dw, terms.abs().sum(0) * (terms.shape[0] + n + off / E + 2) * E * (1 + u) + dw.abs() * u + tiny)
    return out


def codes(s, weight=None, eps=None):
    """(codes, scales) of rows, float64; eps: with a norm in front."""
    v = s.detach().double()
    p = v if weight is None else v * weight.detach().double()
    top = p.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(p * 127 / top), 0.0)
    root = torch.ones_like(top) if eps is None else 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    return q, (top * root / 127)[..., 0]


def scale_bound(K, norm):
    return (1 + ((K // 64 + 17) / 2 + 6 if norm else 1)) * E


def product(x, x_scales, w, w_scales, bias, dtype):
    sums = torch.mm(x.reshape(-1, x.shape[-1]).double(), w.double().t().contiguous())
    y = sums * x_scales.reshape(-1, 1).double() * w_scales.double()
    bound = y.abs() * 3 * E * (1 + 4 * E)
    if bias is not None:
        y = y + bias.double()
    bound = (bound + y.abs() * E) * (1 + HALF[dtype]) + y.abs() * HALF[dtype] + TINY[dtype]
    return y.reshape(*x.shape[:-1], w.shape[0]), bound.reshape(*x.shape[:-1], w.shape[0])


def check(name, got, value, bound):
    err = (got.detach().double() - value).abs()
    worst = float((err / bound.clamp(min=1e-300)).max()) if err.numel() else 0.0
    assert got.shape == value.shape, (name, tuple(got.shape), tuple(value.shape))
    assert bool((err <= bound).all()), f"{name}: {worst} of what it may be off, at {int((err / bound.clamp(min=1e-300)).argmax())}"
