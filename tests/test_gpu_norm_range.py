"""rms_norm and the codes behind it at the ends of what they take: rows of millions of values, millions of rows, values whose squares
leave float32, more rows than workgroups in every form of a row, and what its results' gradients are.

Bounds, with E = 2^-24: where a row's sum is right to E or better, a norm is off by the root's rounding, two products and the result's
(int8_reference has those of the shorter rows, which grow with a row's length)."""
import pytest
import torch

import int8_reference as ref
from test_gpu_int8 import BF16, F16, F32, randn
from test_gpu_int8_calls import room

pytestmark = pytest.mark.gpu
E = ref.E


def close(name, got, value, relative, scale=None):
    """|got - value| <= relative * scale (|value| where there is none) + the result's rounding."""
    err = (got.double() - value).abs()
    bound = (value.abs() if scale is None else scale) * relative + value.abs() * ref.HALF[got.dtype] * (1 + 2 * relative) + ref.TINY[got.dtype]
    assert bool((err <= bound).all()), f"{name}: {float((err / bound).max())} of what it may be off"


def drifting(rows, K):
    """[rows, K] of numbers that a float32 sum drifts away from where they are the same again and again, and of others."""
    dy = randn(1, rows, K)
    dy[:, :K // 2] = torch.tensor([1 / 3, 0.7, 0.1, 0.9, 0.55], device="cuda").repeat(K)[:K // 2]
    return dy


# ---- the weight's gradient -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,K,sums", [(512, 4096, 0), (300, 8192, 0), (512, 1000, 3), (512, 4097, 0), (512, 40001, 0)])
def test_weight_gradient_is_rounded_once(rows, K, sums):
    """Rows of 1 and -1, whose normalised values are these: dw is the sum of dy.  A workgroup has a row of its own (or four, three float32
    additions); what it hands on is added up without any other rounding than the result's (float64: 512 of 2^-53)."""
    import mflux_amd

    print(f"rows={rows} K={K}", flush=True)
    x = torch.ones(rows, K, device="cuda")
    x[:, ::2] = -1
    w, dy = torch.ones(K, device="cuda").requires_grad_(), drifting(rows, K)
    dw, = torch.autograd.grad(mflux_amd.rms_norm(x, w, eps=0.0), w, dy)
    terms = dy.double() * x.double()
    close("dw", dw, terms.sum(0), sums * E + 2.0 ** -43, terms.abs().sum(0))


@pytest.mark.parametrize("rows,K,sums", [(1 << 22, 64, 130), (1 << 21, 500, 130), (1 << 19, 1030, 127), (1 << 17, 4100, 127), (150_000, 4097, 127),
                                         (140_000, 2048, 127)])
def test_weight_gradient_of_many_rows(rows, K, sums):
    """As above: a lane adds up 128 rows at most (and a workgroup its four wavefronts') in float32."""
    import mflux_amd

    room(40)
    print(f"rows={rows} K={K}", flush=True)
    x = torch.ones(rows, K, device="cuda")
    x[:, ::2] = -1
    w, dy, n = torch.ones(K, device="cuda").requires_grad_(), drifting(500, K), -(-rows // 500)
    dw, = torch.autograd.grad(mflux_amd.rms_norm(x, w, eps=0.0), w, dy.repeat(n, 1)[:rows])
    terms = dy.double() * x[:500].double()
    rest = terms[:rows - (n - 1) * 500]
    spread = (n - 1) * terms.abs().sum(0) + rest.abs().sum(0)
    close("dw", dw, (n - 1) * terms.sum(0) + rest.sum(0), sums * E + 2.0 ** -37, spread)


# ---- long rows -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("K", [(1 << 22) + 4, (1 << 23) + 12])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_of_rows_of_millions(K, dtype):
    """Equal values, whose squares no short sum of float32 adds up without a drift; the bound does not grow with the row."""
    import mflux_amd

    print(f"K={K} {dtype}", flush=True)
    x = torch.stack([torch.full((K,), 0.7, device="cuda"), torch.full((K,), -0.1, device="cuda"), randn(1, K)]).to(dtype).requires_grad_()
    w = (1 + 0.1 * randn(2, K)).to(dtype).requires_grad_()
    dy = torch.where(torch.arange(K, device="cuda") % 3 == 0, 0.9, 0.3).to(dtype).expand(3, K)
    y = mflux_amd.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    v, g, d = x.detach().double(), w.detach().double(), dy.double()
    root = 1 / (v.square().mean(1, keepdim=True) + 1e-6).sqrt()
    close("y", y.detach(), v * root * g, 4 * E)
    n, a = v * root, d * g
    mean = (a * n).mean(1, keepdim=True)
    # the two terms of dx: each to its factors' roundings
    close("dx", dx, root * (a - n * mean), 8 * E, root * (a.abs() + n.abs() * mean.abs()))
    close("dw", dw, (d * n).sum(0), 8 * E, (d * n).abs().sum(0))
    q, s = mflux_amd.rms_norm_int8(x.detach(), w.detach())
    want_q, want_s = ref.codes(x, w, 1e-6)
    assert torch.equal(q.double(), want_q)
    assert bool(((s.double() - want_s).abs() <= want_s * 5 * E).all())


@pytest.mark.parametrize("K,dtype", [((1 << 26) - 15, F32), (1 << 26, F32), (1 << 26, BF16), (1 << 28, BF16)])
def test_weight_gradient_of_the_longest_rows(K, dtype):
    """More columns than one launch has sixteens for, up to the longest row there is.  Values of 1 and -1, whose sums are exact."""
    import mflux_amd

    room(30)
    print(f"K={K} {dtype}", flush=True)
    sign = torch.ones(K, device="cuda", dtype=dtype)
    sign[::3] = -1
    x, w = sign[None], torch.full((K,), 0.5, device="cuda", dtype=dtype).requires_grad_()
    dy = torch.full((K,), 0.25, device="cuda", dtype=dtype)
    dy[5::7] = -2
    y = mflux_amd.rms_norm(x, w, eps=0.0)
    assert torch.equal(y.detach(), x * 0.5)
    dw, = torch.autograd.grad(y, w, dy[None])
    assert torch.equal(dw, sign * dy)


# ---- values whose squares leave float32 --------------------------------------------------------------------------------------

SIZES = [1e18, 3e25, 1e38]


@pytest.mark.parametrize("K", [1, 64, 67, 1024, 1100, 3840, 5000, 16384, 16400, 40001])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_of_large_values(K, dtype):
    """Finite rows whose sum of squares is beyond float32's range: normalised like any others, among others."""
    import mflux_amd

    print(f"K={K} {dtype}", flush=True)
    unit = randn(1, 6, K).clamp(-3, 3)
    size = torch.tensor([1.0, *SIZES, 1e-3, 1e19], device="cuda")[:, None]
    x = (unit * size).to(dtype)
    x[3, K // 2] = torch.finfo(dtype).max
    x[4, 0] = 1e30  # alone in a row of small ones
    x, r = x.requires_grad_(), (randn(2, 6, K).clamp(-3, 3) * size * 0.01).to(dtype)
    r[3] = 0
    w = (1 + 0.1 * randn(3, K)).to(dtype).requires_grad_()
    dy, ds = randn(4, 6, K, dtype=dtype), randn(5, 6, K, dtype=dtype) * 1e-20
    for residual, dsum in ((None, None), (r, ds)):
        s = ref.total(x.detach(), residual)
        assert bool(s.isfinite().all())
        out = mflux_amd.rms_norm(x, w, residual=residual)
        y = out if residual is None else out[0]
        want = ref.rms_norm(s, w, 1e-6, dy, dsum)
        ref.check("y", y, *want["y"])
        dx, dw = torch.autograd.grad(out, (x, w), dy if residual is None else (dy, dsum))
        ref.check("dx", dx, *want["dx"])
        ref.check("dw", dw, *want["dw"])
        q, sc, *_ = mflux_amd.rms_norm_int8(x.detach(), None, residual=residual)
        want_q, want_s = ref.codes(s, None, 1e-6)
        assert torch.equal(q.double(), want_q)
        ref.check("scales", sc, want_s, want_s * ref.scale_bound(K, True))


@pytest.mark.parametrize("K", [1, 64, 67, 1100, 3840, 16384, 40001])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-42])
def test_norm_of_tiny_values(K, dtype, eps):
    """Rows whose squares vanish in float32, with an eps that leaves them their size."""
    import mflux_amd

    print(f"K={K} {dtype} {eps}", flush=True)
    unit = randn(1, 4, K)
    unit[:, 0] = 1
    x = (unit * torch.tensor([1.0, 1e-18, 1e-21, 1e-30], device="cuda")[:, None]).to(dtype).requires_grad_()
    w = (1 + 0.1 * randn(2, K)).to(dtype).requires_grad_()
    dy = randn(3, 4, K, dtype=dtype) * 1e-6
    y = mflux_amd.rms_norm(x, w, eps=eps)
    held = torch.tensor(eps, dtype=F32).double().item()  # as the call holds it
    want = ref.rms_norm(x, w, held, dy)
    ref.check("y", y, *want["y"])
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref.check("dx", dx, *want["dx"])
    ref.check("dw", dw, *want["dw"])
    q, sc = mflux_amd.rms_norm_int8(x.detach(), None, eps=eps)
    want_q, want_s = ref.codes(x, None, held)
    assert torch.equal(q.double(), want_q)
    ref.check("scales", sc, want_s, want_s * ref.scale_bound(K, True) + 2.0 ** -149)


@pytest.mark.parametrize("K", [64, 67, 3840, 40001])
def test_norm_of_the_largest_values_bfloat16_has(K):
    """Rows of nothing but the largest number and its negative: a norm of one."""
    import mflux_amd

    top = torch.finfo(BF16).max
    x = torch.where(randn(1, 3, K) > 0, top, -top).to(BF16)
    y = mflux_amd.rms_norm(x)
    ref.check("y", y, *ref.rms_norm(x, None, 1e-6)["y"])
    assert bool((y.abs() == 1).all())
    q, s = mflux_amd.rms_norm_int8(x)
    assert bool((q.abs() == 127).all())
    close("values", mflux_amd.int8_dequantize(q, s, F32), x.double().sign(), (ref.scale_bound(K, True) / E + 2) * E)


# ---- more rows than workgroups -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("K", [1, 17, 513, 1025, 4099, 16392, 33001])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_of_more_rows_than_workgroups(K, dtype):
    """A workgroup's second row and those after it, in the forms of odd, of long and of short rows."""
    import mflux_amd

    rows = 2100 if K > 4096 else 20000 if K < 600 else 9000
    print(f"rows={rows} K={K} {dtype}", flush=True)
    x, r, w = randn(1, rows, K, dtype=dtype).requires_grad_(), randn(2, rows, K, dtype=dtype), randn(3, K, dtype=dtype).requires_grad_()
    dy, ds = randn(4, rows, K, dtype=dtype), randn(5, rows, K, dtype=dtype)
    y, s = mflux_amd.rms_norm(x, w, residual=r)
    want = ref.rms_norm(ref.total(x.detach(), r), w, 1e-6, dy, ds)
    ref.check("y", y, *want["y"])
    dx, dw = torch.autograd.grad((y, s), (x, w), (dy, ds))
    ref.check("dx", dx, *want["dx"])
    ref.check("dw", dw, *want["dw"])
    del want, dx, dw, y
    q, sc, _ = mflux_amd.rms_norm_int8(x.detach(), w.detach(), residual=r)
    want_q, want_s = ref.codes(s.detach(), w, 1e-6)
    assert torch.equal(q.double(), want_q)
    ref.check("scales", sc, want_s, want_s * ref.scale_bound(K, True))


# ---- what the sum's gradient is --------------------------------------------------------------------------------------------------

def test_the_sum_wants_no_gradient_of_a_weight():
    """x + residual does not depend on the weight: with the weight the only leaf the sum is a constant, and the next block's norm takes it in
    8 bits; with x or the residual a leaf it is none."""
    import mflux_amd
    from mflux_amd import nn

    norm = nn.RMSNorm(64, 1e-6, device="cuda", dtype=F32)
    x, h, dy = randn(1, 5, 64), randn(2, 5, 64), randn(3, 5, 64)
    y, s = norm(x, residual=h)
    assert y.requires_grad and not s.requires_grad and s.grad_fn is None
    want = ref.rms_norm(ref.total(x, h), norm.weight, 1e-6, dy)
    ref.check("dw", torch.autograd.grad(y, norm.weight, dy)[0], *want["dw"])
    q, sc, total = norm.int8(x, residual=s)
    assert torch.equal(total, s + x) and not total.requires_grad
    for leaf in ("x", "h"):
        x1, h1 = (t.clone().requires_grad_(n == leaf) for n, t in (("x", x), ("h", h)))
        y, s = mflux_amd.rms_norm(x1, norm.weight, residual=h1)
        assert y.requires_grad and s.requires_grad
        d, = torch.autograd.grad(s, x1 if leaf == "x" else h1, dy)
        assert torch.equal(d, dy)
