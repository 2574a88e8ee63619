"""rms_norm, rms_norm_int8, int8_quantize, int8_dequantize and int8_matmul against float64, element by element within the
bounds that int8_reference derives, at the sizes, strides, types and values where they can go wrong."""
import math

import pytest
import torch

import int8_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]


def randn(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def codes(seed, *shape, low=-128):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(low, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def scales(seed, *shape):
    return randn(seed, *shape).abs() * 0.02 + 0.001


# ---- norm ------------------------------------------------------------------------------------------------------------------
# one value; below, at and behind a lane's, a wavefront's, a workgroup's pieces; odd; longer than the registers
ROWS = [(1, 1), (3, 8), (5, 17), (1, 64), (7, 513), (2, 512), (300, 520), (65, 768), (9, 2048), (4, 2056), (3, 3840), (1030, 1024), (2, 8192),
        (3, 16384), (2, 16392), (2, 40001)]


@pytest.mark.parametrize("rows,K", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted,added", [(True, True), (False, False), (True, False), (False, True)])
def test_rms_norm(rows, K, dtype, weighted, added):
    import mflux_amd

    print(f"rows={rows} K={K} {dtype} {weighted} {added}", flush=True)
    x = randn(1, rows, K, dtype=dtype, std=1.5).requires_grad_()
    r = randn(2, rows, K, dtype=dtype, std=0.7).requires_grad_() if added else None
    w = randn(3, K, dtype=dtype).requires_grad_() if weighted else None
    out = mflux_amd.rms_norm(x, w, residual=r)
    out = list(out) if added else [out]
    s = ref.total(x.detach(), None if r is None else r.detach())
    dy, dsum = randn(4, rows, K, dtype=dtype), randn(5, rows, K, dtype=dtype) if added else None
    leaves = [t for t in (x, r, w) if t is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad(out, leaves, [dy, dsum][:len(out)])))
    want = ref.rms_norm(s, w, 1e-6, dy, dsum)
    ref.check("y", out[0], *want["y"])
    if added:
        assert torch.equal(out[1], s)
        assert torch.equal(got[id(r)], got[id(x)])
    ref.check("dx", got[id(x)], *want["dx"])
    if weighted:
        ref.check("dw", got[id(w)], *want["dw"])
    with torch.no_grad():  # without gradients: the same call, the same bits
        again = mflux_amd.rms_norm(x, w, residual=r)
    assert all(torch.equal(a, b) for a, b in zip(again if added else [again], out))


@pytest.mark.parametrize("rows,K", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted,added", [(True, True), (False, False)])
def test_rms_norm_int8(rows, K, dtype, weighted, added):
    import mflux_amd

    print(f"rows={rows} K={K} {dtype} {weighted} {added}", flush=True)
    x, r = randn(1, rows, K, dtype=dtype, std=1.5), randn(2, rows, K, dtype=dtype, std=0.7) if added else None
    w = randn(3, K, dtype=dtype) if weighted else None
    q, sc, *rest = mflux_amd.rms_norm_int8(x, w, residual=r)
    s = ref.total(x, r)
    want_q, want_sc = ref.codes(s, w, 1e-6)
    assert q.dtype == torch.int8 and q.shape == x.shape and sc.dtype == F32 and sc.shape == (rows,)
    assert torch.equal(q.double(), want_q)
    ref.check("scales", sc, want_sc, want_sc * ref.scale_bound(K, True))
    if added:
        assert torch.equal(rest[0], s)
    q2, sc2 = mflux_amd.int8_quantize(s)
    want_q, want_sc = ref.codes(s)
    assert torch.equal(q2.double(), want_q)
    ref.check("scales", sc2, want_sc, want_sc * ref.scale_bound(K, False))
    for out in TYPES:
        back = mflux_amd.int8_dequantize(q2, sc2, out)
        value = q2.double() * sc2.double()[:, None]
        ref.check("values", back, value, value.abs() * (ref.HALF[out] + 2 * ref.E) + ref.TINY[out])


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_next_to_a_border(dtype):
    """Rows whose quotients lie on a border between two codes, or one step of the type beside it."""
    import mflux_amd

    top = torch.tensor([127.0, 1.0, 254.0, 0.3, 100.0, 3.0], device="cuda").to(dtype)
    half = torch.arange(-126, 127, device="cuda").double() + 0.5
    on = (half[None, :-1] * top.double()[:, None] / 127).to(dtype)
    bits = on.view(torch.int32 if dtype == F32 else torch.int16)
    rows = torch.cat([top[:, None], on, (bits + 1).view(dtype), (bits - 1).view(dtype)], dim=1)
    for t in (rows, rows[:, :760], rows[:, :1]):  # 16-byte pieces, and one by one
        q, _ = mflux_amd.int8_quantize(t)
        assert torch.equal(q.double(), ref.codes(t)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [64, 67, 2048])
def test_rows_of_zeros_infinities_and_extremes(dtype, K):
    import mflux_amd

    info = torch.finfo(dtype)
    rows = randn(1, 8, K, dtype=dtype)
    rows[1] = 0
    rows[2, 5], rows[3, 5], rows[4, 5] = math.inf, -math.inf, math.nan
    rows[5] = torch.where(rows[5] > 0, info.max, info.min).to(dtype)
    rows[6] = rows[6] * info.tiny  # and below it
    rows[7] = 0
    rows[7, K - 1] = info.smallest_normal
    q, sc = mflux_amd.int8_quantize(rows)
    fine = [0, 1, 5, 6, 7]
    want_q, want_sc = ref.codes(rows[fine])
    assert torch.equal(q[fine].double(), want_q)
    assert bool(((sc[fine].double() - want_sc).abs() <= want_sc * 2 * ref.E + 2.0 ** -149).all())
    assert bool(sc[2:5].isnan().all()) and not q[2:5].any()
    q, sc = mflux_amd.rms_norm_int8(rows, torch.ones(K, device="cuda", dtype=dtype))
    assert bool(sc[2:5].isnan().all()) and not q[2:5].any() and float(sc[1]) == 0
    y = mflux_amd.rms_norm(rows)
    assert bool(y[4].isnan().all()) and not y[1].any() and bool(y[2, 5].isnan())
    ref.check("y", y[[0, 1, 7]], *ref.rms_norm(rows[[0, 1, 7]], None, 1e-6)["y"])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_strides_and_shapes(dtype):
    """Slices of a stacked product, transposed and expanded rows, odd addresses, leading axes, no rows."""
    import mflux_amd

    big = randn(1, 2, 9, 3 * 256 + 8, dtype=dtype)
    w = randn(2, 256, dtype=dtype)
    flat = torch.empty(10 * 256 + 3, device="cuda", dtype=dtype)
    flat.copy_(randn(3, 10 * 256 + 3))
    cases = [big[:, :, 256:512], big[:, :, 3:259], big.transpose(0, 1)[:, :, :256], big[:, :1, :256].expand(2, 9, 256), big[0, 0, :256],
             flat[3:3 + 2560].view(10, 256), big[:, :, ::3][:, :, :256], big[:0, :, :256]]
    for t in cases:
        x = t.detach().requires_grad_()
        y, s = mflux_amd.rms_norm(x, w, residual=t)
        want = ref.rms_norm(ref.total(t, t), w, 1e-6, torch.ones_like(t), torch.ones_like(t))
        ref.check("y", y, *want["y"])
        assert y.is_contiguous() and y.shape == t.shape and torch.equal(s, ref.total(t, t))
        one = torch.ones((), device="cuda", dtype=dtype).expand(t.shape)
        ref.check("dx", torch.autograd.grad((y, s), x, (one, one))[0], *want["dx"])
        q, sc = mflux_amd.int8_quantize(t)
        assert torch.equal(q.double(), ref.codes(t)[0]) and sc.shape == t.shape[:-1]
        assert torch.equal(mflux_amd.int8_dequantize(q, sc, F32), q.float() * sc[..., None])


def test_norm_partial_gradients():
    """One of the two results, one of the inputs, the same tensor twice; a second derivative is refused."""
    import mflux_amd

    x, r, w = randn(1, 5, 264).requires_grad_(), randn(2, 5, 264).requires_grad_(), randn(3, 264).requires_grad_()
    dy = randn(4, 5, 264)
    want = ref.rms_norm(ref.total(x.detach(), r.detach()), w, 1e-6, dy, None)
    y, s = mflux_amd.rms_norm(x, w, residual=r)
    ref.check("dx", torch.autograd.grad(y, x, dy, retain_graph=True)[0], *want["dx"])
    ref.check("dw", torch.autograd.grad(y, w, dy, retain_graph=True)[0], *want["dw"])
    assert torch.equal(torch.autograd.grad(s, r, dy, retain_graph=True)[0], dy)
    dw, = torch.autograd.grad(s, w, dy, retain_graph=True)
    assert not dw.any()
    y2, _ = mflux_amd.rms_norm(x.detach(), w, residual=r.detach())
    ref.check("dw", torch.autograd.grad(y2, w, dy)[0], *want["dw"])
    y2, _ = mflux_amd.rms_norm(x.detach(), w.detach(), residual=r)
    ref.check("dr", torch.autograd.grad(y2, r, dy)[0], *want["dx"])
    y, s = mflux_amd.rms_norm(x, w, residual=x)
    want = ref.rms_norm(ref.total(x.detach(), x.detach()), w, 1e-6, dy, dy)
    value, bound = want["dx"]
    ref.check("dx", torch.autograd.grad((y, s), x, (dy, dy))[0], 2 * value, 2 * bound)
    g, = torch.autograd.grad(mflux_amd.rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative|differentiate twice"):
        g.sum().backward()
    # .grad of both leaves, which share one gradient, stay apart
    x, r = randn(1, 4, 64).requires_grad_(), randn(2, 4, 64).requires_grad_()
    mflux_amd.rms_norm(x, residual=r)[0].sum().backward()
    before = r.grad.clone()
    x.grad.add_(1)
    assert torch.equal(r.grad, before)


def test_norm_gradient_against_differences():
    import mflux_amd

    x, w, dy = randn(1, 3, 40), randn(2, 40), randn(3, 3, 40)
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(mflux_amd.rms_norm(leaf, w), leaf, dy)
    step = 2.0 ** -10
    for i in range(0, 120, 7):
        d = torch.zeros(120, device="cuda", dtype=torch.float64)
        d[i] = step
        d = d.view(3, 40)
        slope = (along(x.double() + d, w, dy) - along(x.double() - d, w, dy)) / (2 * step)
        # the third derivative of a normalised row of this size is some tens: step^2 / 6 of that
        assert abs(float(got.reshape(-1)[i]) - float(slope)) < 1e-4 * (1 + abs(float(slope)))


def along(v, w, dy):
    return (v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double() * dy.double()).sum()


# ---- product ---------------------------------------------------------------------------------------------------------------
PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 17, 100), (3, 40, 128), (8, 129, 144), (9, 16, 4096), (16, 1000, 1040), (5, 3840, 3840), (17, 64, 64),
            (17, 1, 2048), (32, 300, 272), (33, 127, 4112), (64, 512, 1000), (65, 129, 129), (128, 128, 112), (200, 1023, 640), (333, 1152, 2500),
            (130, 8, 16384), (257, 5000, 16), (3300, 3900, 272), (3329, 4001, 131), (4100, 12300, 128)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("dtype,biased", [(BF16, True), (F16, False), (F32, True), (F32, False)])
def test_int8_matmul(M, N, K, dtype, biased):
    import mflux_amd

    print(f"M={M} N={N} K={K} {dtype} {biased}", flush=True)
    x, w = codes(1, M, K), codes(2, N, K)
    x[0], w[N - 1] = -128, -128  # the largest sum there is
    xs, ws = scales(3, M), scales(4, N)
    b = randn(5, N, dtype=dtype) if biased else None
    y = mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype)
    assert y.dtype == dtype and y.is_contiguous()
    ref.check("y", y, *ref.product(x, xs, w, ws, b, dtype))
    if dtype == F32 and not biased:  # the integers themselves
        one = torch.ones_like
        sums = mflux_amd.int8_matmul(x, one(xs), w, one(ws), dtype=F32)
        assert torch.equal(sums, torch.mm(x.double(), w.double().t().contiguous()).float())


def test_int8_matmul_of_the_longest_rows():
    import mflux_amd

    K = (1 << 17) - 16
    for M, N in ((1, 20), (40, 70), (130, 140)):
        x, w = torch.full((M, K), -128, device="cuda", dtype=torch.int8), torch.full((N, K), -128, device="cuda", dtype=torch.int8)
        one = torch.ones(max(M, N), device="cuda")
        y = mflux_amd.int8_matmul(x, one[:M], w, one[:N], dtype=F32)
        assert bool((y == float(K * 16384)).all())


@pytest.mark.parametrize("M", [1, 12, 30, 60, 140])
def test_int8_matmul_strides(M):
    """Rows apart, of odd lengths and addresses, repeated, transposed; leading axes; codes that int8_quantize laid out."""
    import mflux_amd

    N, K = 200, 160
    big_x, big_w = codes(1, M, 2 * K + 5), codes(2, N, 2 * K + 5)
    xs, ws = scales(3, M), scales(4, N)
    for x, w in ((big_x[:, :K], big_w[:, :K]), (big_x[:, 1:1 + K], big_w[:, 16:16 + K]), (big_x[:1, :K].expand(M, K), big_w[:1, :K].expand(N, K)),
                 (codes(5, K, M).t(), codes(6, K, N).t()), (big_x[:, ::2][:, :K], big_w[:, ::2][:, :K]), (big_x[:, :77], big_w[:, :77])):
        y = mflux_amd.int8_matmul(x, xs, w, ws, dtype=F32)
        ref.check("y", y, *ref.product(x, xs, w, ws, None, F32))
    x = codes(7, 2, 3, M, K)
    y = mflux_amd.int8_matmul(x, scales(8, 2, 3, M), big_w[:, :K], ws)
    ref.check("y", y, *ref.product(x, scales(8, 2, 3, M), big_w[:, :K], ws, None, BF16))
    for odd in (1, 15, 17, 100, 1001):
        q, s = mflux_amd.int8_quantize(randn(9, 2, M, odd))
        p, t = mflux_amd.int8_quantize(randn(10, N, odd))
        ref.check("y", mflux_amd.int8_matmul(q, s, p, t, dtype=F32), *ref.product(q, s, p, t, None, F32))
    assert mflux_amd.int8_matmul(x[:, :0], scales(8, 2, 3, M)[:, :0], big_w[:, :K], ws).shape == (2, 0, M, N)
    assert mflux_amd.int8_matmul(x, scales(8, 2, 3, M), big_w[:0, :K], ws[:0]).shape == (2, 3, M, 0)


def test_int8_matmul_scales_that_are_not_finite():
    """The scale of a row that held an infinity makes its products NaN, and no others."""
    import mflux_amd

    for M in (4, 40, 140):
        x = randn(1, M, 256)
        x[2, 7] = math.inf
        q, s = mflux_amd.int8_quantize(x)
        w, t = mflux_amd.int8_quantize(randn(2, 64, 256))
        y = mflux_amd.int8_matmul(q, s, w, t)
        assert bool(y[2].isnan().all()) and not bool(y[[0, 1, 3]].isnan().any())


def plan(M, N, K, dtype=0):
    import ctypes

    from mflux_amd import _lib

    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("shapes are chosen for 256 compute units")
    ranges, rows, columns = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    kernel = _lib.load().mfq_int8_matmul_plan(M, N, K, dtype, ctypes.byref(ranges), ctypes.byref(rows), ctypes.byref(columns))
    return kernel, rows.value, columns.value, ranges.value > 1


@pytest.mark.parametrize("M,N,K,want", [
    (3, 3840, 3840, (1, 8, 8, False)), (16, 2056, 1040, (1, 16, 8, False)), (1, 40, 131056, (2, 32, 64, True)), (30, 10000, 3840, (2, 32, 64, False)),
    (24, 600, 8208, (2, 32, 64, True)), (60, 3840, 3856, (2, 64, 64, True)), (200, 3840, 3856, (2, 64, 64, False)), (500, 3850, 1040, (2, 64, 128, False)),
    (1000, 3840, 1152, (2, 128, 128, False)), (2048, 3840, 1040, (2, 128, 128, False)), (130, 1000, 16400, (2, 64, 128, True)),
    (200, 3840, 8208, (2, 128, 128, True)), (333, 3840, 8208, (2, 128, 192, True)),
    (500, 10240, 656, (2, 128, 192, False)), (4352, 3840, 1168, (2, 256, 256, False)), (4352, 12300, 272, (2, 256, 256, False)),
])
def test_int8_matmul_on_every_kernel(M, N, K, want):
    """Each tile, with and without a cut K, against the integers: the last tile of either axis partly empty, K no whole step."""
    import mflux_amd

    print(f"M={M} N={N} K={K}", flush=True)
    assert plan(M, N, K, 2) == want
    x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
    for dtype in (BF16, F16):
        b = randn(5, N, dtype=dtype)
        y = mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype)
        ref.check("y", y, *ref.product(x, xs, w, ws, b, dtype))
        assert torch.equal(y, mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype))


@pytest.mark.parametrize("M,N,K,first", [(2000, 10250, 1040, 8192), (2000, 10240, 1152, 8192), (2000, 10251, 1040, 8192)])
def test_int8_matmul_of_columns_in_two_launches(M, N, K, first):
    """Where the largest tiles would leave a last round mostly idle: the same bits as of each columns' own product, to the last column."""
    import mflux_amd

    print(f"M={M} N={N} K={K}", flush=True)
    assert plan(M, N, K, 2) == (2, 256, 256, False)
    x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
    for dtype in (BF16, F16):
        b = randn(5, N, dtype=dtype)
        y = mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype)
        ref.check("y", y, *ref.product(x, xs, w, ws, b, dtype))
        for part in (slice(0, first), slice(first, N)):
            assert torch.equal(y[:, part], mflux_amd.int8_matmul(x, xs, w[part], ws[part], bias=b[part], dtype=dtype))
        assert torch.equal(mflux_amd.int8_matmul(x, xs, w, ws, dtype=dtype), mflux_amd.int8_matmul(x, xs, w, ws, bias=torch.zeros_like(b), dtype=dtype))


def test_rows_behind_others_are_left_alone():
    """A call writes its own results: what lies in front of and behind them in memory stays."""
    from mflux_amd import _lib

    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for M, N, K in ((3, 24, 64), (30, 72, 256), (140, 136, 256), (3300, 3864, 128)):
        x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
        room = torch.full((M + 4, N), 7.0, device="cuda", dtype=BF16)
        need = lib.mfq_int8_matmul_workspace_bytes(M, N, K, _lib.BF16)
        work = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
        y = room[2:2 + M]
        _lib.check("mfq_int8_matmul", lib.mfq_int8_matmul(x.data_ptr(), K, xs.data_ptr(), w.data_ptr(), K, ws.data_ptr(), None, M, N, K, y.data_ptr(),
                                                          _lib.BF16, work.data_ptr(), need, stream))
        ref.check("y", y, *ref.product(x, xs, w, ws, None, BF16))
        assert bool((room[:2] == 7).all()) and bool((room[2 + M:] == 7).all())


# ---- streams, graphs, layers -----------------------------------------------------------------------------------------------

def chain(x, h, norm, up, down):
    """A feed-forward in 8 bits: the residual's addition and the norm, gate and up, down."""
    import mflux_amd

    q, s, h = norm.int8(x, residual=h)
    gate, value = up((q, s)).chunk(2, dim=-1)
    return down(torch.nn.functional.silu(gate) * value), h


def layers(K=512, inner=768, dtype=BF16):
    from mflux_amd import nn

    norm = nn.RMSNorm(K, 1e-6, device="cuda", dtype=dtype)
    up, down = nn.Linear(K, 2 * inner, bias=False, device="cuda", dtype=dtype), nn.Linear(inner, K, bias=True, device="cuda", dtype=dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + randn(11, K) * 0.1)
        up.weight.copy_(randn(12, 2 * inner, K) * 0.05)
        down.weight.copy_(randn(13, K, inner) * 0.05)
        down.bias.copy_(randn(14, K))
    return norm, up, down


@pytest.mark.parametrize("tokens", [1, 77, 600])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layers_together(tokens, dtype):
    """Every layer against float64 on what it was given, and the whole near the float layers."""
    norm, up, down = layers(dtype=dtype)
    up8, down8 = up.to_int8(), down.to_int8()
    x, h = randn(1, 2, tokens, 512, dtype=dtype), randn(2, 2, tokens, 512, dtype=dtype)
    with torch.no_grad():
        y, total = chain(x, h, norm, up8, down8)
        assert torch.equal(total, ref.total(x, h))
        q, s, _ = norm.int8(x, residual=h)
        want_q, want_s = ref.codes(total, norm.weight, 1e-6)
        assert torch.equal(q.double(), want_q)
        ref.check("scales", s, want_s, want_s * ref.scale_bound(512, True))
        u = up8((q, s))
        assert u.dtype == dtype
        ref.check("up", u, *ref.product(q, s, up8.weight, up8.scales, None, dtype))
        gate, value = u.chunk(2, dim=-1)
        a = torch.nn.functional.silu(gate) * value
        qa, sa = (t.float() for t in ref.codes(a))
        ref.check("down", down8(a), *ref.product(qa.to(torch.int8), (ref.codes(a)[1]).float(), down8.weight, down8.scales, down8.bias, dtype))
        assert torch.equal(down8(a), y)
        exact, _ = norm(x, residual=h)
        gate, value = up(exact).chunk(2, dim=-1)
        exact = down(torch.nn.functional.silu(gate) * value)
    # rounding to 8 bits: a step is at most max|row| / 127, some 1/35 of a row's root mean square at these lengths, off by its root
    # mean square of 0.29; four such operands (two rows, two weights) on the way to y, whose bias has no such error
    assert float((y - exact).float().norm() / exact.float().norm()) < 0.29 / 35 * 4
    assert up8((q[:, :0], s[:, :0])).shape == (2, 0, 1536)


def test_layers_refuse_gradients_and_load():
    import mflux_amd
    from mflux_amd import nn

    norm, up, _ = layers()
    up8 = up.to_int8()
    x = randn(1, 3, 512, dtype=BF16).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        up8(x)
    with pytest.raises(ValueError, match="no gradient"):
        norm.int8(x)
    other = nn.Int8Linear(512, 1536, bias=False, device="cuda")
    other.load_state_dict(up8.state_dict())
    assert torch.equal(other(x.detach()), up8(x.detach()))
    odd = torch.nn.Linear(77, 40, device="cuda", dtype=F32)
    odd8 = nn.Int8Linear.from_linear(odd)
    fresh = nn.Int8Linear(77, 40, device="cuda", dtype=F32)
    fresh.load_state_dict(odd8.state_dict())
    t = randn(2, 5, 77)
    assert torch.equal(fresh(t), odd8(t))
    q, s = mflux_amd.int8_quantize(t)
    ref.check("y", odd8(t), *ref.product(q, s, odd8.weight, odd8.scales, odd8.bias.detach(), F32))
    # trained through the norm
    leaf = randn(3, 3, 512, dtype=BF16).requires_grad_()
    y, h = norm(leaf, residual=x)
    (y.float().sum() + h.float().sum()).backward()
    assert leaf.grad.shape == leaf.shape and norm.weight.grad.shape == (512,) and torch.equal(leaf.grad, x.grad)


def test_int8_other_stream():
    norm, up, down = layers()
    up8, down8 = up.to_int8(), down.to_int8()
    x, h = randn(1, 40, 512, dtype=BF16), randn(2, 40, 512, dtype=BF16)
    want = chain(x, h, norm, up8, down8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = chain(x, h, norm, up8, down8)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_int8_captured_and_replayed():
    """Two graphs (a chain of layers whose products cut K, a training step of the norm) and eager calls in between."""
    import mflux_amd

    norm, up, down = layers(K=2048, inner=8192)
    up8, down8 = up.to_int8(), down.to_int8()
    assert plan(40, 2048, 8192, 2)[3]  # down's K is cut: planes, and a second kernel
    x, h = randn(1, 40, 2048, dtype=BF16), randn(2, 40, 2048, dtype=BF16)
    t, w = randn(3, 300, 264).requires_grad_(), randn(4, 264).requires_grad_()
    dy, dh = randn(5, 300, 264), randn(6, 300, 264)

    def step():
        y, s = mflux_amd.rms_norm(t, w, residual=dh)
        return (y, s, *torch.autograd.grad((y, s), (t, w), (dy, dh)))

    def work():
        with torch.no_grad():
            return chain(x, h, norm, up8, down8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), work()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs = [], []
    for f in (step, work):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs.append(f())
        graphs.append(g)
    for i in range(4):
        with torch.no_grad():
            t.copy_(randn(20 + i, 300, 264))
            x.copy_(randn(30 + i, 40, 2048, dtype=BF16))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs[0], step()))
        assert all(torch.equal(a, b) for a, b in zip(outputs[1], work()))


def test_norm_capture_next_to_a_living_graph_is_refused():
    """An eager result of the same leaf on the default stream: its nodes would end the process when the captured backward pass
    reaches them.  Refused before anything is captured; without it the same capture works."""
    import mflux_amd

    t = randn(1, 20, 64).requires_grad_()
    ones = torch.ones_like(t)
    want = torch.autograd.grad(mflux_amd.rms_norm(t), t, ones)[0]
    held = mflux_amd.rms_norm(t)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="graph is being captured"):
        with torch.cuda.graph(graph):
            mflux_amd.rms_norm(t)
    torch.cuda.synchronize()
    del held, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(mflux_amd.rms_norm(t), t, ones)[0]
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_int8_no_forward_mode():
    """A tangent is refused, not dropped."""
    import mflux_amd
    from torch.autograd import forward_ad

    x, w, q = randn(1, 3, 64), randn(2, 64), codes(3, 3, 64)
    s = scales(4, 3)
    calls = [((x, w, x.clone()), lambda x, w, r: mflux_amd.rms_norm(x, w, residual=r)[0]),
             ((x, w, x.clone()), lambda x, w, r: mflux_amd.rms_norm_int8(x, w, residual=r)[1]),
             ((x,), lambda x: mflux_amd.int8_quantize(x)[1]), ((s,), lambda s: mflux_amd.int8_dequantize(q, s, F32)),
             ((s, s.clone(), randn(5, 3)), lambda a, b, c: mflux_amd.int8_matmul(q, a, q, b, bias=c, dtype=F32))]
    for operands, call in calls:
        for i, t in enumerate(operands):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward mode"):
                    call(*operands[:i], dual, *operands[i + 1:])
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                    call(*operands[:i], dual, *operands[i + 1:])
                assert torch.equal(call(*operands), call(*operands))


def test_int8_routes_agree():
    """The ops, the C functions that the ordinary call takes, and the C ABI give the same bits."""
    import ctypes

    from mflux_amd import _lib

    lib, ops, native, stream = _lib.load(), _lib.ops(), _lib.native(), torch.cuda.current_stream().cuda_stream
    x, r, w = randn(1, 2, 9, 256, dtype=BF16), randn(2, 2, 9, 256, dtype=BF16), randn(3, 256, dtype=BF16)
    y, s = ops.rms_norm(x, w, r, 1e-6)
    got = native.rms_norm(x, w, r, 1e-6)
    assert torch.equal(got[0], y) and torch.equal(got[1], s)
    a = _lib.RmsNormArgs(dtype=_lib.BF16, eps=1e-6, rows=18, columns=256, x=x.data_ptr(), residual=r.data_ptr(), weight=w.data_ptr(), x_stride=256,
                         residual_stride=256)
    y2, s2 = torch.empty_like(y), torch.empty_like(s)
    a.y, a.sum = y2.data_ptr(), s2.data_ptr()
    _lib.check("mfq_rms_norm", lib.mfq_rms_norm(ctypes.byref(a), stream))
    assert torch.equal(y2, y) and torch.equal(s2, s)
    for norm in (True, False):
        q = ops.rms_norm_int8(x, w, r, 1e-6)[:2] if norm else ops.int8_quantize(x)
        got = native.int8_rows(x, w if norm else None, r if norm else None, 1e-6, norm)
        assert torch.equal(got[0], q[0]) and torch.equal(got[1], q[1])
    p, t = ops.int8_quantize(randn(4, 70, 256, dtype=BF16))
    b = randn(5, 70, dtype=BF16)
    assert torch.equal(native.int8_matmul(*q, p, t, b, _lib.BF16), ops.int8_matmul(*q, p, t, b, BF16))
    # what the C functions leave to the ops
    assert native.rms_norm(x[:, :, 1:], None, None, 1e-6) is None and native.rms_norm(x, w, r, -1.0) is None
    assert native.rms_norm(x.clone().requires_grad_(), w, r, 1e-6) is None and native.int8_rows(x[..., :40], None, None, 0.0, False) is None
    assert native.int8_matmul(q[0].cpu(), q[1], p, t, None, 2) is None and native.int8_matmul(*q, p, t, b, _lib.F16) is None
