"""The norm and the products of 8-bit integers where calls differ from the ordinary one: more elements than 32 bits count, two
threads at once, operands at odd addresses, broadcast and overlapping rows, no rows, eps of zero, copies of a layer."""
import copy
import io
import threading

import pytest
import torch

import int8_reference as ref
from test_gpu_int8 import BF16, F16, F32, codes, plan, randn, scales

pytestmark = pytest.mark.gpu


def room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB")


def repeats(big, small):
    """Whether `big` is `small` again and again, compared a copy at a time."""
    n = big.shape[0] // small.shape[0]
    return all(torch.equal(big[i * small.shape[0]:(i + 1) * small.shape[0]], small) for i in range(n))


def test_norm_of_more_than_32_bits():
    """2^32 elements and some: every row as in a call of the first ones (4099 of them, so that no wrapped offset meets its like)."""
    import mflux_amd

    room(80)
    n, rows, K = 512, 4099, 2048
    assert n * rows * K > 1 << 32
    x, r, w = randn(1, rows, K, dtype=BF16), randn(2, rows, K, dtype=BF16), randn(3, K, dtype=BF16).requires_grad_()
    dy, ds = randn(4, rows, K, dtype=BF16), randn(5, rows, K, dtype=BF16)
    X, R = x.repeat(n, 1), r.repeat(n, 1).requires_grad_()
    print("forward", flush=True)
    y, s = mflux_amd.rms_norm(X, w, residual=R)
    small = mflux_amd.rms_norm(x, w.detach(), residual=r)
    assert repeats(y.detach(), small[0]) and repeats(s.detach(), small[1])
    print("backward", flush=True)
    want = ref.rms_norm(small[1], w.detach(), 1e-6, dy, ds)
    q = r.clone().requires_grad_()
    d_small, = torch.autograd.grad(mflux_amd.rms_norm(x, w.detach(), residual=q), q, (dy, ds))
    d, dw = torch.autograd.grad((y, s), (R, w), (dy.repeat(n, 1), ds.repeat(n, 1)))
    assert repeats(d, d_small)
    # a workgroup adds up 4099 rows or a few more as the oracle's bound has it, then some hundred workgroups meet
    ref.check("dw", dw, n * want["dw"][0], 1.1 * n * want["dw"][1])
    del y, s, d, dw
    print("codes", flush=True)
    c, t = mflux_amd.int8_quantize(X)
    c_small, t_small = mflux_amd.int8_quantize(x)
    assert repeats(c, c_small) and repeats(t, t_small)
    print("values", flush=True)
    assert repeats(mflux_amd.int8_dequantize(c, t), mflux_amd.int8_dequantize(c_small, t_small))


@pytest.mark.parametrize("M", [3, 40, 333])
def test_int8_matmul_of_long_operands(M):
    """w, then x, of more bytes than 32 bits count."""
    import mflux_amd

    room(40)
    n, rows, K = 257, 4099, 4096
    assert n * rows * K > 1 << 32
    a, b, sa, sb = codes(1, rows, K), codes(2, M, K), scales(3, rows), scales(4, M)
    A, SA = a.repeat(n, 1), sa.repeat(n)
    print(f"M={M} long w", flush=True)
    small = mflux_amd.int8_matmul(b, sb, a, sa)
    y = mflux_amd.int8_matmul(b, sb, A, SA)
    assert all(torch.equal(part, small) for part in y.split(rows, 1))
    print(f"N={M} long x", flush=True)
    assert repeats(mflux_amd.int8_matmul(A, SA, b, sb), mflux_amd.int8_matmul(a, sa, b, sb))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_int8_matmul_of_more_than_32_bits_of_results(dtype):
    import mflux_amd

    room(60)
    n, M, N, K = 64, 1031, 1033, 16
    assert n * n * M * N > 1 << 32
    x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
    print(f"{n * M} x {n * N} x {K}", flush=True)
    y = mflux_amd.int8_matmul(x.repeat(n, 1), xs.repeat(n), w.repeat(n, 1), ws.repeat(n), dtype=dtype)
    small = mflux_amd.int8_matmul(x, xs, w, ws, dtype=dtype)
    ref.check("y", small, *ref.product(x, xs, w, ws, None, dtype))
    assert repeats(y, small.repeat(1, n))


def test_int8_in_two_threads():
    """Each on its stream, with products whose K is cut (planes of their own) and the norm's backward pass (partial sums)."""
    import mflux_amd

    assert plan(40, 2048, 8192, 2)[3]
    w, ws = codes(1, 2048, 8192), scales(2, 2048)
    g = randn(3, 264)

    def work(i, out, rounds):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            for _ in range(rounds):
                y = mflux_amd.int8_matmul(xs[i], ss[i], w, ws)
                t, h = ts[i].clone().requires_grad_(), g.clone().requires_grad_()
                out.append((y, *torch.autograd.grad(mflux_amd.rms_norm(t, h).square().sum(), (t, h))))
        stream.synchronize()

    xs, ss, ts = [codes(10 + i, 40, 8192) for i in range(2)], [scales(20 + i, 40) for i in range(2)], [randn(30 + i, 300, 264) for i in range(2)]
    torch.cuda.synchronize()
    want, got = [[], []], [[], []]
    for i in range(2):
        work(i, want[i], 1)
    threads = [threading.Thread(target=work, args=(i, got[i], 20)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(a, b) for one in got[i] for a, b in zip(one, want[i][0]))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M", [2, 40, 200])
def test_int8_matmul_of_vectors_at_odd_addresses(M, dtype):
    """Scales and a bias that begin behind their storage's first element, and ones with a stride."""
    import mflux_amd

    N, K = 210, 4112
    x, w = codes(1, M, K), codes(2, N, K)
    xs, ws, b = scales(3, M), scales(4, N), randn(5, N, dtype=dtype)
    want = mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype)
    ref.check("y", want, *ref.product(x, xs, w, ws, b, dtype))

    def behind(t):
        flat = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
        flat[1:] = t
        return flat[1:]

    def apart(t):
        flat = torch.zeros(t.numel(), 3, device="cuda", dtype=t.dtype)
        flat[:, 1] = t
        return flat[:, 1]

    for how in (behind, apart):
        assert torch.equal(mflux_amd.int8_matmul(x, how(xs), w, how(ws), bias=how(b), dtype=dtype), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_and_codes_of_overlapping_rows(dtype):
    """Windows of a vector, a row for all, and gradients that are one number."""
    import mflux_amd

    flat = randn(1, 1000, dtype=dtype)
    w = randn(2, 256, dtype=dtype)
    for x in (flat.as_strided((20, 256), (8, 1)), flat.as_strided((20, 256), (3, 1)), flat[:256].expand(20, 256), flat.as_strided((4, 5, 256), (80, 16, 1))):
        r = x.detach().requires_grad_()
        g = w.clone().requires_grad_()
        y, s = mflux_amd.rms_norm(x.contiguous(), g, residual=r)
        dy = torch.full((), 0.5, device="cuda", dtype=dtype).expand(y.shape)
        want = ref.rms_norm(ref.total(x, x), w, 1e-6, dy, dy)
        ref.check("y", y, *want["y"])
        dr, dw = torch.autograd.grad((y, s), (r, g), (dy, dy))
        ref.check("dr", dr, *want["dx"])
        ref.check("dw", dw, *want["dw"])
        q, sc = mflux_amd.int8_quantize(x)
        assert torch.equal(q.double(), ref.codes(x)[0])
        c = codes(3, 1000).as_strided(x.shape, x.stride())
        assert torch.equal(mflux_amd.int8_dequantize(c, sc, F32), c.float() * sc[..., None])
        p, ps = codes(4, 50, 256), scales(5, 50)
        ref.check("product", mflux_amd.int8_matmul(c, sc, p, ps), *ref.product(c, sc, p, ps, None, BF16))


def test_int8_of_no_rows():
    import mflux_amd

    x = torch.empty(0, 64, device="cuda", dtype=BF16)
    w = randn(1, 64, dtype=BF16).requires_grad_()
    leaf = x.clone().requires_grad_()
    y, s = mflux_amd.rms_norm(leaf, w, residual=x)
    dx, dw = torch.autograd.grad((y, s), (leaf, w), (x, x))
    assert dx.shape == x.shape and not dw.any()
    q, t, s = mflux_amd.rms_norm_int8(x, w.detach(), residual=x)
    assert q.shape == (0, 64) and t.shape == (0,) and s.shape == (0, 64) and q.dtype == torch.int8 and t.dtype == F32
    q, t = mflux_amd.int8_quantize(torch.empty(3, 0, 77, device="cuda"))
    assert q.shape == (3, 0, 77) and t.shape == (3, 0)
    assert mflux_amd.int8_dequantize(q, t).shape == (3, 0, 77)
    assert mflux_amd.int8_matmul(q, t, codes(2, 5, 77), scales(3, 5)).shape == (3, 0, 5)


def test_norm_with_eps_zero():
    """A row of zeros is then 0 times infinity, in the norm and in the scale; others are what they are."""
    import mflux_amd

    for K in (64, 67, 2048):
        x = randn(1, 5, K)
        x[2] = 0
        y = mflux_amd.rms_norm(x, eps=0.0)
        q, s = mflux_amd.rms_norm_int8(x, eps=0.0)
        assert bool(y[2].isnan().all()) and bool(s[2].isnan()) and not q[2].any()
        rest = x[[0, 1, 3, 4]]
        ref.check("y", y[[0, 1, 3, 4]], *ref.rms_norm(rest, None, 0.0)["y"])
        assert torch.equal(q[[0, 1, 3, 4]].double(), ref.codes(rest)[0])


def test_norm_inputs_changed_before_the_gradient():
    """What the gradient reads again has been written to: an error, not a wrong gradient."""
    import mflux_amd

    x, r, w = randn(1, 5, 64).requires_grad_(), randn(2, 5, 64), randn(3, 64).requires_grad_()
    for change in ("sum", "weight", "x"):
        t = x.clone()
        y, s = mflux_amd.rms_norm(t, w, residual=None if change == "x" else r), None
        if change != "x":
            y, s = y
        with torch.no_grad():
            {"sum": s, "weight": w, "x": t}[change].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
    # the residual's sum of the next block may change what this one's result does not need
    y, s = mflux_amd.rms_norm(x, w, residual=r)
    want = ref.rms_norm(ref.total(x.detach(), r), w, 1e-6, torch.ones_like(r), None)
    with torch.no_grad():
        r.add_(1)
        y.mul_(2)
    ref.check("dx", torch.autograd.grad(y, x, torch.ones_like(r))[0], *want["dx"])


def test_int8_layers_copied_and_moved():
    from mflux_amd import nn

    for K in (512, 77):
        torch.manual_seed(K)
        layer = nn.Linear(K, 40, bias=True, device="cuda", dtype=BF16).to_int8()
        x = randn(2, 6, K, dtype=BF16)
        want = layer(x)
        assert want.dtype == BF16
        for other in (copy.deepcopy(layer), layer.cpu().cuda(), nn.Int8Linear(K, 40).cuda()):
            if other is not layer:
                other.load_state_dict(layer.state_dict())
            assert torch.equal(other(x), want) and other.scales.dtype == F32 and other.weight.dtype == torch.int8
        file = io.BytesIO()
        torch.save(layer.state_dict(), file)
        file.seek(0)
        fresh = nn.Int8Linear(K, 40, device="cuda")
        fresh.load_state_dict(torch.load(file, weights_only=True))
        assert torch.equal(fresh(x), want)
        half = copy.deepcopy(layer).half()
        assert half.scales.dtype == F32 and torch.equal(half.scales, layer.scales) and half.dtype == F16
        assert half(x.half()).dtype == F16


def test_int8_dequantize_routes_agree():
    from mflux_amd import _lib

    native, ops = _lib.native(), _lib.ops()
    for dtype, code in ((BF16, _lib.BF16), (F16, _lib.F16), (F32, _lib.F32)):
        for shape in ((3, 77), (2, 5, 256), (64,), (1, 1)):
            q, s = codes(1, *shape), scales(2, *shape[:-1], 1)[..., 0].contiguous()
            got = native.int8_dequantize(q, s, code)
            assert got.dtype == dtype and torch.equal(got, ops.int8_dequantize(q, s, dtype))
            assert torch.equal(got, (q.float() * s[..., None]).to(dtype))
    q, s = codes(1, 3, 80), scales(2, 3)
    # what the C function leaves to the op, or to the checks
    assert native.int8_dequantize(q[:, 1:], s, _lib.BF16) is None and native.int8_dequantize(q[:0], s[:0], _lib.BF16) is None
    assert native.int8_dequantize(q, s[:2], _lib.BF16) is None and native.int8_dequantize(q, s, None) is None
    assert native.int8_dequantize(q, s.double(), _lib.BF16) is None and native.int8_dequantize(q, s, 7) is None
    assert native.int8_dequantize(q, s.clone().requires_grad_(), _lib.BF16) is None


@pytest.mark.parametrize("M,N,K,want", [
    (17, 40, 1040, (1, 24, 8, False)), (24, 2051, 528, (1, 24, 8, False)), (31, 2048, 1024, (1, 32, 8, False)), (32, 77, 16, (1, 32, 8, False)),
    (33, 512, 2064, (1, 24, 8, False)), (47, 100, 1296, (1, 24, 8, False)), (63, 300, 144, (1, 32, 8, False)), (65, 256, 4096, (1, 24, 8, False)),
    (90, 513, 768, (1, 32, 8, False)), (100, 9, 112, (1, 32, 8, False)), (127, 512, 2048, (1, 32, 8, False)), (128, 1000, 400, (1, 32, 8, False)),
    (24, 3843, 3840, (1, 24, 8, False)), (129, 512, 2048, (2, 32, 64, False)),
])
def test_int8_matmul_of_small_weights(M, N, K, want):
    """17 to 128 rows through the kernel of few rows, in one to four groups, the last token, row of w and step partly there."""
    import mflux_amd

    print(f"M={M} N={N} K={K}", flush=True)
    assert plan(M, N, K, 2) == want
    x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
    for dtype in (BF16, F16, F32):
        b = randn(5, N, dtype=dtype)
        y = mflux_amd.int8_matmul(x, xs, w, ws, bias=b, dtype=dtype)
        ref.check("y", y, *ref.product(x, xs, w, ws, b, dtype))
        # each row as by itself
        for m in (0, M // 2, M - 1):
            assert torch.equal(y[m], mflux_amd.int8_matmul(x[m], xs[m], w, ws, bias=b, dtype=dtype))


@pytest.mark.parametrize("M", [18, 50, 129, 200])
def test_int8_matmul_strides_above_sixteen_rows(M):
    """The same layouts through both kernels: rows apart, at odd addresses, repeated, transposed, of an odd length; nothing behind y is written."""
    import mflux_amd

    N, K = 120, 160
    big_x, big_w = codes(1, M, 2 * K + 5), codes(2, N, 2 * K + 5)
    xs, ws = scales(3, M), scales(4, N)
    for x, w in ((big_x[:, :K], big_w[:, :K]), (big_x[:, 1:1 + K], big_w[:, 16:16 + K]), (big_x[:1, :K].expand(M, K), big_w[:1, :K].expand(N, K)),
                 (codes(5, K, M).t(), codes(6, K, N).t()), (big_x[:, ::2][:, :K], big_w[:, ::2][:, :K]), (big_x[:, :77], big_w[:, :77])):
        y = mflux_amd.int8_matmul(x, xs, w, ws, dtype=F32)
        ref.check("y", y, *ref.product(x, xs, w, ws, None, F32))


@pytest.mark.parametrize("M,N,K", [(20, 70, 256), (50, 70, 256), (100, 9, 256), (129, 70, 256)])
def test_int8_matmul_writes_no_further(M, N, K):
    from mflux_amd import _lib

    lib = _lib.load()
    x, w, xs, ws = codes(1, M, K), codes(2, N, K), scales(3, M), scales(4, N)
    y = torch.full((M * N + 4096,), 7.0, device="cuda")
    _lib.check("mfq_int8_matmul", lib.mfq_int8_matmul(x.data_ptr(), K, xs.data_ptr(), w.data_ptr(), K, ws.data_ptr(), None, M, N, K, y.data_ptr(), _lib.F32,
                                                      None, 0, torch.cuda.current_stream().cuda_stream))
    ref.check("y", y[:M * N].view(M, N), *ref.product(x, xs, w, ws, None, F32))
    assert bool((y[M * N:] == 7).all())
