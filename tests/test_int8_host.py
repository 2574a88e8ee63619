"""The refusals of rms_norm, rms_norm_int8, int8_quantize, int8_dequantize and int8_matmul: worded before a device is
looked for, and at the C ABI an error code before anything is launched.  No GPU."""
import ctypes

import pytest
import torch

import mflux_amd
from mflux_amd import _lib, nn

BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


X, W = z(2, 5, 64), z(64)


@pytest.mark.parametrize("call", [mflux_amd.rms_norm, mflux_amd.rms_norm_int8])
@pytest.mark.parametrize("arguments,keywords,match", [
    ((z(2, 64, dtype=torch.int32),), {}, "float32, float16 or bfloat16"),
    ((z(2, 64, dtype=torch.float64),), {}, "float32, float16 or bfloat16"),
    ((z(2, 0),), {}, "values a row"),
    ((torch.zeros((), dtype=BF16),), {}, "values a row"),
    ((X, z(63)), {}, "weight must be"),
    ((X, z(64, dtype=F32)), {}, "weight must be"),
    ((X, z(1, 64)), {}, "weight must be"),
    ((X, W), {"residual": z(2, 5, 63)}, "residual must be as x"),
    ((X, W), {"residual": z(1, 5, 64)}, "residual must be as x"),
    ((X, W), {"residual": z(2, 5, 64, dtype=F32)}, "residual must be as x"),
    ((X, W), {"eps": -1e-6}, "eps"),
    ((X, W), {"eps": float("nan")}, "eps"),
    ((X, W), {"eps": float("inf")}, "eps"),
])
def test_norm_refusals(call, arguments, keywords, match):
    with pytest.raises(ValueError, match=match):
        call(*arguments, **keywords)


def test_cpu_tensors_and_gradients_are_refused():
    for call in (lambda: mflux_amd.rms_norm(X, W), lambda: mflux_amd.rms_norm_int8(X), lambda: mflux_amd.int8_quantize(X),
                 lambda: mflux_amd.int8_dequantize(z(2, 16, dtype=I8), z(2, dtype=F32)),
                 lambda: mflux_amd.int8_matmul(z(2, 16, dtype=I8), z(2, dtype=F32), z(3, 16, dtype=I8), z(3, dtype=F32))):
        with pytest.raises(RuntimeError, match="HIP device only"):
            call()
    leaf = X.clone().requires_grad_()
    scale = z(2, dtype=F32).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        mflux_amd.int8_quantize(leaf)
    with pytest.raises(ValueError, match="no gradient"):
        mflux_amd.int8_dequantize(z(2, 16, dtype=I8), scale)
    with pytest.raises(ValueError, match="no gradient"):
        mflux_amd.int8_matmul(z(2, 16, dtype=I8), scale, z(3, 16, dtype=I8), z(3, dtype=F32))
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device only"):
        mflux_amd.int8_quantize(leaf)


C, S, V, T = z(2, 5, 32, dtype=I8), z(2, 5, dtype=F32), z(7, 32, dtype=I8), z(7, dtype=F32)


@pytest.mark.parametrize("arguments,keywords,match", [
    ((C.float(), S, V, T), {}, "int8"),
    ((C, S, V.to(torch.uint8), T), {}, "int8"),
    ((C, S[0], V, T), {}, "scales of x"),
    ((C, S.to(BF16), V, T), {}, "scales of x"),
    ((C, S, V, T[:6]), {}, "scales of w"),
    ((C, S, V[None], T[None]), {}, "agree in K"),
    ((C, S, z(7, 31, dtype=I8), T), {}, "agree in K"),
    ((C[..., :0], S, V[:, :0], T), {}, "int8"),
    ((z(1, 1 << 17, dtype=I8), z(1, dtype=F32), z(1, 1 << 17, dtype=I8), z(1, dtype=F32)), {}, "32-bit sum"),
    ((C, S, V, T), {"dtype": torch.float64}, "dtype must be"),
    ((C, S, V, T), {"dtype": torch.int32}, "dtype must be"),
    ((C, S, V, T), {"bias": z(6)}, "bias must be"),
    ((C, S, V, T), {"bias": z(7, dtype=F32)}, "bias must be"),
])
def test_matmul_refusals(arguments, keywords, match):
    with pytest.raises(ValueError, match=match):
        mflux_amd.int8_matmul(*arguments, **keywords)


def test_other_refusals():
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        mflux_amd.int8_quantize(C)
    with pytest.raises(ValueError, match="dtype must be"):
        mflux_amd.int8_dequantize(C, S, torch.int8)
    with pytest.raises(ValueError, match="scales of codes"):
        mflux_amd.int8_dequantize(C, S[:1])
    with pytest.raises(ValueError, match="floating point weight"):
        nn.Int8Linear.from_linear(nn.QuantizedLinear(64, 32))
    with pytest.raises(ValueError, match="no gradient"):
        mflux_amd.lora.LoRALinear.from_linear(nn.Int8Linear(64, 32))


def test_the_layers_tensors():
    layer = nn.Int8Linear(48, 20, dtype=torch.float16)
    assert {k: (tuple(v.shape), v.dtype) for k, v in layer.state_dict().items()} == {
        "weight": ((20, 48), I8), "scales": ((20,), F32), "bias": ((20,), torch.float16)}
    assert layer.input_dims == 48 and layer.output_dims == 20
    layer.bfloat16()
    assert layer.scales.dtype == F32 and layer.bias.dtype == BF16 and layer.dtype == BF16
    layer.float()
    assert layer.scales.dtype == F32 and layer.dtype == F32 and layer.weight.dtype == I8
    assert nn.Int8Linear(48, 20, bias=False).bias is None
    norm = nn.RMSNorm(24, 1e-4, dtype=F32)
    assert list(norm.state_dict()) == ["weight"] and norm.eps == 1e-4 and bool((norm.weight == 1).all())


def test_abi_refusals():
    lib = _lib.load()
    E = {"dtype": -1, "shape": -4, "null": -5, "align": -6, "unsupported": -8, "scratch": -9}
    buf = ctypes.create_string_buffer(4096 + 64)
    base = (ctypes.addressof(buf) + 15) & ~15

    def norm(fn=lib.mfq_rms_norm, **kw):
        a = dict(dtype=_lib.BF16, eps=1e-6, rows=4, columns=64, x=base, y=base, x_stride=64)
        a.update(kw)
        args = _lib.RmsNormArgs(**a)
        return fn(ctypes.byref(args), None) if fn is lib.mfq_rms_norm else fn(ctypes.byref(args), None, 0, None)

    assert lib.mfq_rms_norm(None, None) == E["null"]
    assert norm(dtype=7) == E["dtype"]
    assert norm(rows=0) == E["shape"]
    assert norm(columns=0) == E["shape"]
    assert norm(columns=(1 << 28) + 1) == E["shape"]
    assert norm(rows=1 << 31) == E["shape"]
    assert norm(eps=-1.0) == E["shape"]
    assert norm(eps=float("nan")) == E["shape"]
    assert norm(x=None) == E["null"]
    assert norm(y=None) == E["null"]
    assert norm(x_stride=-64) == E["shape"]
    assert norm(residual=base, residual_stride=64) == E["null"]  # and nowhere to write the sum
    assert norm(codes=base, scales=base, code_stride=64) == E["unsupported"]  # codes or y
    assert norm(codes=base, y=None, code_stride=64) == E["null"]
    assert norm(codes=base, scales=base, y=None, code_stride=63) == E["shape"]
    back = lib.mfq_rms_norm_backward
    assert norm(back) == E["null"]
    assert norm(back, dy=base, dy_stride=64) == E["null"]  # no result wanted
    assert norm(back, dy=base, dy_stride=64, dweight=base) == E["null"]  # of no weight
    assert norm(back, dy=base, dy_stride=64, dx=base, dsum=base, dsum_stride=-1) == E["shape"]
    full = dict(dy=base, dy_stride=64, dx=base, weight=base, dweight=base)
    assert norm(back, **full) == E["null"]  # its workspace
    args = _lib.RmsNormArgs(dtype=_lib.BF16, eps=1e-6, rows=4, columns=64, x=base, x_stride=64, **full)
    need = lib.mfq_rms_norm_workspace_bytes(ctypes.byref(args))
    assert need >= 4 * 64
    assert back(ctypes.byref(args), base, need - 1, None) == E["scratch"]
    assert back(ctypes.byref(args), base + 4, need, None) == E["align"]

    q = lib.mfq_int8_quantize
    assert q(base, 9, 4, 64, 64, base, 64, base, None) == E["dtype"]
    assert q(base, 0, 0, 64, 64, base, 64, base, None) == E["shape"]
    assert q(base, 0, 4, 64, 64, None, 64, base, None) == E["null"]
    assert q(base, 0, 4, 64, 64, base, 64, None, None) == E["null"]
    assert q(base, 0, 4, 64, 64, base, 60, base, None) == E["shape"]
    d = lib.mfq_int8_dequantize
    assert d(base, 64, base, 4, 64, base, 9, None) == E["dtype"]
    assert d(base, 64, base, 4, 0, base, 0, None) == E["shape"]
    assert d(base, -64, base, 4, 64, base, 0, None) == E["shape"]
    assert d(base, 64, None, 4, 64, base, 0, None) == E["null"]

    def product(x=base, xs=64, x_scales=base, w=base, ws=64, w_scales=base, bias=None, M=4, N=8, K=64, y=base, dtype=0, work=None, size=0):
        return lib.mfq_int8_matmul(x, xs, x_scales, w, ws, w_scales, bias, M, N, K, y, dtype, work, size, None)

    assert product(dtype=5) == E["dtype"]
    for name in ("M", "N", "K"):
        assert product(**{name: 0}) == E["shape"]
    assert product(K=40) == E["shape"]
    assert product(K=1 << 17, xs=1 << 17, ws=1 << 17) == E["shape"]
    assert product(M=1 << 30, N=1 << 30) == E["shape"]
    assert product(xs=-64) == E["shape"] and product(ws=1 << 20) == E["shape"]
    assert product(xs=72) == E["align"] and product(w=base + 8) == E["align"] and product(y=base + 4) == E["align"]
    for name in ("x", "x_scales", "w", "w_scales", "y"):
        assert product(**{name: None}) == E["null"]
    ranges = ctypes.c_int()
    assert lib.mfq_int8_matmul_plan(24, 512, 8192, 0, ctypes.byref(ranges), None, None) == _lib.INT8_TILES and ranges.value > 1
    need = lib.mfq_int8_matmul_workspace_bytes(24, 512, 8192, 0)
    assert need == ranges.value * 24 * 512 * 4
    cut = dict(M=24, N=512, K=8192, xs=8192, ws=8192)
    assert product(**cut) == E["null"]
    assert product(**cut, work=base, size=need - 1) == E["scratch"]
    assert product(**cut, work=base + 4, size=need) == E["align"]
    assert lib.mfq_int8_matmul_plan(24, 512, 8192, 9, None, None, None) == E["dtype"]
    assert lib.mfq_int8_matmul_plan(24, 512, 8190, 0, None, None, None) == E["shape"]
    assert lib.mfq_int8_matmul_workspace_bytes(24, 512, 8190, 0) == 0


def test_every_size_has_a_plan():
    """Of any number of rows, columns and steps, within what a launch and the LDS take."""
    lib = _lib.load()
    seen = set()
    for M in (1, 2, 8, 9, 16, 17, 33, 64, 65, 129, 333, 1000, 4352, 1 << 20, 1 << 30):
        for N in (1, 7, 64, 65, 3840, 20480):
            if M * N > 1 << 42:
                continue
            for K in (16, 64, 112, 128, 144, 512, 3840, 10240, (1 << 17) - 16):
                for dtype in (_lib.F32, _lib.F16, _lib.BF16):
                    ranges, rows, columns = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
                    kernel = lib.mfq_int8_matmul_plan(M, N, K, dtype, ctypes.byref(ranges), ctypes.byref(rows), ctypes.byref(columns))
                    assert kernel in (_lib.INT8_FEW, _lib.INT8_TILES) and 1 <= ranges.value <= max(1, -(-K // 128) // 4)
                    assert kernel == _lib.INT8_TILES or (M <= 128 and ranges.value == 1 and rows.value * -(-M // 32) >= M)
                    seen.add((kernel, rows.value, columns.value))
    assert seen >= {(1, 8, 8), (1, 16, 8), (1, 24, 8), (1, 32, 8), (2, 32, 64), (2, 64, 64), (2, 64, 128), (2, 128, 128), (2, 128, 192), (2, 256, 256)}


def test_listings_with_scratch_or_fresh_bases_are_refused():
    from mflux_amd import _build

    def listing(*body):
        return "kernel_x:\n" + "\n".join("\t" + s for s in body) + "\n.Lfunc_end0:\n"

    load = "global_load_lds_dwordx4 v1, s[4:5]"
    assert _build.check_no_scratch(listing("v_readlane_b32 s4, v0, 1", "s_nop 4", load, "s_endpgm"), "kernel_x") == 1
    with pytest.raises(RuntimeError, match="just written"):
        _build.check_no_scratch(listing("v_readlane_b32 s5, v0, 1", "s_nop 2", load, "s_endpgm"), "kernel_x")
    with pytest.raises(RuntimeError, match="just written"):
        _build.check_no_scratch(listing("v_cmp_gt_u32_e64 s[4:5], v0, v1", load, "s_endpgm"), "kernel_x")
    with pytest.raises(RuntimeError, match="scratch memory"):
        _build.check_no_scratch(listing("scratch_load_dword v1, off, off", load, "s_endpgm"), "kernel_x")
    with pytest.raises(RuntimeError, match="no load into LDS"):
        _build.check_no_scratch(listing("s_endpgm"), "kernel_x")
