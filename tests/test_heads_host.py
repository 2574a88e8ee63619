"""The refusals of rotary_tables, rotary and attention: worded before a device is
looked for, and at the C ABI an error code before anything is launched.  No GPU."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import mflux_amd
from mflux_amd import _lib

BF16 = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("arguments,keywords,match", [
    ((z(4, dtype=torch.float32), 64), {}, "int32 or int64"),
    ((ints(1, 2)[None, None], 64), {}, r"\[S\] or \[S, A\]"),
    ((ints(1, 2), 63), {}, "positive even number"),
    ((ints(1, 2), 0), {}, "positive even number"),
    ((ints(1, 2), 514), {}, "512 channels"),
    ((ints(1, 2), 64.0), {}, "positive even number"),
    ((ints(1, 2)[None], (16, 16, 16)), {}, "2 axes, dims 3"),
    ((ints(1, 2)[None], (16, 15)), {}, "positive even number"),
    ((ints(1), 64), {"base": 0.0}, "base must be positive"),
    ((ints(1), 64), {"base": float("nan")}, "base must be positive"),
    ((ints(1), 64), {"scaling": {"type": "other", "factor": 2.0}}, "scaling type"),
    ((ints(1), 64), {"scaling": {"type": "linear", "factor": 0.5}}, "at least 1"),
    ((ints(1), 64), {"scaling": {"type": "linear"}}, "at least 1"),
    ((ints(1), 64), {"scaling": {"type": "linear", "factor": 2.0, "extra": 1}}, "unknown scaling entries"),
    ((ints(1), 2), {"scaling": {"type": "ntk", "factor": 2.0}}, "above 2"),
    ((ints(1), 64), {"scaling": {"type": "yarn", "factor": 2.0}}, "original_length"),
    ((ints(1), 64), {"scaling": {"type": "yarn", "factor": 2.0, "original_length": 100, "beta_fast": 1.0, "beta_slow": 2.0}}, "beta_fast"),
])
def test_tables_refusals(arguments, keywords, match):
    with pytest.raises(ValueError, match=match):
        mflux_amd.rotary_tables(*arguments, **keywords)


Q, K, T = z(2, 5, 4, 64), z(2, 5, 2, 64), z(5, 32, dtype=torch.float32)


@pytest.mark.parametrize("arguments,keywords,match", [
    ((Q, K, T, T), {"layout": "pairs"}, "layout"),
    ((Q[0, 0], None, T, T), {}, r"\[B, S, H, D\]"),
    ((Q.to(torch.int32), None, T, T), {}, "float32, float16 or bfloat16"),
    ((z(1, 5, 2, 63), None, T, T), {}, "even size"),
    ((z(1, 5, 2, 514), None, T, T), {}, "even size"),
    ((Q, z(2, 6, 2, 64), T, T), {}, "agree"),
    ((Q, K.half(), T, T), {}, "agree"),
    ((Q, z(2, 5, 0, 64), T, T), {}, "65536 heads"),
    ((Q, K, T.to(BF16), T), {}, "float32"),
    ((Q, K, T, T[:4]), {}, "one shape"),
    ((Q, K, z(5, 33, dtype=torch.float32), z(5, 33, dtype=torch.float32)), {}, "heads have 64"),
    ((Q, K, T[:4], T[:4]), {}, "4 rows for 5 tokens"),
    ((Q, K, T[:0], T[:0]), {"positions": z(5, dtype=torch.int32)}, "empty"),
    ((Q, K, T.clone().requires_grad_(), T), {}, "no gradient"),
    ((Q, K, T, T), {"positions": z(4, dtype=torch.int32)}, "shape"),
    ((Q, K, T, T), {"positions": z(5, dtype=torch.float32)}, "int32 or int64"),
    ((Q, K, T, T), {"q_weight": z(63)}, "q_weight"),
    ((Q, K, T, T), {"q_weight": z(64, dtype=torch.float32)}, "q_weight"),
    ((Q, None, T, T), {"k_weight": z(64)}, "needs its tensor"),
    ((Q, K, T, T), {"eps": -1.0}, "eps"),
])
def test_rotary_refusals(arguments, keywords, match):
    with pytest.raises(ValueError, match=match):
        mflux_amd.rotary(*arguments, **keywords)


P = z(5, 4, 64)


@pytest.mark.parametrize("arguments,keywords,match", [
    ((Q, K, K), {"k_offsets": ints(0, 5)}, "need q_offsets"),
    ((P, z(5, 2, 64), z(5, 2, 64)), {"q_offsets": ints(0, 5), "k_lengths": ints(5)}, "not both"),
    ((Q, K, K), {"q_offsets": ints(0, 5)}, "packed"),
    ((P, P, P), {}, "without offsets"),
    ((Q, K, K[:, :4]), {}, "one shape"),
    ((Q, z(1, 5, 2, 64), z(1, 5, 2, 64)), {}, "batch"),
    ((Q, z(2, 5, 2, 72), z(2, 5, 2, 72)), {}, "head size"),
    ((Q.float(), K.float(), K.float()), {}, "float16 or all bfloat16"),
    ((Q, K.half(), K.half()), {}, "float16 or all bfloat16"),
    ((z(1, 5, 2, 60), z(1, 5, 2, 60), z(1, 5, 2, 60)), {}, "multiple of 8"),
    ((z(1, 5, 2, 264), z(1, 5, 2, 264), z(1, 5, 2, 264)), {}, "multiple of 8"),
    ((Q, z(2, 5, 3, 64), z(2, 5, 3, 64)), {}, "evenly"),
    ((Q, z(2, 5, 0, 64), z(2, 5, 0, 64)), {}, "evenly"),
    ((Q, K, K), {"scale": 0.0}, "scale"),
    ((Q, K, K), {"scale": float("inf")}, "scale"),
    ((Q, K, K), {"scale": float("nan")}, "scale"),
    ((Q, K, K), {"k_lengths": ints(1, 2, 3)}, "2 values"),
    ((Q, K, K), {"k_lengths": torch.zeros(2)}, "int32 or int64"),
    ((P, P, P), {"q_offsets": ints(0)}, "one more than"),
    ((P, P, P), {"q_offsets": ints(0, 5), "k_offsets": ints(0, 2, 5)}, "2 values"),
])
def test_attention_refusals(arguments, keywords, match):
    with pytest.raises(ValueError, match=match):
        mflux_amd.attention(*arguments, **keywords)


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="HIP device"):
        mflux_amd.attention(Q, K, K)
    with pytest.raises(RuntimeError, match="HIP device"):
        mflux_amd.rotary(Q, K, T, T)
    with pytest.raises(RuntimeError, match="HIP device"):
        mflux_amd.rotary_tables(ints(1, 2), 64)


# ---- the C ABI ------------------------------------------------------------------------------------------------------

E = {"dtype": -1, "shape": -4, "null": -5, "align": -6, "unsupported": -8, "scratch": -9}
AT = 1 << 20  # an address that is never followed: every call here is refused


def attention_args(**changes):
    a = _lib.AttentionArgs(dtype=_lib.BF16, dim=64, scale=0.125, batch=2, heads=4, kv_heads=2, q_tokens=100, k_tokens=100)
    for name in ("q", "k", "v", "y", "dy"):
        heads = 4 if name in ("q", "y", "dy") else 2
        setattr(a, name, _lib.AttentionTensor(AT, (ctypes.c_int64 * 3)(100 * heads * 64, heads * 64, 64)))
    a.out = a.dq = a.dk = a.dv = a.lse = a.delta = AT
    for name, value in changes.items():
        if "_stride" in name:
            getattr(a, name[0]).stride[int(name[-1])] = value
        elif name in ("q", "k", "v", "y", "dy"):
            getattr(a, name).p = value
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,code", [
    ({"dtype": _lib.F32}, "dtype"), ({"dtype": 7}, "dtype"), ({"dim": 0}, "shape"), ({"dim": 60}, "shape"), ({"dim": 264}, "shape"),
    ({"heads": 3}, "shape"), ({"kv_heads": 0}, "shape"), ({"heads": 0}, "shape"), ({"batch": 0}, "shape"), ({"q_tokens": 0}, "shape"),
    ({"k_tokens": 0}, "shape"), ({"k_tokens": -1}, "shape"), ({"q_tokens": 1 << 30}, "shape"), ({"k_tokens": 1 << 31}, "shape"),
    ({"scale": 0.0}, "shape"), ({"scale": float("nan")}, "shape"), ({"q": None}, "null"), ({"k": None}, "null"), ({"v": None}, "null"),
    ({"out": None}, "null"), ({"q_offsets": AT}, "null"), ({"q_offsets": AT, "k_offsets": AT, "k_lengths": AT}, "unsupported"),
    ({"q": AT + 2}, "align"), ({"out": AT + 8}, "align"), ({"k_stride1": 129}, "align"), ({"k_stride1": -128}, "shape"),
    ({"v_stride1": 1 << 24}, "shape"), ({"rest": AT + 4}, "align"),
])
def test_attention_abi_refusals(changes, code):
    lib = _lib.load()
    assert lib.mfq_attention(ctypes.byref(attention_args(**changes)), None, 0, None) == E[code]
    assert lib.mfq_attention_workspace_bytes(ctypes.byref(attention_args(**changes))) == 0


def test_attention_abi_workspaces_and_backward():
    lib = _lib.load()
    assert lib.mfq_attention(None, None, 0, None) == E["null"] and lib.mfq_attention_backward(None, None, 0, None) == E["null"]
    few = attention_args(q_tokens=1, k_tokens=10000)
    need = lib.mfq_attention_workspace_bytes(ctypes.byref(few))
    assert need > 0
    assert lib.mfq_attention(ctypes.byref(few), None, 0, None) == E["null"]
    assert lib.mfq_attention(ctypes.byref(few), AT, need - 1, None) == E["scratch"]
    assert lib.mfq_attention(ctypes.byref(few), AT + 4, need, None) == E["align"]
    grouped = attention_args()
    need = lib.mfq_attention_backward_workspace_bytes(ctypes.byref(grouped))
    assert need == 2 * 2 * (2 * 100 * 2 * 64) * 4  # two parts of two planes
    assert lib.mfq_attention_backward(ctypes.byref(grouped), AT, need - 1, None) == E["scratch"]
    for changes, code in (({"dy": None}, "null"), ({"y": None}, "null"), ({"lse": None}, "null"), ({"delta": None}, "null"),
                          ({"dq": None, "dk": None, "dv": None}, "null"), ({"dq": AT + 2}, "align")):
        assert lib.mfq_attention_backward(ctypes.byref(attention_args(**changes)), AT, 1 << 30, None) == E[code], changes


def rotary_args(**changes):
    r = _lib.RotaryArgs(dtype=_lib.BF16, layout=1, dim=64, rotated=64, batch=2, tokens=10, table_rows=10, cos=AT, sin=AT, eps=1e-6)
    for t, heads in ((r.q, 4), (r.k, 2)):
        t.x = t.dy = t.weight = t.out = t.dweight = AT
        t.heads = heads
        t.x_stride[:] = t.dy_stride[:] = (10 * heads * 64, heads * 64, 64)
    for name, value in changes.items():
        where = getattr(r, name[0]) if name[1] == "_" and name[0] in "qk" else r
        name = name[2:] if where is not r else name
        if name.startswith("stride"):
            where.x_stride[int(name[-1])] = value
        else:
            setattr(where, name, value)
    return r


@pytest.mark.parametrize("changes,code", [
    ({"dtype": 9}, "dtype"), ({"layout": 2}, "shape"), ({"dim": 0}, "shape"), ({"dim": 63}, "shape"), ({"dim": 514}, "shape"),
    ({"rotated": 66}, "shape"), ({"rotated": 3}, "shape"), ({"rotated": -2}, "shape"), ({"batch": 0}, "shape"), ({"tokens": 0}, "shape"),
    ({"tokens": 1 << 30}, "shape"), ({"table_rows": 0}, "shape"), ({"position_batch": -1}, "shape"), ({"eps": -1.0}, "shape"),
    ({"q_heads": 0}, "shape"), ({"k_heads": -1}, "shape"), ({"q_stride1": -1}, "shape"), ({"cos": None}, "null"), ({"q_x": None}, "null"),
    ({"k_out": None}, "null"),
])
def test_rotary_abi_refusals(changes, code):
    assert _lib.load().mfq_rotary(ctypes.byref(rotary_args(**changes)), None) == E[code]


def test_rotary_abi_backward_and_tables():
    lib = _lib.load()
    assert lib.mfq_rotary(None, None) == E["null"] and lib.mfq_rotary_backward(None, None, 0, None) == E["null"]
    r = rotary_args()
    need = lib.mfq_rotary_workspace_bytes(ctypes.byref(r))
    assert need > 0
    assert lib.mfq_rotary_backward(ctypes.byref(r), None, 0, None) == E["null"]
    assert lib.mfq_rotary_backward(ctypes.byref(r), AT, need - 1, None) == E["scratch"]
    assert lib.mfq_rotary_backward(ctypes.byref(r), AT + 4, need, None) == E["align"]
    assert lib.mfq_rotary_backward(ctypes.byref(rotary_args(q_dy=None)), AT, need, None) == E["null"]
    assert lib.mfq_rotary_backward(ctypes.byref(rotary_args(q_weight=None)), AT, need, None) == E["null"]
    f, axis = (ctypes.c_double * 32)(), (ctypes.c_uint8 * 32)(*([0] * 31 + [2]))
    tables = lambda n=4, axes=2, pairs=32, p=AT, f=f, axis=axis, cos=AT: lib.mfq_rotary_tables(p, n, axes, pairs, f, axis, 1.0, cos, AT, None)
    assert tables() == E["shape"]  # an axis that there is not
    axis[31] = 1
    assert tables(n=0) == tables(axes=0) == tables(pairs=0) == tables(pairs=257) == E["shape"]
    assert tables(p=None) == tables(f=None) == tables(axis=None) == tables(cos=None) == E["null"]


def test_structures_match_the_header(tmp_path):
    """The ctypes structures have the header's layout."""
    lines = []
    for c_name, py in (("mfq_rotary_tensor", _lib.RotaryTensor), ("mfq_rotary_args", _lib.RotaryArgs),
                       ("mfq_attention_tensor", _lib.AttentionTensor), ("mfq_attention_args", _lib.AttentionArgs)):
        lines.append((f"sizeof({c_name})", ctypes.sizeof(py)))
        lines += [(f"offsetof({c_name}, {f[0]})", getattr(py, f[0]).offset) for f in py._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stdio.h>\n#include "mfq.h"\nint main(void) {\n' +
                      "".join(f'  printf("%zu\\n", {expression});\n' for expression, _ in lines) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [value for _, value in lines]


def test_every_attention_kernel_raises_its_own_limit():
    """A kernel's limit of dynamic LDS is raised once per device and remembered; what remembers it belongs to that kernel alone, or
    the second of two kernels would be launched with the limit it was built with."""
    lines = subprocess.run(["nm", "-C", os.path.join(ROOT, "mflux_amd", "csrc", "libmfq.so")], capture_output=True, text=True, check=True).stdout
    names = [line.split(maxsplit=2)[2] for line in lines.splitlines() if len(line.split(maxsplit=2)) == 3]
    kernels = {n for n in names if re.search(r"::attention_(split_|dq_|dkv_)?kernel<", n) and "__device_stub__" not in n}
    flags = [n for n in names if n.endswith("::configured") and "AttentionCall" in n and "guard variable" not in n]
    if not names:
        pytest.skip("a library without symbols")
    assert len(kernels) >= 40 and len(flags) == len(kernels)


@pytest.mark.parametrize("base,dims", [(0.2, 64), (1e-12, 4), (5e-324, 128), (0.01, (2, 8))])
def test_tables_refuse_angles_that_grow_too_fast(base, dims):
    """Above 4 a position an angle leaves the range that its reduction holds for."""
    positions = ints(1) if isinstance(dims, int) else ints(1, 2)[None]
    with pytest.raises(ValueError, match="base is too small"):
        mflux_amd.rotary_tables(positions, dims, base)
    for base, dims, scaling in ((0.25, 64, None), (0.1, 2, None), (0.2, 4, None), (0.1, 64, {"type": "linear", "factor": 4.0}),
                                (0.1, 64, {"type": "ntk", "factor": 4.0})):  # these go on to the next refusal
        with pytest.raises(RuntimeError, match="HIP device"):
            mflux_amd.rotary_tables(ints(1), dims, base, scaling)
    with pytest.raises(ValueError, match="base is too small"):
        mflux_amd.rotary_tables(ints(1), 64, 0.01, {"type": "ntk", "factor": 2.0})
    with pytest.raises(ValueError, match="attention_factor"):
        mflux_amd.rotary_tables(ints(1), 64, scaling={"type": "yarn", "factor": 2.0, "original_length": 100, "attention_factor": 1e39})


def test_tables_abi_refuses_what_cannot_be_reduced():
    lib = _lib.load()
    axis = (ctypes.c_uint8 * 2)()
    for frequency, factor in ((4.1, 1.0), (-4.1, 1.0), (float("nan"), 1.0), (float("inf"), 1.0), (1.0, float("inf")), (1.0, float("nan"))):
        f = (ctypes.c_double * 2)(1.0, frequency)
        assert lib.mfq_rotary_tables(AT, 1, 1, 2, f, axis, factor, AT, AT, None) == E["shape"]


@pytest.mark.parametrize("shape", [(0,), (1, 0), (2, 0)])
def test_rotary_of_no_tokens_takes_positions(shape):
    with pytest.raises(RuntimeError, match="HIP device"):  # nothing else is wrong with the call
        mflux_amd.rotary(z(2, 0, 4, 64), None, T, T, positions=z(*shape, dtype=torch.int32))


def test_rotary_abi_refuses_a_weight_gradient_of_no_heads():
    """Nothing would write the partial sums that it is made of."""
    lib = _lib.load()
    r = rotary_args(k_heads=0)
    need = lib.mfq_rotary_workspace_bytes(ctypes.byref(r))
    assert lib.mfq_rotary_backward(ctypes.byref(r), AT, need, None) == E["shape"]


@pytest.mark.parametrize("sizes", [dict(batch=1 << 24, heads=2, kv_heads=2, q_tokens=1, k_tokens=1),       # rows of single tokens
                                   dict(batch=1 << 17, heads=256, kv_heads=256, q_tokens=128, k_tokens=1),  # tiles of 128 queries
                                   dict(batch=1 << 22, heads=4, kv_heads=4, q_tokens=1, k_tokens=129)])
def test_attention_abi_refuses_more_workgroups_than_a_launch_has(sizes):
    lib = _lib.load()
    a = attention_args(**sizes)
    if sizes["k_tokens"] == 1:
        assert lib.mfq_attention(ctypes.byref(a), None, 0, None) == E["shape"]
    assert lib.mfq_attention_backward(ctypes.byref(a), AT, 1 << 62, None) == E["shape"]
