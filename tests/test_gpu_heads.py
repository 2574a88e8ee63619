"""rotary_tables, rotary and attention against float64, element by element within the
bounds that heads_reference derives, at the sizes, masks, strides and alignments where
they can go wrong."""
import math

import pytest
import torch

import heads_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- rotary tables -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("positions,dims,base,scaling", [
    ([0], 2, 10000.0, None),
    (list(range(-5, 300)), 64, 10000.0, None),
    ([2 ** 31 - 1, -2 ** 31, 1000003, 131071], 128, 1000000.0, None),
    (list(range(1000, 1100)), 128, 10000.0, {"type": "linear", "factor": 4.0}),
    (list(range(1000, 1100)), 128, 10000.0, {"type": "ntk", "factor": 8.0}),
    (list(range(100000, 100100)), 128, 1000000.0, {"type": "yarn", "factor": 4.0, "original_length": 32768}),
    (list(range(5)), 512, 10000.0, {"type": "yarn", "factor": 2, "original_length": 100, "attention_factor": 1.0}),
    ([[0, -3, 7], [0, 90, -90], [512, 0, 1]], (16, 56, 56), 10000.0, None),
    ([[3]], (6,), 10000.0, None),
])
def test_tables(positions, dims, base, scaling):
    import mflux_amd

    p = ints(positions)
    cos, sin = mflux_amd.rotary_tables(p, dims, base, scaling)
    columns, factor = [], 1.0
    for a, d in enumerate((dims,) if isinstance(dims, int) else dims):
        f, factor = ref.rotary_frequencies(d, base, scaling)
        columns.append((p if p.ndim == 1 else p[:, a])[:, None].double() * torch.tensor(f, dtype=torch.float64, device="cuda"))
    angle = torch.cat(columns, 1)
    for got, want in ((cos, angle.cos() * factor), (sin, angle.sin() * factor)):
        assert got.dtype == F32 and got.shape == want.shape
        # float64 throughout: half a float32 step, and a float64 angle of up to 2^31 is off by 2^-22
        err = (got.double() - want).abs()
        assert bool((err <= 2.0 ** -24 * want.abs() * 1.01 + angle.abs() * 2.0 ** -50).all()), float(err.max())
    assert torch.equal(cos, mflux_amd.rotary_tables(p.long(), dims, base, scaling)[0])


@pytest.mark.parametrize("base", [0.25, 0.5, 1.0])
def test_tables_of_small_bases(base):
    """Up to what is allowed: angles of almost 2^33."""
    import mflux_amd

    p = ints([2 ** 31 - 1, -2 ** 31, 1000003, -7, 0])
    cos, sin = mflux_amd.rotary_tables(p, 64, base)
    angle = p[:, None].double() * torch.tensor(ref.rotary_frequencies(64, base, None)[0], dtype=torch.float64, device="cuda")
    for got, want in ((cos, angle.cos()), (sin, angle.sin())):
        err = (got.double() - want).abs()
        assert bool((err <= 2.0 ** -24 * want.abs() * 1.01 + angle.abs() * 2.0 ** -50).all()), float(err.max())


def test_tables_of_positions_beyond_int32():
    """As documented: the nearest position that int32 holds."""
    import mflux_amd

    far = torch.tensor([2 ** 31, 2 ** 40, -2 ** 31 - 1, -2 ** 63, 5], dtype=torch.int64, device="cuda")
    near = ints([2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, -2 ** 31, 5])
    assert all(torch.equal(a, b) for a, b in zip(mflux_amd.rotary_tables(far, 64), mflux_amd.rotary_tables(near, 64)))


# ---- rotary ------------------------------------------------------------------------------------------------------------

ROTARY = [  # B, S, H, Hkv (0: no k), D, R
    (1, 1, 1, 1, 2, 2), (1, 1, 32, 8, 128, 128), (2, 37, 24, 24, 128, 128), (3, 5, 16, 4, 128, 64), (1, 300, 4, 2, 72, 72),
    (2, 17, 3, 1, 72, 36), (1, 9, 2, 2, 50, 50), (1, 1030, 2, 0, 64, 64), (1, 3, 2, 1, 512, 512), (1, 4, 2, 1, 510, 6), (2, 3, 5, 2, 256, 0),
]


@pytest.mark.parametrize("B,S,H,Hkv,D,R", ROTARY)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rotary(B, S, H, Hkv, D, R, layout, norm, dtype):
    import mflux_amd

    print(f"B={B} S={S} H={H} Hkv={Hkv} D={D} R={R} {layout} {norm} {dtype}", flush=True)
    angles = randn(1, S + 3, R // 2, std=2.0)
    cos, sin = angles.cos(), angles.sin()
    q = randn(2, B, S, H, D, dtype=dtype, std=1.7).requires_grad_()
    k = randn(3, B, S, Hkv, D, dtype=dtype, std=0.4).requires_grad_() if Hkv else None
    qw = randn(4, D, dtype=dtype).requires_grad_() if norm else None
    kw = randn(5, D, dtype=dtype).requires_grad_() if norm and Hkv else None
    out = mflux_amd.rotary(q, k, cos, sin, layout=layout, q_weight=qw, k_weight=kw)
    out = [out] if k is None else list(out)
    grads = [randn(6 + i, *t.shape, dtype=dtype) for i, t in enumerate(out)]
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad(out, leaves, grads)))
    table = cos[None, :S].expand(B, -1, -1), sin[None, :S].expand(B, -1, -1)
    for i, (x, w) in enumerate(((q, qw), (k, kw))[:len(out)]):
        want = ref.rms_norm_rotary(x.detach(), *table, layout, None if w is None else w.detach(), 1e-6, grads[i])
        ref.check("y", out[i], *want[0])
        ref.check("dx", got[id(x)], *want[1])
        if w is not None:
            ref.check("dw", got[id(w)], *want[2])
    # without gradients: the same call, the same bits
    with torch.no_grad():
        again = mflux_amd.rotary(q, k, cos, sin, layout=layout, q_weight=qw, k_weight=kw)
    assert all(torch.equal(a, b) for a, b in zip([again] if k is None else again, out))


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_strides_positions_and_packed(offset, layout):
    """Slices of a stacked product at any address, table rows by position, a transposed gradient."""
    import mflux_amd

    B, S, H, Hkv, D = 2, 33, 6, 2, 64
    flat = randn(11, offset + B * S * (H + 2 * Hkv) * D, dtype=BF16)
    stacked = flat[offset:].view(B, S, H + 2 * Hkv, D)
    q, k = stacked[:, :, :H], stacked[:, :, H:H + Hkv]
    angles = randn(12, 50, D // 2)
    cos, sin = angles.cos(), angles.sin()
    positions = torch.randint(-20, 70, (B, S), device="cuda")  # clamped to the 50 rows
    w = randn(13, D, dtype=BF16)
    leaf_q = q.detach().requires_grad_()
    yq, yk = mflux_amd.rotary(leaf_q, k, cos, sin, layout=layout, positions=positions, q_weight=w)
    dy = randn(14, B, H, S, D, dtype=BF16).transpose(1, 2)
    dq, = torch.autograd.grad(yq, leaf_q, dy)
    rows = positions.clamp(0, 49)
    want = ref.rms_norm_rotary(q, cos[rows], sin[rows], layout, w, 1e-6, dy)
    ref.check("q", yq, *want[0])
    ref.check("dq", dq, *want[1])
    ref.check("k", yk, *ref.rms_norm_rotary(k, cos[rows], sin[rows], layout, None, 1e-6)[0])
    assert yq.is_contiguous() and yk.is_contiguous()
    # packed, and positions of one entry for all
    one = mflux_amd.rotary(q[0], k[0], cos, sin, layout=layout, positions=positions[0].int(), q_weight=w)
    assert torch.equal(one[0], yq[0]) and torch.equal(one[1], yk[0])
    shared = mflux_amd.rotary(q, None, cos, sin, layout=layout, positions=positions[1])
    each = mflux_amd.rotary(q, None, cos, sin, layout=layout, positions=positions[1:].expand(B, S))
    assert torch.equal(shared, each)


def test_rotary_empty_and_partial_gradients():
    import mflux_amd

    cos, sin = randn(1, 4, 4).cos(), randn(1, 4, 4).sin()
    for shape in ((0, 4, 2, 16), (2, 0, 2, 16)):
        q = torch.empty(shape, device="cuda", dtype=BF16, requires_grad=True)
        w = torch.ones(16, device="cuda", dtype=BF16, requires_grad=True)
        y = mflux_amd.rotary(q, None, cos, sin, q_weight=w)
        assert y.shape == shape
        dq, dw = torch.autograd.grad(y, (q, w), torch.empty_like(y))
        assert dq.shape == shape and bool((dw == 0).all())
    # the weight alone, one of two tensors alone
    q, k, w = randn(2, 1, 4, 2, 16), randn(3, 1, 4, 1, 16), randn(4, 16).requires_grad_()
    yq, yk = mflux_amd.rotary(q, k, cos, sin, q_weight=w)
    assert torch.equal(torch.autograd.grad(yq.sum(), w)[0], torch.autograd.grad(mflux_amd.rotary(q, k, cos, sin, q_weight=w)[0].sum(), w)[0])
    k.requires_grad_()
    yq, yk = mflux_amd.rotary(q, k, cos, sin)
    dk, = torch.autograd.grad(yk.sum() + yq.sum(), k)
    ref.check("dk", dk, *ref.rms_norm_rotary(k.detach(), cos[None], sin[None], "interleaved", None, 0.0, torch.ones_like(k))[1])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_without_a_norm_keeps_no_input(layout):
    """The turn back needs none: inputs that are overwritten afterwards, as buffers are, leave the gradient what it is.  A tensor
    with a norm is needed, and says so."""
    import mflux_amd

    cos, sin = randn(1, 6, 16).cos(), randn(1, 6, 16).sin()
    q, k = randn(2, 2, 6, 3, 32, dtype=BF16).requires_grad_(), randn(3, 2, 6, 1, 32, dtype=BF16).requires_grad_()
    w, dy = randn(4, 32, dtype=BF16), (randn(5, 2, 6, 3, 32, dtype=BF16), randn(6, 2, 6, 1, 32, dtype=BF16))
    want = {}
    for weights in ({}, {"q_weight": w}, {"k_weight": w}):
        for overwritten in (None, "q", "k"):
            a, b = q * 1, k * 1
            out = mflux_amd.rotary(a, b, cos, sin, layout=layout, **weights)
            if overwritten:
                (a if overwritten == "q" else b).detach().zero_()
            key = tuple(weights)
            if overwritten and overwritten + "_weight" in weights:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(out, (q, k), dy)
                continue
            got = torch.autograd.grad(out, (q, k), dy)
            assert all(torch.equal(x, y) for x, y in zip(got, want.setdefault(key, got)))
    # half of the gradients, transposed ones, and one tensor alone
    a = q * 1
    y = mflux_amd.rotary(a, None, cos, sin, layout=layout)
    got, = torch.autograd.grad(y, q, dy[0].transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got, want[()][0])
    a, b = q * 1, k.detach()
    out = mflux_amd.rotary(a, b, cos, sin, layout=layout)
    assert torch.equal(torch.autograd.grad(out[0], q, dy[0])[0], want[()][0])


@pytest.mark.parametrize("shape", [(0,), (1, 0), (2, 0)])
def test_rotary_of_no_tokens_with_positions(shape):
    import mflux_amd

    cos, sin = randn(1, 4, 4).cos(), randn(1, 4, 4).sin()
    q = torch.empty(2, 0, 2, 16, device="cuda", dtype=BF16, requires_grad=True)
    y, k = mflux_amd.rotary(q, q, cos, sin, positions=torch.empty(shape, device="cuda", dtype=torch.int64))
    assert y.shape == k.shape == q.shape and torch.autograd.grad(y, q, torch.empty_like(y))[0].shape == q.shape
    packed = mflux_amd.rotary(q[0], None, cos, sin, positions=torch.empty(0, device="cuda", dtype=torch.int32))
    assert packed.shape == q[0].shape


def test_rotary_turns_back():
    """The gradient of a turn is the turn back: applied to the result it gives the input, to rounding."""
    import mflux_amd

    q = randn(1, 2, 50, 3, 96).requires_grad_()
    angles = randn(2, 50, 32, std=3.0)
    y = mflux_amd.rotary(q, None, angles.cos(), angles.sin(), layout="half")
    back, = torch.autograd.grad(y, q, y.detach())
    assert float((back - q).detach().abs().max()) < 1e-5


# ---- attention --------------------------------------------------------------------------------------------------------

def ranges(q, k, packed_sequences=0):
    """The form that a call takes here (mfq_attention_ranges): 0 for tiles of 128 queries, otherwise the ranges of its keys."""
    import ctypes

    from mflux_amd import _lib

    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("shapes are chosen for 256 compute units")
    a = _lib.AttentionArgs(dtype=_lib.BF16, dim=q.shape[-1], scale=1.0, batch=packed_sequences or q.shape[0], heads=q.shape[-2],
                           kv_heads=k.shape[-2], q_tokens=q.shape[-3], k_tokens=k.shape[-3], out=256)
    for name in ("q", "k", "v"):
        setattr(a, name, _lib.AttentionTensor(256, (ctypes.c_int64 * 3)(8, 8, 8)))
    if packed_sequences:
        a.q_offsets = a.k_offsets = 256
    return _lib.load().mfq_attention_ranges(ctypes.byref(a))


def run_attention(form, dtype, D, H, Hkv, q_lengths, k_lengths, causal, grad, scale=None, spare=0, seed=0, tiles=None):
    """All sequences at once against each of them in float64; rows of no sequence must come out as zeros.  tiles: whether the call
    has to take the form of whole tiles of queries, or the other."""
    import mflux_amd

    n = len(q_lengths)
    if form == "packed":
        qs, ks = [spare], [spare + 1]
        for a, b in zip(q_lengths, k_lengths):
            qs.append(qs[-1] + a)
            ks.append(ks[-1] + b)
        lead_q, lead_k = (qs[-1] + spare,), (ks[-1] + spare + 1,)
        keywords = {"q_offsets": ints(qs), "k_offsets": ints(ks)}
        where = [(slice(qs[i], qs[i + 1]), slice(ks[i], ks[i + 1])) for i in range(n)]
    else:
        lead_q, lead_k = (n, max(q_lengths) + spare), (n, max(k_lengths) + spare)
        keywords = {"q_lengths": ints(q_lengths), "k_lengths": ints(k_lengths)}
        where = [((i, slice(0, q_lengths[i])), (i, slice(0, k_lengths[i]))) for i in range(n)]
    q = randn(seed + 1, *lead_q, H, D, dtype=dtype, std=1.5)
    k = randn(seed + 2, *lead_k, Hkv, D, dtype=dtype)
    v = randn(seed + 3, *lead_k, Hkv, D, dtype=dtype)
    dy = randn(seed + 4, *lead_q, H, D, dtype=dtype) if grad else None
    if tiles is not None:
        assert (ranges(q, k, n if form == "packed" else 0) == 0) == tiles
    # what no sequence holds must not be read into a result
    if spare:
        for t, i in ((q, 0), (k, 1), (v, 1)) + (((dy, 0),) if grad else ()):
            held = torch.zeros(t.shape[:-2], dtype=torch.bool, device="cuda")
            for w in where:
                held[w[i]] = True
            t[~held] = math.nan
    for t in (q, k, v):
        t.requires_grad_(grad)
    y = mflux_amd.attention(q, k, v, causal=causal, scale=scale, **keywords)
    got = {"y": y}
    if grad:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(y, (q, k, v), dy)))
    scale = D ** -0.5 if scale is None else scale
    if Hkv > 40:  # some of very many heads, spread over the compute units
        some = sorted({0, 1, 7, Hkv // 3, Hkv // 2, Hkv - 2, Hkv - 1})
        of_q = [h * (H // Hkv) + i for h in some for i in range(H // Hkv)]
        assert all(bool(t.isfinite().all()) for t in got.values())
        got = {name: t[..., of_q if name in ("y", "dq") else some, :] for name, t in got.items()}
        q, k, v = q.detach()[..., of_q, :], k.detach()[..., some, :], v.detach()[..., some, :]
        dy = None if dy is None else dy[..., of_q, :]
    for name, t in got.items():
        full_v, full_b = torch.zeros(t.shape, dtype=torch.float64, device="cuda"), torch.zeros(t.shape, dtype=torch.float64, device="cuda")
        got[name] = (t, full_v, full_b)
    for qi, ki in where:
        want = ref.attention_sequence(q.detach()[qi], k.detach()[ki], v.detach()[ki], causal, scale, None if dy is None else dy[qi])
        for name, (value, bound) in want.items():
            at = qi if name in ("y", "dq") else ki
            got[name][1][at], got[name][2][at] = value, bound
    for name, (t, value, bound) in got.items():
        ref.check(name, t, value, bound)
    return y


@pytest.mark.parametrize("form", ["batched", "packed"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,H,Hkv,q_lengths,k_lengths", [
    (128, 2, 2, [1], [1]), (128, 2, 1, [128], [128]), (128, 3, 1, [129, 1, 63], [129, 1, 63]), (64, 4, 4, [77, 30, 5], [77, 30, 5]),
    (128, 8, 2, [100, 257], [300, 257]), (80, 2, 1, [65, 200], [65, 200]), (72, 2, 2, [40], [100]), (8, 2, 1, [33], [33]),
    (96, 2, 2, [130], [70]), (256, 2, 1, [70], [70]), (192, 1, 1, [150], [150]), (128, 1, 1, [200, 100], [60, 0]), (64, 2, 1, [0, 40], [10, 40]),
])
def test_attention(form, causal, dtype, D, H, Hkv, q_lengths, k_lengths):
    """Forward and backward; lengths of zero and one, tiles that end inside, queries that see nothing."""
    print(f"{form} causal={causal} {dtype} D={D} H={H}/{Hkv} {q_lengths} {k_lengths}", flush=True)
    run_attention(form, dtype, D, H, Hkv, q_lengths, k_lengths, causal, grad=True, tiles=False)


# heads enough that whole tiles of queries fill the compute units, in the backward pass as well
@pytest.mark.parametrize("form", ["batched", "packed"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,H,Hkv,q_lengths,k_lengths", [
    (128, 530, 530, [1], [200]), (128, 530, 265, [128], [128]), (128, 270, 90, [129, 1, 63], [129, 1, 63]), (64, 260, 260, [77, 30, 5], [77, 30, 5]),
    (128, 260, 65, [100, 257], [300, 257]), (80, 300, 150, [65, 200], [65, 200]), (72, 520, 520, [40], [100]), (8, 520, 260, [33], [33]),
    (96, 264, 264, [130, 600], [70, 601]), (256, 300, 150, [150], [150]), (192, 300, 300, [150], [150]), (128, 260, 260, [200, 100], [60, 0]),
    (64, 520, 260, [0, 40], [10, 40]), (128, 200, 100, [290], [700]), (256, 300, 150, [150], [420]), (192, 300, 300, [140], [390]),
])
def test_attention_whole_tiles(form, causal, dtype, D, H, Hkv, q_lengths, k_lengths):
    """The same in the form of 128 queries to a workgroup: steps of the main loop, blocks at the edges, both parities of them."""
    print(f"{form} causal={causal} {dtype} D={D} H={H}/{Hkv} {q_lengths} {k_lengths}", flush=True)
    if max(q_lengths) * H // Hkv <= 32:
        q_lengths, k_lengths = q_lengths + [140], k_lengths + [150]
    run_attention(form, dtype, D, H, Hkv, q_lengths, k_lengths, causal, grad=True, tiles=True)


@pytest.mark.parametrize("causal", [False, True])
def test_attention_whole_tiles_leave_out_what_no_sequence_holds(causal):
    for form in ("batched", "packed"):
        run_attention(form, BF16, 128, 260, 130, [70, 129], [70, 140], causal, grad=True, spare=37, tiles=True)


@pytest.mark.parametrize("form", ["batched", "packed"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,H,Hkv,q_lengths,k_lengths", [
    (128, 8, 2, [1, 1, 1], [1, 900, 31]), (128, 28, 4, [1], [5000]), (64, 4, 4, [1, 1], [0, 700]), (80, 6, 2, [3, 0, 2], [500, 7, 33]),
    (256, 4, 1, [2], [1000]), (192, 2, 2, [1], [600]), (96, 5, 1, [4], [300]), (128, 32, 1, [1], [1030]), (128, 2, 1, [16, 16], [512, 40]),
])
def test_attention_few_queries(form, causal, dtype, D, H, Hkv, q_lengths, k_lengths):
    """The split form: key ranges that end inside a tile, ranges without keys, and its saved sums in the backward pass."""
    print(f"{form} causal={causal} {dtype} D={D} H={H}/{Hkv} {q_lengths} {k_lengths}", flush=True)
    run_attention(form, dtype, D, H, Hkv, q_lengths, k_lengths, causal, grad=True)


@pytest.mark.parametrize("form", ["batched", "packed"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lengths,k_lengths", [([70, 129], [70, 129]), ([1, 1], [300, 700]), ([50, 200], [90, 100])])
def test_attention_leaves_out_what_no_sequence_holds(form, causal, q_lengths, k_lengths):
    """NaN in every row around the sequences: none may reach a result, and the rows' own results are zeros."""
    run_attention(form, BF16, 128, 4, 2, q_lengths, k_lengths, causal, grad=True, spare=37)


def test_attention_empty():
    """No queries, no keys, no entries: nothing, or zeros, in the gradients too."""
    import mflux_amd

    for q_shape, k_shape, offsets in (((2, 0, 4, 64), (2, 5, 2, 64), None), ((2, 5, 4, 64), (2, 0, 2, 64), None), ((0, 5, 4, 64), (0, 5, 2, 64), None),
                                      ((7, 4, 64), (0, 2, 64), [0, 3]), ((0, 4, 64), (7, 2, 64), [0, 0])):
        q, k, v = (torch.ones(shape, device="cuda", dtype=BF16, requires_grad=True) for shape in (q_shape, k_shape, k_shape))
        keywords = {} if offsets is None else {"q_offsets": ints(offsets), "k_offsets": ints([0, 0])}
        y = mflux_amd.attention(q, k, v, **keywords)
        assert y.shape == q.shape and bool((y == 0).all())
        for g, t in zip(torch.autograd.grad(y, (q, k, v), torch.ones_like(y)), (q, k, v)):
            assert g.shape == t.shape and bool((g == 0).all())


def test_attention_many_short_sequences():
    """More sequences than a wavefront has lanes, empty ones among them."""
    lengths = [(7 * i) % 13 if i % 5 else 0 for i in range(150)]
    run_attention("packed", BF16, 64, 2, 1, lengths, lengths, True, grad=True)
    run_attention("packed", BF16, 64, 2, 1, [min(n, 1) for n in lengths], [n * 3 for n in lengths], True, grad=False)


def test_attention_long():
    run_attention("batched", BF16, 128, 2, 1, [2500], [2500], True, grad=True, tiles=False)
    run_attention("batched", F16, 64, 1, 1, [300], [4000], False, grad=True, tiles=False)
    run_attention("batched", BF16, 128, 14, 2, [2500], [2500], True, grad=True, tiles=True)
    run_attention("packed", F16, 64, 20, 10, [2100, 300], [2100, 1000], False, grad=True, tiles=True)


def test_attention_large_scores():
    """Scores of hundreds: the running reference moves far, probabilities of almost all keys vanish."""
    run_attention("batched", BF16, 128, 2, 2, [200], [200], False, grad=True, scale=3.0)
    run_attention("batched", BF16, 128, 260, 260, [200], [400], False, grad=True, scale=3.0, tiles=True)
    run_attention("batched", BF16, 128, 8, 2, [1], [2000], False, grad=False, scale=3.0)


def test_attention_growing_scores():
    """Every tile's maximum is above the last one's, by less and by more than the reference waits for."""
    import mflux_amd

    for step in (0.5, 3.0, 12.0):
        nk = 640
        k = torch.zeros(1, nk, 1, 64, device="cuda", dtype=BF16)
        k[0, :, 0, 0] = (torch.arange(nk, device="cuda") // 64 * step).to(BF16)
        q = torch.zeros(1, 5, 1, 64, device="cuda", dtype=BF16)
        q[..., 0] = 1.0
        v = randn(1, 1, nk, 1, 64, dtype=BF16)
        for queries in (q, q.repeat(1, 40, 1, 1), q.repeat(1, 40, 130, 1)):
            y = mflux_amd.attention(queries, k, v, scale=1.0)
            assert (ranges(queries, k) == 0) == (queries.shape[2] > 1)
            want = ref.attention_sequence(queries[0], k[0], v[0], False, 1.0)["y"]
            ref.check("y", y[0], *want)


@pytest.mark.parametrize("size", [2.0 ** 13, 2.0 ** 6, 2.0 ** -9, 2.0 ** -15])
@pytest.mark.parametrize("n", [3, 700])
def test_attention_float16_gradients_of_any_size(size, n):
    """Large and small gradients that float16 holds, through scores' gradients that it would not.  They are linear in dy: those of
    dy are off by `size` times the bound of dy / size, whose gradients are of order one, and by what is lost in the results."""
    import mflux_amd

    q, k, v = (randn(i, 1, n, 2, 64, dtype=F16).requires_grad_() for i in range(3))
    dy = (randn(5, 1, n, 2, 64) * size).to(F16)
    got = torch.autograd.grad(mflux_amd.attention(q, k, v, causal=True), (q, k, v), dy)
    want = ref.attention_sequence(q.detach()[0], k.detach()[0], v.detach()[0], True, 0.125, dy[0].double() / size)
    for name, g in zip(("dq", "dk", "dv"), got):
        value, bound = want[name][0] * size, want[name][1] * size
        inside = value.abs() + bound < 65000
        assert float(inside.float().mean()) > 0.5
        ref.check(name, g[0][inside], value[inside], bound[inside] + 2.0 ** -25)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,H,nk,form", [(1, 2, 100, 1), (1, 2, 5000, 2), (4, 2, 9000, 2), (140, 90, 300, 0)])
def test_attention_scores_of_minus_infinity(queries, H, nk, form, causal, D):
    """Scores that are all -infinity have no softmax: NaN, in every form of a call (form 2: ranges that are joined), where a row
    that sees no key is zeros.  Among others they weigh nothing."""
    import mflux_amd

    q = randn(1, 5, queries, H, D, dtype=BF16).abs()
    k, v = randn(2, 5, nk, H, D, dtype=BF16), randn(3, 5, nk, H, D, dtype=BF16)
    assert min(ranges(q, k), 2) == form
    want = mflux_amd.attention(q, k[:, 7:8], v[:, 7:8])
    k[:2, :, :, D // 2] = -math.inf
    k[1, 7] = 0.0
    k[4, 60:, :, D // 2] = -math.inf
    y = mflux_amd.attention(q, k, v, causal=causal, k_lengths=ints([nk, nk, 0, nk, nk]))
    last = y[:, -1] if causal else y  # (causal: earlier queries may see fewer keys)
    assert bool(last[0].isnan().all())
    assert torch.equal(last[1], want[1, -1] if causal else want[1])
    assert bool((y[2] == 0).all())
    assert bool(y[3].isfinite().all()) and bool(last[4].isfinite().all())
    short = mflux_amd.attention(q[4:], k[4:, :60].contiguous(), v[4:, :60].contiguous())[0]
    # (each of the two off by three roundings of at most |v|: probabilities, their sum, the result)
    assert float((last[4].float() - (short[-1] if causal else short).float()).abs().max()) <= 6.01 * 2.0 ** -8 * float(v[4, :60].float().abs().max())
    if causal and queries <= nk:  # every query sees keys here
        assert bool(y[0].isnan().all())


@pytest.mark.parametrize("D", [8, 24, 64, 72, 80, 96, 104, 128, 136, 184, 192, 200, 248, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("queries,H,nk,form", [(33, 2, 230, 1), (1, 2, 4000, 2), (140, 270, 331, 0)])
def test_attention_key_of_minus_infinity(queries, H, nk, form, dtype, D):
    """A visible key that ends with -infinity under positive queries weighs nothing, at sizes of a head that fill the kernels' tiles and
    that do not: the others' result and gradients are those of the keys without it (dq but in its own channel, where 0 times it is NaN)."""
    import mflux_amd

    at, some = 100, sorted({0, H - 1})
    q, k, v = (randn(i, 1, n, H, D, dtype=dtype) for i, n in ((1, queries), (2, nk), (3, nk)))
    dy = randn(4, 1, queries, H, D, dtype=dtype)
    q[..., -1] = q[..., -1].abs() + 0.5
    k[0, at, :, -1] = -math.inf
    assert min(ranges(q, k), 2) == form
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = mflux_amd.attention(*leaves)
    got = dict(zip(("y", "dq", "dk", "dv"), (y, *torch.autograd.grad(y, leaves, dy))))
    got = {name: t.detach()[0][:, some] for name, t in got.items()}
    keep = torch.arange(nk, device="cuda") != at
    want = ref.attention_sequence(q[0][:, some], k[0, keep][:, some], v[0, keep][:, some], False, D ** -0.5, dy[0][:, some])
    ref.check("y", got["y"], *want["y"])
    ref.check("dq", got["dq"][..., :-1], want["dq"][0][..., :-1], want["dq"][1][..., :-1])
    for name in ("dk", "dv"):
        ref.check(name, got[name][keep], *want[name])
        assert bool((got[name][at] == 0).all())


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("gap", [10.0, 15.0, 17.0, 18.0, 20.0, 22.0])
@pytest.mark.parametrize("queries,H,n", [(1, 1, 8192), (32, 2, 3000), (128, 260, 4097)])
def test_attention_float16_small_probabilities(queries, H, n, gap, D):
    """A strong key of small value and thousands whose probabilities are e^-gap of its own: together they are the result, and
    their own gradients.  A probability is made as a multiple of 2^-10 of the largest's or more, so that 2^-25 lost of it is 2^-35; for dv
    it is a multiple of 2^-13 of 1: 2^-38."""
    import mflux_amd

    lost = 2.0 ** -35, 2.0 ** -38
    for at in (0, n // 2, n - 1):  # the strong key before, among and behind the others
        k = randn(1, 1, n, 1, D, dtype=F16, std=0.05)
        k[..., 0] = 0.0
        k[0, at, 0, 0] = gap
        v = (randn(2, 1, n, 1, D) + 1.0).to(F16)
        v[0, at] = 0.0
        q = randn(3, 1, queries, 1, D, dtype=F16, std=0.1)
        q[..., 0] = 1.0
        call = [t.expand(-1, -1, H, -1).detach().requires_grad_() for t in (q, k, v)]
        assert (ranges(*call[:2]) == 0) == (H > 2)
        y = mflux_amd.attention(*call, scale=1.0)
        if gap > 20.0 or queries == 1:
            for h in (0, H - 1):
                ref.check("y", y[0, :, h:h + 1], *ref.attention_sequence(q[0], k[0], v[0], False, 1.0, lost_p=lost)["y"])
            continue
        dy = (randn(4, 1, queries, 1, D) + 1.0).to(F16)
        dv, = torch.autograd.grad(y, call[2], dy.expand(-1, -1, H, -1))
        want = ref.attention_sequence(q[0], k[0], v[0], False, 1.0, dy[0], lost_p=lost)
        for h in (0, H - 1):
            ref.check("y", y[0, :, h:h + 1], *want["y"])
            ref.check("dv", dv[0, :, h:h + 1], *want["dv"])


def test_attention_float16_large_scores():
    """Scores of hundreds, in both forms of a call."""
    run_attention("batched", F16, 128, 2, 2, [200], [200], False, grad=True, scale=3.0)
    run_attention("batched", F16, 128, 260, 260, [200], [400], False, grad=True, scale=3.0, tiles=True)
    run_attention("batched", F16, 128, 8, 2, [1], [2000], False, grad=False, scale=3.0)


@pytest.mark.parametrize("queries,H", [(96, 2), (2, 2), (96, 260)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_masked_infinities(queries, H, bad):
    """A key that a query does not see never reaches it, whatever it and its value hold."""
    import mflux_amd

    nk = 200
    q, k, v = randn(1, 1, queries, H, 128, dtype=BF16), randn(2, 1, nk, H, 128, dtype=BF16), randn(3, 1, nk, H, 128, dtype=BF16)
    assert (ranges(q, k) == 0) == (H > 2)
    want = mflux_amd.attention(q, k, v, causal=True)
    at = nk - queries // 2
    k[0, at, 0] = bad
    v[0, at:, 1, 5] = bad
    q2 = q.clone()
    got = mflux_amd.attention(q2, k, v, causal=True)
    sees = torch.arange(queries, device="cuda") + nk - queries >= at
    # (with a row that is not finite its tile is added up row by row: another order of the same sums)
    off = (got.float() - want.float()).abs()[0, ~sees]
    assert bool((off <= 2.0 ** -8 * want.float().abs()[0, ~sees] + 1e-3).all())
    assert bool((~got[0, sees][:, 1, 5].isfinite()).all())
    # a query that is not finite stays alone
    q2[0, 0] = bad
    got2 = mflux_amd.attention(q2, k, v, causal=True)
    assert torch.equal(got2[0, 1:].view(torch.int16), got[0, 1:].view(torch.int16))


@pytest.mark.parametrize("H", [1, 530])
def test_attention_backward_masked_infinities(H):
    """Rows behind a sequence's visible part do not reach gradients either: keys that no query sees but the last."""
    import mflux_amd

    n = 100
    q, k, v, dy = (randn(i, 1, n, H, 64, dtype=BF16) for i in range(4))
    cut = 70

    def gradients(q, k, v, dy, upto):
        q, k, v = (t.detach().clone().requires_grad_() for t in (q, k, v))
        y = mflux_amd.attention(q, k, v, causal=True)
        return torch.autograd.grad(y, (q, k, v), dy)

    want = gradients(q, k, v, dy, n)
    k2, v2 = k.clone(), v.clone()
    k2[0, cut:] = math.nan
    v2[0, cut:] = math.inf
    got = gradients(q, k2, v2, dy, n)
    assert bool((got[0][0, :cut].float() - want[0][0, :cut].float()).abs().max() <= 0.02)
    # a query row that is not finite reaches the keys it sees and no later ones
    q2, dy2 = q.clone(), dy.clone()
    q2[0, :30] = math.nan
    dy2[0, :30] = math.nan
    got = gradients(q2, k, v, dy2, n)
    for a, b in zip(got[1:], want[1:]):
        assert bool(a[0, 30:].isfinite().all()) and float((a[0, 30:].float() - b[0, 30:].float()).abs().max()) <= 0.05


@pytest.mark.parametrize("H,tiles", [(1, False), (260, True)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("D", [128, 136, 192, 200, 256])
def test_attention_masked_infinities_of_large_heads(D, bad, H, tiles):
    """Behind whole tiles, at every size of a head: what is not finite behind a key leaves the queries in front of it what they are in
    the shorter sequence, and in front of a query it leaves the keys behind it what they are without those queries."""
    import mflux_amd

    n, cut, some = 400, 300, [0, H - 1]
    q, k, v, dy = (randn(i + 1, 1, n, H, D, dtype=BF16) for i in range(4))
    assert (ranges(q, k) == 0) == tiles

    def run(q, k, v, dy):
        q, k, v = (t.detach().clone().requires_grad_() for t in (q, k, v))
        y = mflux_amd.attention(q, k, v, causal=True)
        return [t[0][:, some] for t in (y.detach(), *torch.autograd.grad(y, (q, k, v), dy))]

    def sequence(*t):
        return [x[0][:, some] for x in t]

    k2, v2 = k.clone(), v.clone()
    k2[0, cut + 3:] = bad
    v2[0, cut:] = bad
    y, dq, _, _ = run(q, k2, v2, dy)
    a, b, c, d = sequence(q[:, :cut], k[:, :cut], v[:, :cut], dy[:, :cut])
    want = ref.attention_sequence(a, b, c, True, D ** -0.5, d)
    ref.check("y", y[:cut], *want["y"])
    ref.check("dq", dq[:cut], *want["dq"])
    assert bool((~y[cut + 3:].isfinite()).all())
    q2, dy2 = q.clone(), dy.clone()
    q2[0, :cut - 5] = bad
    dy2[0, :cut] = bad
    _, _, dk, dv = run(q2, k, v, dy2)
    a, b, c, d = sequence(q[:, cut:], k, v, dy[:, cut:])
    want = ref.attention_sequence(a, b, c, True, D ** -0.5, d)
    for name, t in (("dk", dk), ("dv", dv)):
        ref.check(name, t[cut:], want[name][0][cut:], want[name][1][cut:])


@pytest.mark.parametrize("queries", [100, 1])
def test_attention_strides(queries):
    """Slices of a stacked product, the [B, H, S, D] order, an odd address, an expanded batch and head: the same bits."""
    import mflux_amd

    B, S, H, Hkv, D = 2, 300, 4, 2, 64
    stacked = randn(1, B, S, H + 2 * Hkv, D, dtype=BF16)
    q, k, v = stacked[:, S - queries:, :H], stacked[:, :, H:H + Hkv], stacked[:, :, H + Hkv:]
    want = mflux_amd.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(mflux_amd.attention(q, k, v, causal=True), want)
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(mflux_amd.attention(*t, causal=True), want)

    def odd(x):
        flat = torch.empty(x.numel() + 3, device="cuda", dtype=x.dtype)
        flat[3:] = x.reshape(-1)
        return flat[3:].view(x.shape)

    assert torch.equal(mflux_amd.attention(odd(q), odd(k), odd(v), causal=True), want)
    wide = torch.empty(B, S, Hkv, D + 5, device="cuda", dtype=BF16)
    wide[..., :D] = k
    assert torch.equal(mflux_amd.attention(q, wide[..., :D], v, causal=True), want)
    one = mflux_amd.attention(q, k[:1].expand(B, -1, -1, -1), v[:1, :, :1].expand(B, S, Hkv, D), causal=True)
    assert torch.equal(one, mflux_amd.attention(q, k[:1].repeat(B, 1, 1, 1), v[:1, :, :1].repeat(B, 1, Hkv, 1), causal=True))
    # gradients of expanded inputs are summed over what they were expanded to
    if queries > 1:
        base = k[:1].detach().clone().requires_grad_()
        y = mflux_amd.attention(q, base.expand(B, -1, -1, -1), v)
        g, = torch.autograd.grad(y, base, torch.ones_like(y).transpose(1, 2).contiguous().transpose(1, 2))
        full = base.detach().repeat(B, 1, 1, 1).requires_grad_()
        g2, = torch.autograd.grad(mflux_amd.attention(q, full, v), full, torch.ones_like(y))
        assert float((g - g2.float().sum(0, keepdim=True)).abs().max()) <= 2.0 ** -7 * float(g2.float().abs().sum(0).max())


def test_attention_of_a_cache_allocated_far_beyond_its_keys():
    """Lengths of an eighth to a thousandth of the keys that there is room for, and none; what lies behind them is NaN."""
    import mflux_amd

    nk, lengths = 20000, [2500, 1, 0, 19, 160]
    q, k, v = randn(1, 5, 1, 8, 128, dtype=BF16), randn(2, 5, nk, 2, 128, dtype=BF16), randn(3, 5, nk, 2, 128, dtype=BF16)
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = math.nan, math.nan
    assert ranges(q, k) > 1
    y = mflux_amd.attention(q, k, v, causal=True, k_lengths=ints(lengths))
    for i, n in enumerate(lengths):
        ref.check("y", y[i], *ref.attention_sequence(q[i], k[i, :n], v[i, :n], True, 128 ** -0.5)["y"])


@pytest.mark.parametrize("strides", [(2 ** 31 + 64, 512, 128), (2 ** 24 * 150, 2 ** 24 - 8, 128)])
def test_offsets_beyond_32_bits(strides):
    """Entries and tokens that lie so far apart that elements, or a tile's bytes, pass 2^31: the bits of dense tensors."""
    import mflux_amd

    n = 140
    buffer = torch.empty((1 * strides[0] + n * strides[1] + 1024), device="cuda", dtype=BF16)
    far = [buffer.as_strided((2, n, 2, 128), (*strides, 1), i * 256) for i in range(2)]
    near = [randn(i, 2, n, 2, 128, dtype=BF16) for i in range(2)]
    for a, b in zip(far, near):
        a.copy_(b)
    q, dy = randn(5, 2, n, 4, 128, dtype=BF16), randn(6, 2, n, 4, 128, dtype=BF16)

    def all_of(k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        y = mflux_amd.attention(*leaves, causal=True)
        single = mflux_amd.attention(q[:, -1:], k, v)
        many = mflux_amd.attention(q.repeat(1, 1, 40, 1), k, v)
        turned = mflux_amd.rotary(k.detach(), v.detach(), cos, sin, layout="half", q_weight=w)
        return (y, single, many, *turned, *torch.autograd.grad(y, leaves, dy))

    cos, sin, w = randn(7, n, 64).cos(), randn(8, n, 64).sin(), randn(9, 128, dtype=BF16)
    for a, b in zip(all_of(*far), all_of(*near)):
        assert torch.equal(a, b)


def test_attention_same_bits_every_time():
    import mflux_amd

    q, k, v = (randn(i, 700, h, 128, dtype=BF16).requires_grad_() for i, h in ((1, 6), (2, 2), (3, 2)))
    offsets = ints([0, 300, 301, 700])
    dy = randn(4, 700, 6, 128, dtype=BF16)
    first = None
    for _ in range(3):
        y = mflux_amd.attention(q, k, v, causal=True, q_offsets=offsets)
        all_ = (y, *torch.autograd.grad(y, (q, k, v), dy))
        first = first or all_
        assert all(torch.equal(a, b) for a, b in zip(first, all_))


def test_attention_bad_offsets_and_lengths_stay_inside():
    """Whatever lengths and offsets hold, they are clamped: what is there is what a clamped call gives."""
    import mflux_amd

    q, k, v = (randn(i, 2, 90, 2, 64, dtype=BF16) for i in range(3))
    got = mflux_amd.attention(q, k, v, q_lengths=ints([-7, 10 ** 6]), k_lengths=ints([2 ** 31 - 1, 40]))
    want = mflux_amd.attention(q, k, v, q_lengths=ints([0, 90]), k_lengths=ints([90, 40]))
    assert torch.equal(got, want)
    p = [t.reshape(180, 2, 64) for t in (q, k, v)]
    got = mflux_amd.attention(*p, q_offsets=ints([-5, 60, 10 ** 9]), causal=True)
    want = mflux_amd.attention(*p, q_offsets=ints([0, 60, 180]), causal=True)
    assert torch.equal(got, want)


def test_attention_against_differences():
    """A gradient against central differences of the result, with the step that float16 values and float32 sums allow."""
    import mflux_amd

    torch.manual_seed(3)
    q, k, v = (randn(i, 1, 12, 2, 32, dtype=F16, std=0.5) for i in range(3))
    dy = randn(9, 1, 12, 2, 32, dtype=F16)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(mflux_amd.attention(*leaves, causal=True), leaves, dy)
    step = 2.0 ** -3
    for n, (t, g) in enumerate(zip((q, k, v), grads)):
        direction = torch.randint(0, 2, t.shape, device="cuda").to(F16) * 2 - 1
        ends = []
        for sign in (1, -1):
            moved = [x.double() for x in (q, k, v)]
            moved[n] = moved[n] + sign * step * direction.double() / 16
            out = ref.attention_sequence(*(m[0] for m in moved), True, 32 ** -0.5)["y"][0]
            ends.append((out * dy[0].double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step / 16)
        got = float((g.double() * direction.double()).sum())
        # each gradient's rounding, and the third derivative times the step's square
        assert abs(got - slope) <= 0.02 * float(g.double().abs().sum()) ** 0.5 + 0.02 * abs(slope) + 0.05


# ---- together ----------------------------------------------------------------------------------------------------------

def test_block_together():
    """The stacked q/k/v product, head norms and rotation, attention and the output product, as a block runs them, with gradients
    to the block's input, against the same in float64 on the same quantized weights."""
    import mflux_amd
    from mflux_amd import nn

    torch.manual_seed(0)
    B, S, H, D = 2, 150, 4, 64
    dims = H * D
    layers = [nn.Linear(dims, dims, bias=False, device="cuda", dtype=BF16).to_quantized(bits=8) for _ in range(4)]
    qkv, out = nn.concat_quantized(layers[:3]), layers[3]
    x = randn(1, B, S, dims, dtype=BF16).requires_grad_()
    qw, kw = (randn(i, D, dtype=BF16, std=0.1).add(1).requires_grad_() for i in (2, 3))
    ids = torch.stack([torch.zeros(S), torch.arange(S) // 15, torch.arange(S) % 15], 1).int().cuda()
    cos, sin = mflux_amd.rotary_tables(ids, (16, 24, 24))
    dy = randn(4, B, S, dims, dtype=BF16)

    def block(x, lengths):
        q, k, v = qkv(x).view(B, S, 3, H, D).unbind(2)
        q, k = mflux_amd.rotary(q, k, cos, sin, q_weight=qw, k_weight=kw)
        return out(mflux_amd.attention(q, k, v, k_lengths=lengths).reshape(B, S, dims))

    lengths = ints([S, 90])
    y = block(x, lengths)
    got = torch.autograd.grad(y, (x, qw, kw), dy)

    w = [mflux_amd.dequantize(l.weight, l.scales, l.biases, l.group_size, l.bits).double() for l in layers]
    x64, qw64, kw64 = (t.detach().double().requires_grad_() for t in (x, qw, kw))
    q, k, v = ((x64 @ m.t()).view(B, S, H, D) for m in w[:3])

    def turned(t, g):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * g
        a, b, c, s = t[..., 0::2], t[..., 1::2], cos.double()[None, :, None], sin.double()[None, :, None]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)

    q, k = turned(q, qw64), turned(k, kw64)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(D)
    s = s.masked_fill(torch.arange(S, device="cuda") >= lengths[:, None, None, None], -math.inf)
    want_y = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v).reshape(B, S, dims) @ w[3].t()
    want = torch.autograd.grad(want_y, (x64, qw64, kw64), dy.double())
    # half a dozen roundings to bfloat16 in a row, each 2^-8 of its values: in the 2-norm well below their sum
    for name, a, b in (("y", y, want_y), ("dx", got[0], want[0]), ("dqw", got[1], want[1]), ("dkw", got[2], want[2])):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel <= 8 * 2.0 ** -8, f"{name}: {rel}"


def test_prompt_then_tokens():
    """A prompt's attention row by row as single tokens over the keys so far: the same values to rounding."""
    import mflux_amd

    n, H, Hkv, D = 130, 8, 2, 128
    q, k, v = randn(1, 1, n, H, D, dtype=BF16), randn(2, 1, n, Hkv, D, dtype=BF16), randn(3, 1, n, Hkv, D, dtype=BF16)
    prompt = mflux_amd.attention(q, k, v, causal=True)
    cache_k, cache_v = torch.full((1, 4 * n, Hkv, D), math.nan, device="cuda", dtype=BF16), torch.full((1, 4 * n, Hkv, D), math.nan, device="cuda", dtype=BF16)
    for i in range(n):
        cache_k[:, i], cache_v[:, i] = k[:, i], v[:, i]
        if i % 13 == 0 or i == n - 1:
            token = mflux_amd.attention(q[:, i:i + 1], cache_k, cache_v, causal=True, k_lengths=ints([i + 1]))
            want = ref.attention_sequence(q[0, i:i + 1], k[0, :i + 1], v[0, :i + 1], False, D ** -0.5)["y"]
            ref.check("token", token[0], *want)
            ref.check("prompt", prompt[0, i:i + 1], *want)


# ---- streams, graphs ----------------------------------------------------------------------------------------------------

def test_other_stream():
    import mflux_amd

    q, k, v = (randn(i, 1, 500, 64, 128, dtype=BF16) for i in range(3))
    assert ranges(q, k) == 0
    want = mflux_amd.attention(q, k, v, causal=True)
    token = mflux_amd.attention(q[:, -1:], k, v)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, got_token = mflux_amd.attention(q, k, v, causal=True), mflux_amd.attention(q[:, -1:], k, v)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(got_token, token)


def test_captured_and_replayed():
    """Two graphs (a training step of a prompt, a token over a cache that grows by replays) and eager calls in between."""
    import mflux_amd

    q, k, v = (randn(i, 1, 300, 4, 64, dtype=BF16).requires_grad_() for i in range(3))
    w = randn(7, 64, dtype=BF16).requires_grad_()
    dy = randn(4, 1, 300, 4, 64, dtype=BF16)
    positions = torch.arange(300, device="cuda", dtype=torch.int32)

    def step():
        cos, sin = mflux_amd.rotary_tables(positions, 64)
        a, b = mflux_amd.rotary(q, k, cos, sin, q_weight=w, k_weight=w)
        y = mflux_amd.attention(a, b, v, causal=True)
        return (y, *torch.autograd.grad(y, (q, k, v, w), dy))

    cache_k, cache_v = (randn(i, 2, 900, 2, 128, dtype=BF16) for i in (5, 6))
    token = randn(8, 2, 1, 8, 128, dtype=BF16)
    lengths = ints([1, 500])

    def decode():
        return mflux_amd.attention(token, cache_k, cache_v, causal=True, k_lengths=lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), decode()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs = [], []
    for work in (step, decode):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs.append(work())
        graphs.append(g)
    for i in range(4):
        with torch.no_grad():
            q.copy_(randn(20 + i, *q.shape, dtype=BF16))
            token.copy_(randn(30 + i, *token.shape, dtype=BF16))
            lengths.add_(97)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs[0], step()))
        assert torch.equal(outputs[1], decode())


def test_capture_next_to_a_living_graph_is_refused():
    """An eager result of the same leaves on the default stream: its nodes would end the process when the captured backward pass
    reaches them.  Refused before anything is captured; without it the same capture works."""
    import mflux_amd

    q = randn(1, 1, 20, 2, 64, dtype=BF16).requires_grad_()
    cos, sin = randn(2, 20, 32).cos(), randn(2, 20, 32).sin()
    for call in (lambda: mflux_amd.attention(q, q.detach(), q.detach()), lambda: mflux_amd.rotary(q, None, cos, sin)):
        want = torch.autograd.grad(call(), q, torch.ones_like(q))[0]
        held = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="graph is being captured"):
            with torch.cuda.graph(graph):
                call()
        torch.cuda.synchronize()
        del held, graph
        graph = torch.cuda.CUDAGraph()
        ones = torch.ones_like(q)
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), q, ones)[0]
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_no_second_derivative():
    import mflux_amd

    q, k, v = (randn(i, 1, 9, 2, 32, dtype=BF16).requires_grad_() for i in range(3))
    g, = torch.autograd.grad(mflux_amd.attention(q, k, v).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.float().sum().backward()
    cos, sin = randn(2, 9, 16).cos(), randn(2, 9, 16).sin()
    g, = torch.autograd.grad(mflux_amd.rotary(q, None, cos, sin).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.float().sum().backward()


def test_no_forward_mode():
    """A tangent is refused, not dropped, on every operand and with or without a gradient in reverse mode as well."""
    import mflux_amd
    from torch.autograd import forward_ad

    q, k, v = (randn(i, 1, 9, 2, 32, dtype=BF16) for i in range(3))
    w = randn(4, 32, dtype=BF16)
    cos, sin = randn(2, 9, 16).cos(), randn(2, 9, 16).sin()
    calls = [((q, k, v), lambda q, k, v: mflux_amd.attention(q, k, v)),
             ((q, k, cos, sin, w, w.clone()), lambda q, k, cos, sin, a, b: mflux_amd.rotary(q, k, cos, sin, q_weight=a, k_weight=b)[0])]
    for operands, call in calls:
        for i, t in enumerate(operands):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward mode"):
                    call(*operands[:i], dual, *operands[i + 1:])
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                    call(*operands[:i], dual, *operands[i + 1:])
                # a dual level alone refuses nothing
                assert torch.equal(call(*operands), call(*operands))
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.func.jvp(lambda x: call(*operands[:i], x, *operands[i + 1:]), (t,), (torch.ones_like(t),))


def test_c_entry_points_agree_with_the_ops():
    """The C ABI on the same buffers gives the ops' bits."""
    import ctypes

    import mflux_amd
    from mflux_amd import _lib

    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    q, k, v = randn(1, 2, 70, 4, 64, dtype=BF16), randn(2, 2, 70, 2, 64, dtype=BF16), randn(3, 2, 70, 2, 64, dtype=BF16)
    a = _lib.AttentionArgs(dtype=_lib.BF16, causal=1, dim=64, scale=0.125, batch=2, heads=4, kv_heads=2, q_tokens=70, k_tokens=70)
    y = torch.empty_like(q)
    for name, t in (("q", q), ("k", k), ("v", v)):
        setattr(a, name, _lib.AttentionTensor(t.data_ptr(), (ctypes.c_int64 * 3)(*t.stride()[:3])))
    a.out = y.data_ptr()
    assert lib.mfq_attention_workspace_bytes(ctypes.byref(a)) == 0
    _lib.check("mfq_attention", lib.mfq_attention(ctypes.byref(a), None, 0, stream))
    assert torch.equal(y, mflux_amd.attention(q, k, v, causal=True))
    cos, sin = randn(4, 70, 32).cos(), randn(4, 70, 32).sin()
    r = _lib.RotaryArgs(dtype=_lib.BF16, layout=1, dim=64, rotated=64, batch=2, tokens=70, table_rows=70, cos=cos.data_ptr(), sin=sin.data_ptr())
    yq, yk = torch.empty_like(q), torch.empty_like(k)
    for name, t, out in (("q", q, yq), ("k", k, yk)):
        setattr(r, name, _lib.RotaryTensor(x=t.data_ptr(), out=out.data_ptr(), x_stride=(ctypes.c_int64 * 3)(*t.stride()[:3]), heads=t.shape[2]))
    _lib.check("mfq_rotary", lib.mfq_rotary(ctypes.byref(r), stream))
    want = mflux_amd.rotary(q, k, cos, sin, layout="half")
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
