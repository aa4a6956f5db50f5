"""Rotary positions of several axes on the GPU.

The rotation by axes does the arithmetic of the rotation at one position on
other table entries: rows put together by hand (each pair's column of the row at
its axis' position) are what it has to agree with. Halves, whose multiply-adds
are written out: bit for bit with the plain ops, outputs and gradients alike.
Neighbouring pairs, where the compiler chooses which product of u c - v s goes
into the multiply-add, in each kernel as it likes: both are within the bounds of
the plain ops against the formulas in 64 bits (test_gpu_qk_rope.py derives them:
rotation 2^-23, norm 2^-18, its gradients 2^-17 of the terms' magnitudes beside
the result's rounding).
"""

import math

import pytest
import torch
from test_gpu_qk_rope import check, grads64, norm64, rotate64

from triton_ops import RoPEAxes

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(math.prod(shape), device="cuda", generator=g).view(shape).to(DT[dtype])


def make(b, s, hq, hk, d, axes, dtype, table, rows=300, seed=0, index=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    angle = torch.rand(rows, sum(axes.sections), generator=g, device="cuda", dtype=torch.float64) * 2 * math.pi
    cos, sin = (torch.cat([f(angle)] * 2, -1).to(DT[table]) for f in (torch.cos, torch.sin))
    at = torch.randint(rows, (len(axes.sections), b, s), device="cuda", generator=g, dtype=index)
    qkv = randn((b, s, hq + 2 * hk, d), dtype, seed + 2)
    return qkv[:, :, :hq], qkv[:, :, hq:hq + hk], cos, sin, at


def joined(cos, sin, at, axes):
    """Tables of a row for each token, and the tokens' places in them."""
    which = axes.axis_of_pairs()
    rows = []
    for t in (cos, sin):
        half = torch.stack([t[at[a].long(), i] for i, a in enumerate(which)], -1)
        rows.append(torch.cat([half, half], -1).flatten(0, -2))
    return (*rows, torch.arange(rows[0].shape[0], device="cuda").view(at.shape[1:]))


# batch, seq, q heads, k heads, head_dim, sections, order, pairs, dtype, table dtype
CASES = [
    (64, 1, 32, 8, 128, (16, 24, 24), "blocks", False, "bf16", "f32"),
    (1, 1, 1, 1, 6, (1, 1, 1), "cycle", False, "f32", "f32"),
    (2, 7, 5, 2, 64, (12, 10, 10), "cycle", False, "f16", "f16"),
    (2, 7, 5, 2, 64, (12, 10, 10), "cycle", True, "f16", "f16"),
    (3, 5, 4, 1, 128, (8, 28, 28), "blocks", True, "bf16", "bf16"),
    (1, 40, 3, 3, 80, (8, 16, 16), "blocks", False, "bf16", "f32"),
    (1, 9, 3, 1, 96, (9, 20, 19), "cycle", False, "f32", "f32"),
    (1, 9, 3, 1, 96, (9, 20, 19), "blocks", True, "f16", "f32"),
    (2, 6, 2, 2, 128, (16, 16, 16), "blocks", False, "bf16", "f32"),       # part of the head
    (2, 6, 2, 2, 36, (9, 8), "cycle", False, "f16", "bf16"),               # no vector width fits
    (2, 6, 2, 1, 7, (1, 1), "blocks", True, "f32", "f16"),                 # odd head width
    (1, 5, 2, 1, 512, (200, 20, 16, 20), "cycle", False, "bf16", "f32"),   # four axes
    (1, 3, 1, 1, 1024, (300, 100, 112), "cycle", True, "f32", "f32"),
    (4, 700, 8, 2, 64, (8, 12, 12), "blocks", False, "bf16", "f32"),
    (1, 2500, 8, 2, 128, (24, 20, 20), "cycle", False, "bf16", "f32"),     # four heads a group, then the stream
    (2, 3001, 8, 3, 128, (24, 20, 20), "cycle", False, "bf16", "bf16"),
    (1, 6100, 13, 3, 80, (8, 16, 16), "cycle", True, "f16", "f32"),
    (1, 6100, 12, 4, 128, (16, 24, 24), "blocks", True, "f32", "f32"),
    (1, 9000, 9, 5, 64, (16, 16), "blocks", False, "f16", "f16"),
]


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_agrees_with_joined_rows(cuda, monkeypatch, case, extension):
    from triton_ops import _lib, fused_qk_norm_rope, fused_rope

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    b, s, hq, hk, d, sections, order, pairs, dtype, table = case
    axes = RoPEAxes(sections, order)
    q, k, cos, sin, at = make(b, s, hq, hk, d, axes, dtype, table, index=torch.int32 if pairs else torch.int64)
    rows = joined(cos, sin, at, axes)
    wq, wk = 1 + 0.3 * randn((d,), "f32", 7), 1 + 0.3 * randn((d,), "f32", 8)
    gq, gk = randn(q.shape, dtype, 9), randn(k.shape, dtype, 10)

    def passes(*tables, **more):
        with torch.no_grad():
            served = (*fused_rope(q, k, *tables, interleaved=pairs, **more),
                      *fused_qk_norm_rope(q, k, wq, wk, *tables, 1e-5, interleaved=pairs, **more))
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        out = fused_rope(*leaves[:2], *tables, interleaved=pairs, **more)
        normed = fused_qk_norm_rope(*leaves, *tables, 1e-5, interleaved=pairs, **more)
        return (*served, *torch.autograd.grad(out, leaves[:2], [gq, gk]), *torch.autograd.grad(normed, leaves, [gq, gk]))

    got = passes(cos, sin, at, axes=axes)
    if not pairs:
        for i, (x, y) in enumerate(zip(got, passes(*rows))):
            assert x.dtype == y.dtype and torch.equal(x, y), i
        return
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        x, w, g = x.double(), w.double(), g.double()
        for value, seen, share in ((x, got[i], 2.0**-23), (norm64(x, w, 1e-5)[0], got[2 + i], 2.0**-18)):
            check(seen, rotate64(value, *rows, True), share * rotate64(value, *rows, True, magnitude=True), "outputs")
        check(got[4 + i], rotate64(g, *rows, True, inverse=True), 2.0**-23 * rotate64(g, *rows, True, magnitude=True), "rotation back")
        dx, dx_m, dw, dw_m = grads64(x, w, g, *rows, True, 1e-5)
        check(got[6 + i], dx, 2.0**-17 * dx_m, "gradient")
        check(got[8 + i], dw, 2.0**-17 * dw_m, "weight")


@pytest.mark.parametrize("case", [CASES[0], CASES[3], CASES[8]], ids=str)
def test_against_formulas(cuda, case):
    from triton_ops import fused_qk_norm_rope, fused_rope
    from triton_ops.kernels.rope import rope_heads_reference

    b, s, hq, hk, d, sections, order, pairs, dtype, table = case
    axes = RoPEAxes(sections, order)
    q, k, cos, sin, at = make(b, s, hq, hk, d, axes, dtype, table)
    w = 1 + 0.3 * randn((d,), "f32", 7)
    g = randn(q.shape, dtype, 9)
    x = q.detach().requires_grad_()
    y, _ = fused_rope(x, None, cos, sin, at, interleaved=pairs, axes=axes)
    z, _ = fused_qk_norm_rope(x, None, w, None, cos, sin, at, 1e-5, interleaved=pairs, axes=axes)
    wide = q.detach().double().requires_grad_()
    normed = wide / torch.sqrt(wide.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    # magnitudes: a rotated column has at most |u| + |v| of its pair
    for got, ref, share in ((y, rope_heads_reference(wide, cos, sin, at, pairs, axes), 2.0**-22),
                            (z, rope_heads_reference(normed, cos, sin, at, pairs, axes), 2.0**-17)):
        (dx,) = torch.autograd.grad(got, x, g)
        (ref_dx,) = torch.autograd.grad(ref, wide, g.double(), retain_graph=True)
        for a, e, most in ((got, ref, ref), (dx, ref_dx, ref_dx)):
            slack = share * 4 * most.detach().abs().amax(-1, keepdim=True)
            bound = e.detach().abs() * (torch.finfo(a.dtype).eps / 2) * 1.01 + slack + 2.0**-25
            assert ((a.detach().double() - e.detach()).abs() <= bound).all()


@pytest.mark.parametrize("extension", [True, False])
def test_positions_of_any_stride(cuda, monkeypatch, extension):
    """[batch, seq, axes] storage, positions shared by the batch, flattened tokens."""
    from triton_ops import _lib, fused_rope

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    axes = RoPEAxes((8, 12, 12), "cycle")
    q, k, cos, sin, at = make(3, 10, 4, 2, 64, axes, "bf16", "f32")
    want = fused_rope(q, k, cos, sin, at, axes=axes)
    last = at.movedim(0, -1).contiguous().movedim(-1, 0)
    assert all(torch.equal(x, y) for x, y in zip(fused_rope(q, k, cos, sin, last, axes=axes), want))
    every_second = torch.stack([at, at + 1], -1)[..., 0]
    assert all(torch.equal(x, y) for x, y in zip(fused_rope(q, k, cos, sin, every_second, axes=axes), want))
    flat = fused_rope(q.reshape(30, 4, 64), None, cos, sin, at.reshape(3, 30), axes=axes)[0]
    assert torch.equal(flat.view(3, 10, 4, 64), want[0])
    shared = fused_rope(q, k, cos, sin, at[:, 0], axes=axes)
    same = fused_rope(q, k, cos, sin, at[:, :1].expand(3, 3, 10), axes=axes)
    assert all(torch.equal(x, y) for x, y in zip(shared, same))
    one = fused_rope(q, k, cos, sin, at[:, :1, :1], axes=axes)
    assert all(torch.equal(x, y) for x, y in zip(one, fused_rope(q, k, cos, sin, at[:, :1, :1].expand(3, 3, 10).contiguous(), axes=axes)))
    four = fused_rope(q, k, cos[None, :, None], sin[None, :, None], at, axes=axes)
    assert all(torch.equal(x, y) for x, y in zip(four, want))


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("order,tokens", [("blocks", 6), ("cycle", 6), ("cycle", 6000)])
def test_bad_positions(cuda, pairs, order, tokens):
    """NaN in the columns of the axis alone, the error word's bit, and no read outside the tables."""
    from triton_ops import _lib, fused_qk_norm_rope, fused_rope

    axes = RoPEAxes((8, 12, 12), order)
    q, k, cos, sin, at = make(1, tokens, 8, 2, 64, axes, "f32", "f32")
    good = fused_rope(q, k, cos, sin, at, interleaved=pairs, axes=axes)
    assert _lib.device_error_flags(clear=True) == 0
    bad = at.clone()
    bad[1, 0, 2], bad[2, 0, 4], bad[0, 0, 5] = cos.shape[0], -1, 2**40
    which = torch.tensor(axes.axis_of_pairs(), device="cuda")
    out = fused_rope(q, k, cos, sin, bad, interleaved=pairs, axes=axes)
    assert _lib.device_error_flags(clear=True) == _lib.ERR_BAD_POSITION
    for x, y in zip(out, good):
        for token, axis in ((2, 1), (4, 2), (5, 0)):
            columns = (which == axis).repeat_interleave(2) if pairs else (which == axis).repeat(2)
            assert torch.isnan(x[0, token][:, columns]).all()
            assert torch.equal(x[0, token][:, ~columns], y[0, token][:, ~columns])
        rest = [i for i in range(6) if i not in (2, 4, 5)]
        assert torch.equal(x[0, rest], y[0, rest]) and torch.equal(x[0, 6:], y[0, 6:])
    leaf = q.detach().requires_grad_()
    y, _ = fused_qk_norm_rope(leaf, None, None, None, cos, sin, bad, interleaved=pairs, axes=axes)
    torch.autograd.grad(y.sum(), leaf)
    assert _lib.device_error_flags(clear=True) == _lib.ERR_BAD_POSITION


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sections,order,spectrum", [((16, 24, 24), "blocks", "shared"), ((24, 20, 20), "cycle", "own"),
                                                     ((9, 8), "cycle", "shared"), ((1, 2, 3, 4), "blocks", "own")])
def test_tables(cuda, monkeypatch, sections, order, spectrum, dtype, extension):
    """Rows of several positions hold each pair's column of the rows at one; the count's table serves the gather."""
    from triton_ops import RoPEScaling, _lib, fused_rope, rope_tables

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    axes = RoPEAxes(sections, order, spectrum)
    rot = 2 * sum(sections)
    for scaling in (None, RoPEScaling("linear", 4.0)):
        for shape in ((5,), (2, 33), (0,), (1000,)):
            g = torch.Generator(device="cuda").manual_seed(1)
            at = torch.randint(-50, 100000, (len(sections), *shape), device="cuda", generator=g)
            got = rope_tables(at, rot, 10000.0, scaling, axes=axes, dtype=DT[dtype])
            single = [rope_tables(at[a].contiguous(), rot, 10000.0, scaling, dtype=DT[dtype]) for a in range(len(sections))]
            if spectrum == "own":
                single = [None] * len(sections)
                for a, n in enumerate(sections):
                    single[a] = rope_tables(at[a].contiguous(), 2 * n, 10000.0, scaling, dtype=DT[dtype])
            which, seen = axes.axis_of_pairs(), [0] * len(sections)
            for t in (0, 1):
                seen = [0] * len(sections)
                for i, a in enumerate(which):
                    column = seen[a] if spectrum == "own" else i
                    seen[a] += 1
                    assert torch.equal(got[t][..., i], single[a][t][..., column])
                    assert torch.equal(got[t][..., i + rot // 2], got[t][..., i])
                assert got[t].shape == (*shape, rot)
    # the two ways to the same rotation
    at = torch.randint(64, (len(sections), 2, 9), device="cuda")
    q = randn((2, 9, 3, rot), "f32", 3)
    rows = rope_tables(at, rot, axes=axes)
    one = fused_rope(q, None, *rope_tables(64, rot, axes=axes), at, axes=axes)[0]  # halves: the same bits
    other = fused_rope(q.view(18, 3, rot), None, *(t.view(18, rot) for t in rows))[0]
    assert torch.equal(one, other.view_as(one))


def test_module_streams_and_graphs(cuda):
    from triton_ops import FusedQKNormRoPE

    axes = RoPEAxes((8, 12, 12), "cycle")
    m = FusedQKNormRoPE(64, axes=axes).cuda()
    q, k, cos, sin, at = make(2, 50, 4, 2, 64, axes, "bf16", "f32")

    def step(q, k, at):
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        out = m(*leaves, cos, sin, at)
        return (*out, *torch.autograd.grad(out, [*leaves, m.q_weight, m.k_weight], [q.detach(), k.detach()]))

    other = make(2, 50, 4, 2, 64, axes, "bf16", "f32", seed=30)
    plain = [[t.detach() for t in step(*v)] for v in ((q, k, at), (other[0], other[1], other[4]))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = [t.clone() for t in (q, k, at)]
    with torch.cuda.stream(side):
        step(*static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(*static)
    for values, want in (((other[0], other[1], other[4]), plain[1]), ((q, k, at), plain[0])):
        for a, b in zip(static, values):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_rotation_differentiates_twice(cuda):
    from triton_ops import fused_rope

    axes = RoPEAxes((8, 12, 12))
    q, _, cos, sin, at = make(1, 4, 2, 1, 64, axes, "f32", "f32")
    x = q.detach().requires_grad_()
    y, _ = fused_rope(x, None, cos, sin, at, axes=axes)
    way = randn(y.shape, "f32", 5).requires_grad_()
    (dx,) = torch.autograd.grad(y, x, way, create_graph=True)
    v = randn(y.shape, "f32", 6)
    (back,) = torch.autograd.grad(dx, way, v)
    assert torch.equal(back, fused_rope(v, None, cos, sin, at, axes=axes)[0])


def test_refusals(cuda):
    from triton_ops import fused_qk_norm_rope, fused_rope, rope_tables
    from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

    axes = RoPEAxes((8, 12, 12))
    q, k, cos, sin, at = make(2, 3, 4, 2, 64, axes, "f32", "f32")
    for more, error in [
        (dict(positions=None), ValueError),
        (dict(positions=at[:2]), ShapeMismatchError),
        (dict(positions=at[0]), ShapeMismatchError),
        (dict(positions=at[:, :, :2]), ShapeMismatchError),
        (dict(positions=at.float()), UnsupportedDtypeError),
        (dict(positions=at.cpu()), DeviceError),
        (dict(axes=RoPEAxes((8, 8, 8))), ShapeMismatchError),
        (dict(axes=(8, 12, 12)), TypeError),
        (dict(axes=None), ShapeMismatchError),
    ]:
        for op in (fused_rope, lambda q, k, *a, **m: fused_qk_norm_rope(q, k, None, None, *a, **m)):
            with pytest.raises(error):
                op(q, k, cos, sin, **{"positions": at, "axes": axes, **more})
    with pytest.raises(ShapeMismatchError):
        rope_tables(at[:2], 64, axes=axes)
    with pytest.raises(ShapeMismatchError):
        rope_tables(at, 48, axes=axes)
    with pytest.raises(DeviceError):
        rope_tables(at.cpu(), 64, axes=axes)
