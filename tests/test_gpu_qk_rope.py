"""rope_tables, fused_rope and fused_qk_norm_rope on the GPU against plain formulas in 64 bits.

Error bounds, from the kernels' fp32 arithmetic on the given inputs (one fp32
rounding is 2^-24 relative, the result's own rounding eps/2 of its type):

* rotation: two products and a sum, 2^-23 (|u c| + |v s|)
* norm: a head's sum of squares is at most 32 sequential and 5 tree additions
  of positive terms, halved by the root, rsqrtf is within 2 ulp: below 2^-19;
  with the products below 2^-18 of the rotated terms' magnitudes
* gradient of the norm: three factors 1/rms and a dot product: 2^-17 of the
  magnitudes that are added up; its weight sums add at most 64 roundings
* tables: the angle's fraction is exact and rounded once to fp32 (pi 2^-25), sincospif is
  within 2 ulp, the factor's product adds 2^-23: below 2^-21 of the factor
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}


def rounding(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) * 1.01 + TINY[dtype]


def check(got, ref, slack, what):
    """|got - ref| <= the result's rounding + slack, NaN and infinity in the same places."""
    assert got.shape == ref.shape, what
    g = got.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), what
    assert torch.equal(g[~fine].nan_to_num(0.5), ref[~fine].nan_to_num(0.5)), what
    bound = rounding(ref, got.dtype) + slack
    over = ((g - ref).abs() - bound)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {over.max().item():.3e} over the bound"


def table(rows, rot, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 2 * math.pi
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()


def rotate64(x, cos, sin, at, pairs, inverse=False, magnitude=False):
    """The rotation in 64 bits, or the sum of its terms' magnitudes."""
    rot = cos.shape[-1]
    c, s = (t.double()[at][..., None, : rot // 2] for t in (cos, sin))
    if inverse:
        s = -s
    u, v = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., : rot // 2], x[..., rot // 2:rot])
    if magnitude:
        u, v, c, s = u.abs(), v.abs(), c.abs(), s.abs()
        y = u * c + v * s, u * s + v * c
        tail = x[..., rot:].abs()
    else:
        y = u * c - v * s, u * s + v * c
        tail = x[..., rot:]
    y = torch.stack(y, -1).flatten(-2) if pairs else torch.cat(y, -1)
    return torch.cat([y, tail], -1)


def norm64(x, w, eps):
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    return x * r * w, r


def positions_of(x, positions):
    return torch.arange(x.shape[-3], device="cuda") if positions is None else positions.long()


def grads64(x, w, g, cos, sin, at, pairs, eps):
    """dx and dw in 64 bits, and the magnitudes that their sums add up."""
    d = x.shape[-1]
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    b = rotate64(g, cos, sin, at, pairs, inverse=True)
    m = rotate64(g, cos, sin, at, pairs, inverse=True, magnitude=True)
    dx = r * b * w - x * r**3 * (b * w * x).sum(-1, keepdim=True) / d
    dx_m = r * m * w.abs() + x.abs() * r**3 * (m * w.abs() * x.abs()).sum(-1, keepdim=True) / d
    over = tuple(range(x.dim() - 1))
    return dx, dx_m, (b * x * r).sum(over), (m * x.abs() * r).sum(over)


def heads(shape, dtype, seed, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = math.prod(shape)
    flat = torch.randn(n + offset, device="cuda", generator=g).to(DT[dtype])
    return flat[offset:].view(shape)


# batch, seq, q heads, k heads, head_dim, rotary_dim, pairs, dtype, table dtype, positions
CASES = [
    (1, 1, 1, 1, 2, 2, False, "f32", "f32", None),
    (1, 1, 32, 8, 128, 128, False, "bf16", "f32", "given"),
    (2, 5, 3, 1, 64, 64, True, "f16", "f16", None),
    (3, 7, 4, 2, 128, 64, False, "bf16", "bf16", "given"),
    (1, 33, 5, 5, 80, 80, False, "f16", "f32", "given"),
    (1, 9, 5, 1, 80, 40, False, "f16", "f32", None),     # half = 20: 8-byte vectors
    (2, 3, 2, 1, 96, 48, True, "bf16", "f32", "shared"),
    (1, 4, 3, 2, 72, 72, True, "f32", "f32", None),
    (1, 4, 3, 2, 72, 12, True, "f16", "f16", None),      # a lane with one rotated vector of two
    (1, 6, 2, 2, 36, 34, False, "f16", "bf16", "given"),  # no vector width fits
    (2, 2, 2, 1, 7, 6, True, "f32", "f16", None),        # odd head width
    (1, 3, 2, 1, 256, 256, False, "f32", "f32", None),
    (1, 3, 2, 1, 512, 512, False, "bf16", "f32", None),
    (1, 2, 1, 1, 1024, 1000, True, "f16", "f32", None),   # wider than a warp's vectors
    (4, 700, 8, 2, 64, 64, False, "bf16", "f32", None),
    (1, 1500, 7, 3, 32, 16, True, "f32", "f32", "given"),
    # enough tokens for four heads per group, then for the streaming kernel
    (1, 2500, 8, 2, 128, 128, False, "bf16", "f32", "given"),
    (3, 901, 5, 1, 128, 64, True, "f16", "f16", "shared"),
    (2, 3001, 8, 3, 128, 128, False, "bf16", "bf16", "given"),
    (1, 6100, 13, 3, 80, 80, False, "f16", "f32", None),   # five lanes a head, six heads a warp
    (1, 6100, 9, 5, 64, 24, True, "f16", "f32", "given"),
    (2, 3500, 6, 2, 80, 40, False, "bf16", "f32", None),   # ten lanes of 8-byte vectors
    (1, 4100, 4, 1, 256, 64, False, "f32", "f32", "given"),
]


def make(case, seed=0, offset=0):
    b, s, hq, hk, d, rot, pairs, dt, ct, pos = case
    q = heads((b, s, hq, d), dt, seed + 2, offset)
    k = heads((b, s, hk, d), dt, seed + 3, offset)
    rows = s if pos is None else s + 50
    cos, sin = table(rows, rot, DT[ct])
    g = torch.Generator(device="cuda").manual_seed(seed + 4)
    positions = None
    if pos == "given":
        positions = torch.randint(rows, (b, s), device="cuda", generator=g)
    elif pos == "shared":
        positions = torch.randint(rows, (s,), device="cuda", generator=g, dtype=torch.int32)
    return q, k, cos, sin, positions, pairs


@pytest.mark.parametrize("case", CASES, ids=str)
def test_rope(cuda, case):
    from triton_ops import fused_rope

    q, k, cos, sin, positions, pairs = make(case)
    out = fused_rope(q, k, cos, sin, positions, interleaved=pairs)
    for x, y in zip((q, k), out):
        at = positions_of(x, positions)
        ref = rotate64(x.double(), cos, sin, at, pairs)
        check(y, ref, 2.0**-23 * rotate64(x.double(), cos, sin, at, pairs, magnitude=True), str(case))
    rot = cos.shape[1]
    assert torch.equal(out[0][..., rot:], q[..., rot:])  # copied bit for bit
    alone, none = fused_rope(q, None, cos, sin, positions, interleaved=pairs)
    assert none is None and torch.equal(alone, out[0])


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("wd", ["f32", "bf16", None])
def test_qk_norm_rope(cuda, case, wd):
    from triton_ops import fused_qk_norm_rope

    q, k, cos, sin, positions, pairs = make(case, 10)
    d, eps = q.shape[-1], 1e-5
    wq, wk = ((1 + 0.3 * heads((d,), "f32", s)).to(DT[wd]) for s in (7, 8)) if wd else (None, None)
    out = fused_qk_norm_rope(q, k, wq, wk, cos, sin, positions, eps, interleaved=pairs)
    for x, w, y in zip((q, k), (wq, wk), out):
        at = positions_of(x, positions)
        u, _ = norm64(x.double(), w.double() if wd else torch.ones(d, device="cuda", dtype=torch.float64), eps)
        check(y, rotate64(u, cos, sin, at, pairs), 2.0**-18 * rotate64(u, cos, sin, at, pairs, magnitude=True), str(case))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_rope_gradient(cuda, case):
    from triton_ops import fused_rope

    q, k, cos, sin, positions, pairs = make(case, 20)
    q.requires_grad_()
    k.requires_grad_()
    out = fused_rope(q, k, cos, sin, positions, interleaved=pairs)
    gq, gk = heads(q.shape, case[7], 31), heads(k.shape, case[7], 32)
    dq, dk = torch.autograd.grad(out, [q, k], [gq, gk])
    for x, g, d in ((q, gq, dq), (k, gk, dk)):
        at = positions_of(x, positions)
        check(d, rotate64(g.double(), cos, sin, at, pairs, inverse=True),
              2.0**-23 * rotate64(g.double(), cos, sin, at, pairs, magnitude=True), str(case))


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("wd", ["f32", "f16", None])
def test_qk_norm_rope_gradient(cuda, case, wd):
    from triton_ops import fused_qk_norm_rope

    q, k, cos, sin, positions, pairs = make(case, 40)
    d, eps = q.shape[-1], 1e-5
    leaves = [q.requires_grad_(), k.requires_grad_()]
    wq = wk = None
    if wd:
        wq, wk = ((1 + 0.3 * heads((d,), "f32", s)).to(DT[wd]).requires_grad_() for s in (7, 8))
        leaves += [wq, wk]
    out = fused_qk_norm_rope(q, k, wq, wk, cos, sin, positions, eps, interleaved=pairs)
    gq, gk = heads(q.shape, case[7], 51), heads(k.shape, case[7], 52)
    grads = torch.autograd.grad(out, leaves, [gq, gk])
    again = fused_qk_norm_rope(q, k, wq, wk, cos, sin, positions, eps, interleaved=pairs)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again, leaves, [gq, gk])))  # fixed order
    h = 1e-5
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        at = positions_of(x, positions)
        x64, g64 = x.detach().double(), g.double()
        w64 = w.detach().double() if wd else torch.ones(d, device="cuda", dtype=torch.float64)
        dx, dx_m, dw, dw_m = grads64(x64, w64, g64, cos, sin, at, pairs, eps)
        check(grads[i], dx, 2.0**-17 * dx_m, str(case))
        if wd:
            check(grads[2 + i], dw, 2.0**-17 * dw_m, str(case))
        # and against differences of the 64-bit forward along one direction
        step = heads(x.shape, "f32", 60 + i).double()

        def value(t):
            return (rotate64(norm64(t, w64, eps)[0], cos, sin, at, pairs) * g64).sum()

        diff = (value(x64 + h * step) - value(x64 - h * step)) / (2 * h)
        slack = ((2.0**-17 * dx_m + rounding(dx, x.dtype)) * step.abs()).sum()
        # the difference's own error: h^2 times a third derivative of order |g| |w| / rms^3 of small heads
        r = 1 / torch.sqrt(x64.pow(2).mean(-1, keepdim=True) + eps)
        slack += 1e-9 * (1 + (g64.abs() * w64.abs() * r**3 * (1 + step.abs().pow(3).sum(-1, keepdim=True))).sum())
        assert abs((grads[i].double() * step).sum() - diff) <= slack


@pytest.mark.parametrize("offset", [1, 4])
@pytest.mark.parametrize("case", [CASES[1], CASES[4]], ids=str)
def test_unaligned_heads(cuda, case, offset):
    """Views that start off a 16- or 8-byte border give the values of aligned copies."""
    from triton_ops import fused_qk_norm_rope, fused_rope

    q, k, cos, sin, positions, pairs = make(case, 0, offset)
    assert q.data_ptr() % 16 == 2 * offset % 16
    for y, z in zip(fused_rope(q, k, cos, sin, positions), fused_rope(q.clone(), k.clone(), cos, sin, positions)):
        check(y, z.double(), rounding(z.double(), z.dtype) + 2.0**-22 * 8, "rope")  # each side rounds once
    w = 1 + 0.1 * heads((q.shape[-1],), "f32", 3)
    off = torch.cat([w[:1], w])[1:]  # a weight off its border too
    a = fused_qk_norm_rope(q, k, off, w, cos, sin, positions)
    b = fused_qk_norm_rope(q.clone(), k.clone(), w, w, cos, sin, positions)
    for y, z in zip(a, b):
        check(y, z.double(), rounding(z.double(), z.dtype) + 2.0**-17 * 8, "norm")


def test_strided_views(cuda):
    """Queries and keys inside a fused projection, [batch, heads, seq, dim] storage, broadcast tokens."""
    from triton_ops import fused_qk_norm_rope, fused_rope

    b, s, hq, hk, d = 2, 11, 6, 2, 64
    qkv = heads((b, s, hq + 2 * hk, d), "bf16", 1)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    cos, sin = table(s, d, torch.float32)
    w = 1 + 0.1 * heads((d,), "f32", 3)
    dense = (q.contiguous(), k.contiguous())
    for other in (
        (q, k),
        tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)),
        tuple(t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3) for t in (q, k)),
    ):
        assert all(torch.equal(x, y) for x, y in zip(fused_rope(*other, cos, sin), fused_rope(*dense, cos, sin)))
        got = fused_qk_norm_rope(*other, w, w, cos, sin)
        assert all(torch.equal(x, y) for x, y in zip(got, fused_qk_norm_rope(*dense, w, w, cos, sin)))
        assert all(t.is_contiguous() for t in got)
    # one prompt shared by a batch: stride 0, and its gradient is the sum over the batch
    one = heads((1, s, hq, d), "f32", 5).requires_grad_()
    wide = one.expand(3, -1, -1, -1)
    y, _ = fused_qk_norm_rope(wide, None, w, None, cos, sin)
    g = heads(y.shape, "f32", 6)
    (got,) = torch.autograd.grad(y, one, g)
    parts = [grads64(one.detach().double(), w.double(), g[i:i + 1].double(), cos, sin,
                     torch.arange(s, device="cuda"), False, 1e-6) for i in range(3)]
    check(got, sum(p[0] for p in parts), 2.0**-16 * sum(p[1] for p in parts), "shared prompt")
    # flattened tokens and tables as views: row stride above the width, 4-D
    flat = fused_rope(q.reshape(b * s, hq, d), None, cos, sin, torch.arange(s, device="cuda").repeat(b))[0]
    assert torch.equal(flat.view(b, s, hq, d), fused_rope(q, None, cos, sin)[0])
    wide_cos, wide_sin = (torch.cat([t, t], 1)[:, :d] for t in (cos, sin))
    assert wide_cos.stride(0) == 2 * d
    assert torch.equal(fused_rope(q, None, wide_cos, wide_sin)[0], fused_rope(q, None, cos, sin)[0])
    assert torch.equal(fused_rope(q, None, cos[None, :, None], sin[None, :, None])[0], fused_rope(q, None, cos, sin)[0])


def test_gradients_that_are_views(cuda):
    """sum().backward() hands over an expanded gradient; only one output used leaves the other's undefined."""
    from triton_ops import FusedQKNormRoPE, fused_rope

    q, k = heads((2, 3, 4, 64), "f32", 1).requires_grad_(), heads((2, 3, 2, 64), "f32", 2).requires_grad_()
    cos, sin = table(3, 64, torch.float32)
    at = torch.arange(3, device="cuda")
    out, _ = fused_rope(q, k, cos, sin)
    out.sum().backward()
    ones = torch.ones(q.shape, device="cuda", dtype=torch.float64)
    check(q.grad, rotate64(ones, cos, sin, at, False, inverse=True), 2.0**-22, "dq")
    assert k.grad is None or not k.grad.any()
    m = FusedQKNormRoPE(64).cuda()
    assert m.q_weight.dtype == torch.float32 and torch.equal(m.k_weight, torch.ones(64, device="cuda"))
    _, y = m(q, k, cos, sin)
    k.grad = None
    y.transpose(1, 2).pow(2).sum().backward()
    ref = grads64(k.detach().double(), torch.ones(64, device="cuda").double(), 2 * y.detach().double(), cos, sin, at, False, 1e-6)
    check(k.grad, ref[0], 2.0**-16 * ref[1], "dk")
    check(m.k_weight.grad, ref[2], 2.0**-16 * ref[3], "dwk")
    assert m.q_weight.grad is None or not m.q_weight.grad.any()


def test_rope_differentiates_twice_and_the_norm_refuses(cuda):
    from triton_ops import fused_qk_norm_rope, fused_rope

    q = heads((1, 3, 2, 64), "f32", 1).requires_grad_()
    cos, sin = table(3, 64, torch.float32)
    y, _ = fused_rope(q, None, cos, sin)
    g = heads(y.shape, "f32", 2).requires_grad_()
    (dq,) = torch.autograd.grad(y, q, g, create_graph=True)
    v = heads(y.shape, "f32", 3)
    (back,) = torch.autograd.grad(dq, g, v)
    check(back, rotate64(v.double(), cos, sin, torch.arange(3, device="cuda"), False), 2.0**-21, "second")
    y, _ = fused_qk_norm_rope(q, None, None, None, cos, sin)
    with pytest.raises(RuntimeError, match="once|differentiate twice"):
        (dq,) = torch.autograd.grad(y, q, g, create_graph=True)
        dq.sum().backward()


def test_nan_and_infinity_stay_in_their_pairs(cuda):
    from triton_ops import fused_qk_norm_rope, fused_rope

    for pairs in (False, True):
        q = heads((1, 4, 2, 64), "f16", 1)
        q[0, 1, 0, 60] = float("inf")   # not rotated
        q[0, 2, 1, 5] = float("nan")    # rotated
        q[0, 3, 1, 63] = float("-inf")
        cos, sin = table(4, 32, torch.float32)
        at = torch.arange(4, device="cuda")
        y, _ = fused_rope(q, None, cos, sin, interleaved=pairs)
        check(y, rotate64(q.double(), cos, sin, at, pairs), 2.0**-23 * 8, f"pairs={pairs}")
        assert torch.isnan(y).sum() == 2
        z, _ = fused_qk_norm_rope(q, None, None, None, cos, sin, interleaved=pairs)
        u, _ = norm64(q.double(), torch.ones(64, device="cuda", dtype=torch.float64), 1e-6)
        check(z, rotate64(u, cos, sin, at, pairs), 2.0**-18 * 16, f"norm pairs={pairs}")
    zero = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, _ = fused_qk_norm_rope(zero, None, None, None, cos, sin)
    assert not y.any()
    (d,) = torch.autograd.grad(y, zero, torch.ones_like(y))
    ref = grads64(zero.detach().double(), torch.ones(64, device="cuda").double(), torch.ones_like(y).double(), cos, sin, at, False, 1e-6)
    check(d, ref[0], 2.0**-17 * ref[1], "zero head")


def test_positions_outside_the_table(cuda):
    from triton_ops import _lib, fused_qk_norm_rope, fused_rope

    _lib.device_error_flags(clear=True)
    cos, sin = table(10, 32, torch.float32)
    for d in (64, 63):  # the vector and the scalar kernels
        q = heads((1, 5, 2, d), "f32", 1).requires_grad_()
        for op in (lambda p: fused_rope(q, None, cos, sin, p)[0],
                   lambda p: fused_qk_norm_rope(q, None, None, None, cos, sin, p)[0]):
            good = torch.tensor([[0, 9, 3, 3, 9]], device="cuda")
            base = op(good).detach()
            assert _lib.device_error_flags(clear=True) == 0
            for bad in (10, -1, 2**40, -2**62):
                at = good.clone()
                at[0, 2] = bad
                y = op(at)
                assert _lib.device_error_flags(clear=True) == _lib.ERR_BAD_POSITION
                assert torch.isnan(y[0, 2, :, :32]).all()
                assert torch.equal(y[0, 2, :, 32:], base[0, 2, :, 32:])
                keep = [0, 1, 3, 4]
                assert torch.equal(y[0, keep], base[0, keep])
                (g,) = torch.autograd.grad(y, q, torch.ones_like(y))
                assert _lib.device_error_flags(clear=True) == _lib.ERR_BAD_POSITION
                assert torch.isfinite(g[0, keep]).all() and torch.isnan(g[0, 2]).any()


@pytest.mark.parametrize("shape", [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64), (0, 2, 64)])
def test_empty(cuda, shape):
    from triton_ops import fused_qk_norm_rope, fused_rope

    q = torch.empty(shape, device="cuda", requires_grad=True)
    cos, sin = table(4, 64, torch.float32)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, _ = fused_rope(q, None, cos, sin)
    assert y.shape == q.shape
    y, _ = fused_qk_norm_rope(q, None, w, None, cos, sin)
    dq, dw = torch.autograd.grad(y.sum(), [q, w])
    assert dq.shape == q.shape and not dw.any()


def test_keys_without_queries(cuda):
    from triton_ops import fused_qk_norm_rope

    cos, sin = table(4, 64, torch.float32)
    q, k = torch.empty(1, 4, 0, 64, device="cuda"), heads((1, 4, 3, 64), "f32", 1)
    w = (torch.ones(64, device="cuda") * 2).requires_grad_()
    y, z = fused_qk_norm_rope(q, k, w, w, cos, sin)
    assert y.numel() == 0
    u, _ = norm64(k.double(), w.detach().double(), 1e-6)
    check(z.detach(), rotate64(u, cos, sin, torch.arange(4, device="cuda"), False), 2.0**-17 * 8, "k only")
    (dw,) = torch.autograd.grad(z.sum(), w)
    ref = grads64(k.double(), w.detach().double(), torch.ones_like(k).double(), cos, sin, torch.arange(4, device="cuda"), False, 1e-6)
    check(dw, ref[2], 2.0**-17 * ref[3], "dw")


def test_offsets_past_32_bits(cuda):
    """Tokens 2.2e9 elements apart in one 8.8 GB buffer."""
    from triton_ops import fused_qk_norm_rope

    far = 2_200_000_000
    big = torch.empty(2 * far + 256, device="cuda", dtype=torch.bfloat16)
    q = big.as_strided((1, 3, 2, 64), (0, far, 64, 1))
    q.copy_(heads((1, 3, 2, 64), "bf16", 1))
    cos, sin = table(3, 64, torch.float32)
    w = torch.ones(64, device="cuda")
    leaf = q.detach().requires_grad_()
    y, _ = fused_qk_norm_rope(leaf, None, w, None, cos, sin)
    dense = q.clone().requires_grad_()
    z, _ = fused_qk_norm_rope(dense, None, w, None, cos, sin)
    assert torch.equal(y, z)
    g = heads(z.shape, "bf16", 2)
    ref = torch.autograd.grad(z, dense, g)[0]
    # the gradient of a strided leaf is dense here: ask the node itself
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rot", [2, 10, 64, 128, 512])
def test_tables(cuda, dtype, rot):
    from triton_ops import RoPEScaling, rope_tables
    from triton_ops.kernels.rope import rope_frequencies

    scalings = [None, RoPEScaling("linear", 4.0), RoPEScaling("yarn", 16.0, 4096), RoPEScaling("wavelength", 8.0, 8192),
                RoPEScaling("linear", 2.0, attention_factor=0.5)]
    if rot > 2:
        scalings.append(RoPEScaling("ntk", 8.0))
    at = torch.tensor([[0, 1, 7, -3], [4095, 131071, 10**6, 2**31 - 1]], device="cuda")
    for scaling in scalings:
        freq, gain = rope_frequencies(rot, 10000.0, scaling)
        f = torch.tensor(freq, dtype=torch.float64, device="cuda")
        for pos in (at, at.int(), at.t(), 300):
            cos, sin = rope_tables(pos, rot, 10000.0, scaling, dtype=DT[dtype])
            p = pos if isinstance(pos, torch.Tensor) else torch.arange(pos, device="cuda")
            angle = p.double()[..., None] * f
            angle = torch.cat([angle, angle], -1)
            # the 64-bit angle of the oracle is itself off by 2^-53 of its size
            slack = gain * (2.0**-21 + 2.0**-52 * angle.abs())
            check(cos, angle.cos() * gain, slack, f"{scaling} cos")
            check(sin, angle.sin() * gain, slack, f"{scaling} sin")
    assert rope_tables(0, rot)[0].shape == (0, rot)
    assert rope_tables(torch.empty(2, 0, dtype=torch.int64, device="cuda"), rot)[1].shape == (2, 0, rot)


def test_tables_serve_the_row_op(cuda):
    """The tables are those that fused_rmsnorm_rope takes."""
    from triton_ops import fused_rmsnorm_rope, fused_rope, rope_tables

    x = heads((2, 16, 256), "f16", 1)
    cos, sin = rope_tables(16, 64, dtype=torch.float16)
    w = torch.ones(256, device="cuda", dtype=torch.float16)
    y = fused_rmsnorm_rope(x, w, cos, sin)
    u = (x.double() / torch.sqrt(x.double().pow(2).mean(-1, keepdim=True) + 1e-6)).half()
    z, _ = fused_rope(u.view(2, 16, 4, 64), None, cos, sin)
    # u rounds the normed row as the row op does, up to one step where its fp32 row sum decides
    m = rotate64(u.double().view(2, 16, 4, 64), cos, sin, torch.arange(16, device="cuda"), False, magnitude=True)
    check(y.view_as(z), z.double(), 2.0**-9 * m, "row op")


def test_streams_and_graphs(cuda):
    """A side stream, and two captured graphs (forward and backward) replayed on new inputs."""
    from triton_ops import fused_qk_norm_rope, rope_tables

    side = torch.cuda.Stream()
    b, s, hq, hk, d = 1, 40, 4, 2, 64
    at = torch.randint(1000, (b, s), device="cuda")
    torch.cuda.synchronize()

    def step(q, k, w, gq, gk):
        cos, sin = rope_tables(at, d)
        out = fused_qk_norm_rope(q, k, w, w, cos.view(-1, d), sin.view(-1, d), torch.arange(s, device="cuda").expand(b, s))
        return (*out, *torch.autograd.grad(out, [q, k, w], [gq, gk]))

    def inputs(seed):
        return [heads((b, s, hq, d), "bf16", seed), heads((b, s, hk, d), "bf16", seed + 1),
                1 + 0.1 * heads((d,), "f32", seed + 2), heads((b, s, hq, d), "bf16", seed + 3),
                heads((b, s, hk, d), "bf16", seed + 4)]

    def leaves(t):
        return [x.clone().requires_grad_(i < 3) for i, x in enumerate(t)]

    plain = {seed: [t.detach() for t in step(*leaves(inputs(seed)))] for seed in (1, 2, 3)}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = step(*leaves(inputs(1)))
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, plain[1]))
    graphs = []
    for seed in (1, 2):
        static = leaves(inputs(seed))
        with torch.cuda.stream(side):
            step(*static)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(*static)
        graphs.append((graph, static, out))
    for seed in (3, 1, 2):
        new = inputs(seed)
        for graph, static, _ in graphs:
            with torch.no_grad():
                for x, y in zip(static, new):
                    x.copy_(y)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, plain[seed]))


@pytest.mark.parametrize("extension", [True, False])
def test_gradients_of_threads_on_one_stream(cuda, monkeypatch, extension):
    """Gradients of two threads and calls that use scratch memory beside them, all on one stream."""
    import threading

    from triton_ops import _lib, fused_lora, fused_qk_norm_rope

    cos, sin = table(600, 64, torch.float32)
    cases = [(1, 600, 4, 64), (2, 37, 3, 64), (1, 300, 8, 64)]
    tensors = [(heads(s, "bf16", i), 1 + 0.1 * heads((64,), "f32", i + 9), heads(s, "bf16", i + 20))
               for i, s in enumerate(cases)]
    lora = (heads((400, 64), "bf16", 1), heads((3, 8, 64), "bf16", 2), heads((3, 64, 8), "bf16", 3),
            torch.arange(400, device="cuda") % 4 - 1)

    def grads(i):
        q, w, g = tensors[i]
        leaves = [q.clone().requires_grad_(), w.clone().requires_grad_()]
        out, _ = fused_qk_norm_rope(leaves[0], None, leaves[1], None, cos, sin)
        return torch.autograd.grad(out, leaves, g)

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    ref = [grads(i) for i in range(len(cases))]
    lora_ref = fused_lora(*lora)
    wrong, done, start = [], [], threading.Barrier(len(cases) + 1)

    def work(i):
        start.wait(60)
        for _ in range(40):
            if i == len(cases):
                same = torch.equal(fused_lora(*lora), lora_ref)
            else:
                same = all(torch.equal(x, y) for x, y in zip(grads(i), ref[i]))
            if not same:
                wrong.append(i)
        done.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases) + 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(done) == len(threads)


def test_without_the_extension(cuda, monkeypatch):
    """The same kernels through ctypes: the same bits, forward and backward."""
    from triton_ops import _lib, fused_qk_norm_rope, fused_rope, rope_tables

    q, k, cos, sin, positions, pairs = make(CASES[3], 70)
    w = 1 + 0.1 * heads((q.shape[-1],), "f32", 3)

    def everything():
        leaves = [t.clone().requires_grad_() for t in (q, k, w)]
        a = fused_rope(leaves[0], leaves[1], cos, sin, positions, interleaved=pairs)
        b = fused_qk_norm_rope(*leaves, leaves[2], cos, sin, positions, interleaved=pairs)
        ga = torch.autograd.grad(a, leaves[:2], [q, k])
        gb = torch.autograd.grad(b, leaves, [q, k])
        one = fused_qk_norm_rope(leaves[0], None, leaves[2], None, cos, sin, positions)[0]
        return [*a, *b, *ga, *gb, one, *torch.autograd.grad(one, leaves[::2], q), *rope_tables(positions, 64)]

    with_ext = everything()
    monkeypatch.setattr(_lib, "ext", lambda: None)
    assert all(torch.equal(x, y) for x, y in zip(with_ext, everything()))


def test_refusals(cuda):
    from triton_ops import RoPEScaling, fused_qk_norm_rope, fused_rope, rope_tables
    from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

    q = heads((2, 4, 2, 64), "f16", 1)
    cos, sin = table(4, 64, torch.float32)
    for bad, error in (
        ((q.cpu(), None, cos, sin), DeviceError),
        ((q, q.cpu(), cos, sin), DeviceError),
        ((q, None, cos.cpu(), sin), DeviceError),
        ((q.int(), None, cos, sin), UnsupportedDtypeError),
        ((q, q.float(), cos, sin), UnsupportedDtypeError),
        ((q, None, cos.double(), sin.double()), UnsupportedDtypeError),
        ((q, q[:, :3], cos, sin), ShapeMismatchError),
        ((q, q[..., :32], cos, sin), ShapeMismatchError),
        ((q[0, 0], None, cos, sin), ShapeMismatchError),
        ((q, None, cos[:3], sin[:3]), ShapeMismatchError),
        ((q, None, cos, sin[:, :32]), ShapeMismatchError),
        ((q, None, cos[:, :63], sin[:, :63]), ShapeMismatchError),
        ((q[..., :32], None, cos, sin), ShapeMismatchError),
        ((q.transpose(2, 3), None, cos[:, :2], sin[:, :2]), ValueError),
        ((q, None, cos, sin, torch.zeros(2, 4, device="cuda")), UnsupportedDtypeError),
        ((q, None, cos, sin, torch.zeros(2, 5, device="cuda", dtype=torch.int64)), ShapeMismatchError),
        ((q, None, cos, sin, torch.zeros(2, 4, dtype=torch.int64)), DeviceError),
        ((q, None, cos.clone().requires_grad_(), sin), ValueError),
    ):
        with pytest.raises(error):
            fused_rope(*bad)
        with pytest.raises(error):
            fused_qk_norm_rope(bad[0], bad[1], None, None, *bad[2:])
    for w, error in ((torch.ones(63, device="cuda"), ShapeMismatchError), (torch.ones(64), DeviceError),
                     (torch.ones(128, device="cuda")[::2], ValueError), (torch.ones(64, device="cuda").int(), UnsupportedDtypeError)):
        with pytest.raises(error):
            fused_qk_norm_rope(q, q, w, None, cos, sin)
        with pytest.raises(error):
            fused_qk_norm_rope(q, q, None, w, cos, sin)
    with pytest.raises(DeviceError):
        rope_tables(torch.zeros(3, dtype=torch.int64), 64)
    with pytest.raises(DeviceError):
        rope_tables(3, 64, device="cpu")
    with pytest.raises(UnsupportedDtypeError):
        rope_tables(torch.zeros(3, device="cuda"), 64)
    with pytest.raises(UnsupportedDtypeError):
        rope_tables(3, 64, dtype=torch.float64)
    for rot in (0, 3, 514):
        with pytest.raises(ShapeMismatchError):
            rope_tables(3, rot)
    with pytest.raises(ValueError):
        RoPEScaling("yarn", 2.0)
