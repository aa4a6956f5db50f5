"""rope_tables, fused_rope and fused_qk_norm_rope on the GPU: torch's default device, derivatives, small angles."""

import math
from fractions import Fraction

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extension", [True, False])
def test_tables_under_a_default_device(cuda, monkeypatch, extension):
    """The frequencies are read on the host, also when the first call with them comes under another default device."""
    from triton_ops import RoPEScaling, _lib, rope_tables

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    at = torch.tensor([0, 1, 77, 4096], device="cuda")
    base = 4321.0 + extension  # a key of its own
    for scaling in (None, RoPEScaling("yarn", 4.0, 2048)):
        with torch.device("cuda"):
            inside = [*rope_tables(at, 48, base, scaling), *rope_tables(5, 48, base, scaling)]
        outside = [*rope_tables(at, 48, base, scaling), *rope_tables(5, 48, base, scaling)]
        assert all(torch.equal(a, b) for a, b in zip(inside, outside))
        assert torch.equal(inside[2][0], inside[0][0]) and inside[2].device == at.device


def test_the_extension_takes_frequencies_from_the_host_alone(cuda):
    from triton_ops import _lib

    at = torch.arange(3, device="cuda")
    turns = torch.rand(4, dtype=torch.float64)
    assert _lib.ext().rope_tables(at, turns, 1.0, _lib.F32) is not None
    for other in (turns.cuda(), turns.float(), torch.rand(8, dtype=torch.float64)[::2]):
        assert _lib.ext().rope_tables(at, other, 1.0, _lib.F32) is None


@pytest.mark.parametrize("extension", [True, False])
def test_forward_mode_is_refused(cuda, monkeypatch, extension):
    """No output without its tangent, on either path."""
    from triton_ops import _lib, fused_lora, fused_qk_norm_rope, fused_rope

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    q, k, t, w = (torch.ones(s, device="cuda") for s in ((2, 4, 3, 8), (2, 4, 1, 8), (4, 8), (8,)))
    x, a, b, scaling, base = (torch.ones(s, device="cuda") for s in ((3, 8), (2, 4, 8), (2, 6, 4), (2,), (3, 6)))
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    for op, args in (
        (lambda q, k, c, s: fused_rope(q, k, c, s), (q, k, t, t)),
        (lambda q, k, c, s, v, w: fused_qk_norm_rope(q, k, v, w, c, s), (q, k, t, t, w, w)),
        (lambda x, a, b, s, y: fused_lora(x, a, b, ids, s, base=y), (x, a, b, scaling, base)),
        (lambda y: fused_lora(x, a, b, ids, scaling, out=y), (base,)),
    ):
        op(*args)
        with forward_ad.dual_level():
            for i in range(len(args)):
                dual = forward_ad.make_dual(args[i].clone(), torch.ones_like(args[i]))
                with pytest.raises(ValueError, match="tangent"):
                    op(*args[:i], dual, *args[i + 1:])
            op(*args)


@pytest.mark.parametrize("extension", [True, False])
def test_forward_mode_over_a_backward_pass_is_refused(cuda, monkeypatch, extension):
    from triton_ops import _lib, fused_qk_norm_rope, fused_rope

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    q, t = torch.ones(2, 4, 3, 8, device="cuda", requires_grad=True), torch.ones(4, 8, device="cuda")
    for y in (fused_rope(q, None, t, t)[0], fused_qk_norm_rope(q, None, None, None, t, t)[0]):
        g = torch.ones_like(y)
        torch.autograd.grad(y, q, g, retain_graph=True)
        with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(y, q, forward_ad.make_dual(g, g))


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("with_graph", [True, False], ids=["g has a graph", "g is plain"])
def test_gradients_made_with_create_graph(cuda, monkeypatch, extension, with_graph):
    """They are the gradients, another part of the graph may be differentiated, and they themselves raise: also where
    the outputs' gradients ask for none, since they depend on q, k and the weights too."""
    from triton_ops import _lib, fused_qk_norm_rope

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, w = (torch.randn(s, device="cuda", generator=gen).requires_grad_() for s in ((1, 5, 3, 16), (1, 5, 1, 16), (16,)))
    angle = torch.randn(5, 8, device="cuda", generator=gen)
    cos, sin = angle.cos().repeat(1, 2), angle.sin().repeat(1, 2)
    g = torch.randn(q.shape, device="cuda", generator=gen).requires_grad_(with_graph)
    y, z = fused_qk_norm_rope(q, k, w, None, cos, sin)
    plain = torch.autograd.grad([y, z], [q, k, w], [g, torch.ones_like(z)], retain_graph=True)
    got = torch.autograd.grad([y, z], [q, k, w], [g, torch.ones_like(z)], create_graph=True)
    assert all(torch.equal(a, b) and b.requires_grad for a, b in zip(plain, got))
    other = torch.randn(7, device="cuda", generator=gen).requires_grad_()
    (first,) = torch.autograd.grad(other.pow(3).sum() + y.sum() * 0, other, create_graph=True)
    assert torch.equal(torch.autograd.grad(first.sum(), other)[0], 6 * other.detach())
    for d in got:
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(d.square().sum() + q.sum(), q, retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            (d.square().sum() + q.square().sum()).backward(retain_graph=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("base, kind, factor", [(10000.0, None, 1.0), (5e5, "wavelength", 8.0), (1e7, "linear", 4.0), (1e6, "yarn", 16.0)])
def test_small_sines_and_cosines_keep_their_bits(cuda, dtype, base, kind, factor):
    """Tables relative to each value, not to the largest: slow pairs have angles of 1e-8 rad, and far positions pass
    close by multiples of a quarter turn.

    Relative bound in units of 2^-24: the remainder of the angle 1 (x cot x and x tan x are below 1 up to an eighth of
    a turn), its series 2, the factor's own rounding 1 and its product 1: 5, taken as 8; then the type's half step.
    Absolute: half a unit of 2^-64 turns at each position, and the fp16 subnormals' half step.
    """
    from triton_ops import RoPEScaling, rope_tables
    from triton_ops.kernels.rope import rope_frequencies

    dt, rot = getattr(torch, dtype), 128
    at = [0, 1, 2, 3, 5, 100, 1023, 4097, 8191, 65537, 131071, 999983, 1000000, 2**31 - 1, -1, -77]
    scaling = None if kind is None else RoPEScaling(kind, factor, 8192)
    cos, sin = (t.cpu() for t in rope_tables(torch.tensor(at, device="cuda"), rot, base, scaling, dtype=dt))
    freq, gain = rope_frequencies(rot, base, scaling)
    want = torch.empty(2, len(at), rot // 2, dtype=torch.float64)
    for j, f in enumerate(freq):
        turns = Fraction(f / (2 * math.pi))
        for i, p in enumerate(at):
            quarters = turns * p * 4
            near = round(quarters)
            r = float(quarters - near) * (math.pi / 2)
            c, s = ((math.cos(r), math.sin(r)), (-math.sin(r), math.cos(r)), (-math.cos(r), -math.sin(r)), (math.sin(r), -math.cos(r)))[near % 4]
            want[0, i, j], want[1, i, j] = gain * c, gain * s
    slack = gain * math.pi * 2.0**-64 * torch.tensor(at).abs().double()[:, None] + (2.0**-25 if dt == torch.float16 else 0.0)
    for got, ref, name in ((cos, want[0], "cos"), (sin, want[1], "sin")):
        assert torch.equal(got[:, : rot // 2], got[:, rot // 2 :])
        over = (got[:, : rot // 2].double() - ref).abs() - ref.abs() * (8 * 2.0**-24 + torch.finfo(dt).eps / 2 * 1.01) - slack
        assert over.max().item() <= 0, f"{name}: {over.max().item():.3e} over the bound"
