"""fused_dropout on the GPU: what is dropped, values, gradients and refusals.

The mask is exact (whole numbers). A kept value is x / (1 - p) with the factor
rounded to fp32 and, with a residual, one multiply-add: 2^-23 of the product
beside the result's own rounding.
"""

import math

import pytest
import torch

from triton_ops.kernels.dropout import dropout_keep_reference

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}


def check(got, ref, slack, what=""):
    assert got.shape == ref.shape
    over = (got.double() - ref).abs() - ((ref.abs() + slack) * torch.finfo(got.dtype).eps / 2 * 1.01 + TINY[got.dtype] + slack)
    assert over.numel() == 0 or over.max().item() <= 0, what


def randn(shape, dtype, seed, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(math.prod(shape) + offset, device="cuda", generator=g).to(DT[dtype])[offset:].view(shape)


def test_known_words(cuda):
    """The generator's published answer for a counter and key of zeros: 6627e8d5 e169c58d bc57ac4c 9b00dbd8."""
    words = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    for i, w in enumerate(words):
        assert dropout_keep_reference((4,), w / 2**32, 0)[i] and not dropout_keep_reference((4,), (w + 1) / 2**32, 0)[i]


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("dtype,stream", [("f16", None), ("bf16", None), ("f32", None), ("f16", "f16"), ("bf16", "f32"),
                                          ("f16", "f32"), ("f32", "f32"), ("bf16", "bf16")])
def test_values_and_gradients(cuda, monkeypatch, dtype, stream, extension):
    from triton_ops import _lib, fused_dropout

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    for shape, offset in (((1,), 0), ((3,), 0), ((8,), 1), ((5, 7, 11), 0), ((64, 4096), 0), ((64, 4096), 3), ((1999, 1001), 0)):
        for p, seed, at in ((0.1, 5, 0), (0.5, 2**63 + 9, 2**40 + 1), (0.999, -3, 2**64 - 1)):
            x = randn(shape, dtype, 1, offset).requires_grad_()
            res = None if stream is None else randn(shape, stream, 2, offset).requires_grad_()
            g = randn(shape, stream or dtype, 3, offset)
            keep = dropout_keep_reference(shape, p, seed, at, "cuda")
            u = torch.where(keep, x.detach().double() / (1 - p), 0.0)
            given = torch.tensor(seed if seed < 2**63 else seed - 2**64, device="cuda") if at else seed
            out = fused_dropout(x, p, given, offset=at, residual=res)
            assert out.dtype == (x if res is None else res).dtype and out.is_contiguous()
            check(out, u if res is None else u + res.detach().double(), 2.0**-23 * u.abs())
            if res is None:
                assert torch.equal(out != 0, keep & (x != 0) & (out != 0)) and (out[~keep] == 0).all()
            grads = torch.autograd.grad(out, [x] if res is None else [x, res], g)
            dx = torch.where(keep, g.double() / (1 - p), 0.0)
            assert grads[0].dtype == x.dtype
            check(grads[0], dx, 2.0**-23 * dx.abs())
            if res is not None:
                assert torch.equal(grads[1], g)
            with torch.no_grad():
                assert torch.equal(fused_dropout(x, p, given, offset=at, residual=res), out)


def test_probabilities_at_the_borders(cuda):
    from triton_ops import fused_dropout

    x = randn((5, 99), "f32", 1)
    res = randn((5, 99), "f32", 2)
    assert torch.equal(fused_dropout(x, 0.0), x) and torch.equal(fused_dropout(x, 0, residual=res), x + res)
    bad = x.clone()
    bad[0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    for p in (1.0, 1, 1 - 2.0**-40):
        assert (fused_dropout(bad, p, 3) == 0).all() and torch.equal(fused_dropout(bad, p, 3, residual=res), res)
        leaf = bad.clone().requires_grad_()
        (g,) = torch.autograd.grad(fused_dropout(leaf, p, 3), leaf, bad)
        assert (g == 0).all()
    assert torch.equal(fused_dropout(x, 2.0**-40, 3), x)  # rounds to no element dropped


def test_share_that_is_kept(cuda):
    """Within five standard deviations, for two seeds and offsets, and the masks are independent of one another."""
    from triton_ops import fused_dropout

    n, p = 1 << 22, 0.3
    x = torch.ones(n, device="cuda")
    masks = [fused_dropout(x, p, seed, offset=at) != 0 for seed, at in ((1, 0), (2, 0), (1, 1), (1 + 2**32, 0))]
    for m in masks:
        assert abs(m.float().mean().item() - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)
    both = (1 - p) ** 2
    for i in range(4):
        for j in range(i):
            assert abs((masks[i] & masks[j]).float().mean().item() - both) < 5 * math.sqrt(both * (1 - both) / n)


def test_strides_and_empty(cuda):
    from triton_ops import fused_dropout

    x = randn((6, 10, 8), "bf16", 1)
    for v, r in ((x.transpose(0, 1), None), (x[:, ::2], x[:, 1::2]), (x[:1].expand(6, 10, 8), x.transpose(0, 1).reshape(6, 10, 8))):
        leaf = v.detach().requires_grad_()
        out = fused_dropout(leaf, 0.3, 4, residual=r)
        assert torch.equal(out, fused_dropout(v.contiguous(), 0.3, 4, residual=None if r is None else r.contiguous()))
        (g,) = torch.autograd.grad(out.float().sum(), leaf)
        assert torch.equal(g, fused_dropout(torch.ones_like(v).contiguous(), 0.3, 4))
    for shape in ((0,), (3, 0, 2)):
        leaf = torch.empty(shape, device="cuda", requires_grad=True)
        out = fused_dropout(leaf, 0.3, 4)
        assert out.shape == shape and torch.autograd.grad(out.sum(), leaf)[0].shape == shape


@pytest.mark.parametrize("extension", [True, False])
def test_gradients_of_gradients(cuda, monkeypatch, extension):
    """Dropout is linear: its gradient is differentiable as often as wanted."""
    from triton_ops import _lib, fused_dropout

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    for dtype, stream in (("f32", "f32"), ("bf16", "f32"), ("f16", "f16")):
        x = randn((4, 33), dtype, 1).requires_grad_()
        res = randn((4, 33), stream, 2)
        way = randn((4, 33), stream, 3).requires_grad_()
        keep = dropout_keep_reference((4, 33), 0.5, 9, 0, "cuda")
        (dx,) = torch.autograd.grad(fused_dropout(x, 0.5, 9, residual=res), x, way, create_graph=True)
        second = randn((4, 33), dtype, 4)
        (dway,) = torch.autograd.grad(dx, way, second)
        assert dway.dtype == way.dtype and torch.equal(dway.float(), torch.where(keep, 2 * second.float(), 0.0))


def test_large_indexes(cuda):
    """Past 2^32 elements and counters of 2^30: the mask at the far end."""
    from triton_ops import fused_dropout

    n = 2**32 + 40
    x = torch.ones(n, device="cuda", dtype=torch.float16)
    out = fused_dropout(x, 0.5, 77)
    del x
    low = 0xFFFFFFFF
    for first in (0, 2**31 - 8, 2**32 - 16, 2**32, n - 24):
        # the same words by hand for the 24 elements from there
        a = [((first + i) // 4) & low for i in range(24)]
        for i in range(24):
            words, key = [a[i], ((first + i) // 4) >> 32, 0, 0], [77, 0]
            for _ in range(10):
                even, odd = words[0] * 0xD2511F53, words[2] * 0xCD9E8D57
                words = [(odd >> 32) ^ words[1] ^ key[0], odd & low, (even >> 32) ^ words[3] ^ key[1], even & low]
                key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
            assert (out[first + i].item() != 0) == (words[(first + i) % 4] >= 2**31), first + i


def test_module_and_graph(cuda):
    """A captured training step drops other elements with each replay, and the gradient the same ones."""
    from triton_ops import FusedDropout, fused_dropout

    m = FusedDropout(0.5, seed=4).cuda()
    x = randn((64, 64), "f32", 1).requires_grad_()
    m.eval()
    assert m(x) is x and torch.equal(m(x, x), x + x)
    m.train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out = m(x)
        return out, torch.autograd.grad(out.sum(), x)[0]

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, dx = step()
    for i in range(3):
        at = m.seed.item()
        graph.replay()
        torch.cuda.synchronize()
        assert m.seed.item() == at + 1
        assert torch.equal(out, fused_dropout(x.detach(), 0.5, at)) and torch.equal(dx != 0, out != 0)


def test_refusals(cuda):
    from torch.autograd import forward_ad

    from triton_ops import FusedDropout, fused_dropout
    from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError

    x = randn((4, 8), "bf16", 1)
    for args, more, error in [
        ((x.cpu(), 0.1, 1), {}, DeviceError),
        ((x.double(), 0.1, 1), {}, UnsupportedDtypeError),
        ((x.to(torch.int32), 0.1, 1), {}, UnsupportedDtypeError),
        ((x, -0.1, 1), {}, ValueError),
        ((x, 1.1, 1), {}, ValueError),
        ((x, float("nan"), 1), {}, ValueError),
        ((x, 0.1), {}, ValueError),
        ((x, 0.1, "1"), {}, TypeError),
        ((x, 0.1, True), {}, TypeError),
        ((x, 0.1, torch.tensor([1])), {}, DeviceError),
        ((x, 0.1, torch.tensor([1.0], device="cuda")), {}, UnsupportedDtypeError),
        ((x, 0.1, torch.tensor([1, 2], device="cuda")), {}, ShapeMismatchError),
        ((x, 0.1, 1), dict(offset=-1), ValueError),
        ((x, 0.1, 1), dict(offset=2**64), ValueError),
        ((x, 0.1, 1), dict(residual=x.half()), UnsupportedDtypeError),
        ((x.float(), 0.1, 1), dict(residual=x), UnsupportedDtypeError),
        ((x, 0.1, 1), dict(residual=x[:2]), ShapeMismatchError),
        ((x, 0.1, 1), dict(residual=x.cpu()), DeviceError),
    ]:
        with pytest.raises(error):
            fused_dropout(*args, **more)
    with pytest.raises(ValueError):
        FusedDropout(1.5)
    with forward_ad.dual_level():
        with pytest.raises((ValueError, NotImplementedError, RuntimeError)):
            fused_dropout(forward_ad.make_dual(x.float(), x.float()), 0.1, 1)
