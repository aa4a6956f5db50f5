"""Which masks the dropout modules draw, with plain formulas in the kernels' place (no GPU).

What is tested is the modules' own: the seed of each call, under activation checkpointing too.
"""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from triton_ops import FusedDropout, FusedResidualRMSNorm
from triton_ops.kernels import dropout as dropout_module
from triton_ops.kernels import residual as residual_module
from triton_ops.kernels.dropout import dropout_keep_reference
from triton_ops.kernels.residual import residual_rmsnorm_reference


@pytest.fixture
def plain(monkeypatch):
    def dropout(x, p, seed=None, *, offset=0, residual=None):
        out = torch.where(dropout_keep_reference(x.shape, p, int(seed), offset), x / (1 - p), 0.0)
        return out if residual is None else out + residual

    def residual(x, stream, weight=None, gate=None, *, dropout_p=0.0, seed=None, **more):
        keep = dropout_keep_reference(x.shape, dropout_p, int(seed)) if dropout_p else None
        return residual_rmsnorm_reference(x, stream, weight, gate, keep=keep, dropout_p=dropout_p, **more)

    monkeypatch.setattr(dropout_module, "fused_dropout", dropout)
    monkeypatch.setattr(residual_module, "fused_residual_rmsnorm", residual)


def block(first, second):
    def call(x, stream):
        h, y = first(x, stream)
        return second(y, h)

    return call


@pytest.mark.parametrize("reentrant", [True, False])
def test_gradients_under_checkpointing(plain, reentrant):
    """Recomputed in the backward pass the modules draw the masks of the forward pass again."""
    call = block(FusedResidualRMSNorm(16, branch_norm=True, dropout=0.3), FusedDropout(0.5))
    x, stream = (torch.randn(4, 6, 16, generator=torch.Generator().manual_seed(i)) for i in (1, 2))

    def passes(apply):
        torch.manual_seed(3)
        leaves = [t.clone().requires_grad_() for t in (x, stream)]
        outs = []
        for _ in range(2):  # two steps
            out = apply(*leaves)
            outs += [out, *torch.autograd.grad(out.square().sum(), leaves)] if not reentrant else [out]
            if reentrant:
                out.square().sum().backward()
        return [*outs, *(t.grad for t in leaves)] if reentrant else outs

    want = passes(call)
    got = passes(lambda *t: checkpoint(call, *t, use_reentrant=reentrant))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.equal(want[0], want[1 if reentrant else 3])  # the steps drop other elements


def test_masks_of_modules_and_calls(plain):
    x = torch.ones(64, 64)

    def masks(modules, calls=3):
        return [m(x) != 0 for _ in range(calls) for m in modules]

    torch.manual_seed(5)
    drawn = masks([FusedDropout(0.5), FusedDropout(0.5)])
    for i, a in enumerate(drawn):
        for b in drawn[:i]:
            # 4096 fair coins twice: a share of 1/2 that agrees, within five standard deviations
            assert abs((a == b).float().mean().item() - 0.5) < 5 * 0.5 / 64
    torch.manual_seed(5)
    assert all(torch.equal(a, b) for a, b in zip(drawn, masks([FusedDropout(0.5), FusedDropout(0.5)])))
    torch.manual_seed(6)
    assert not torch.equal(drawn[0], masks([FusedDropout(0.5)])[0])


def test_numbered_masks(plain):
    """With a seed given the calls are numbered from it, whatever torch's generators do."""
    m = FusedDropout(0.5, seed=7)
    x = torch.ones(8, 8)
    for i in range(3):
        torch.manual_seed(i)
        state = torch.get_rng_state()
        assert torch.equal(m(x) != 0, dropout_keep_reference((8, 8), 0.5, 7 + i)) and m.seed.item() == 8 + i
        assert torch.equal(torch.get_rng_state(), state)
    assert torch.equal(m.next_seed(), torch.tensor([10])) and m.seed.item() == 11
    n = FusedResidualRMSNorm(8, dropout=0.5, dropout_seed=7)
    h, _ = n(x, torch.zeros_like(x))
    assert torch.equal(h != 0, dropout_keep_reference((8, 8), 0.5, 7)) and n.seed.item() == 8
    n.load_state_dict(m.state_dict(), strict=False)
    assert n.seed.item() == 11


@pytest.mark.parametrize("reentrant", [True, False])
def test_numbered_masks_refuse_recomputation(plain, reentrant):
    """The number of a call is not known again in the backward pass: an error instead of another mask's gradients."""
    x = torch.randn(4, 8, requires_grad=True)
    for call in (FusedDropout(0.5, seed=0), lambda t, m=FusedResidualRMSNorm(8, dropout=0.5, dropout_seed=0): m(t, t)[1]):
        out = checkpoint(call, x, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="seed"):
            out.square().sum().backward()


def test_evaluation_draws_nothing(plain):
    x = torch.randn(4, 8)
    state = torch.get_rng_state()
    assert FusedDropout(0.5).eval()(x) is x and FusedDropout(0.0)(x) is x
    FusedResidualRMSNorm(8, dropout=0.5).eval()(x, x)
    FusedResidualRMSNorm(8)(x, x)
    assert torch.equal(torch.get_rng_state(), state)
