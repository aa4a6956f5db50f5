"""The modules with dropout on the GPU: which masks their calls draw, recomputed and captured ones among them."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from triton_ops import FusedDropout, FusedResidualRMSNorm

pytestmark = pytest.mark.gpu


def randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("reentrant", [True, False])
def test_gradients_under_checkpointing(cuda, reentrant):
    """Bit for bit those without it, for two steps, with parameters between the modules."""
    first, second, drop = FusedResidualRMSNorm(256, branch_norm=True, dropout=0.1), FusedResidualRMSNorm(256, dropout=0.4), FusedDropout(0.5)
    modules = torch.nn.ModuleList([first, second, drop]).cuda()

    def call(x, stream):
        h, y = first(x, stream)
        h, y = second(y, h)
        return drop(y, h)

    def passes(apply):
        torch.manual_seed(3)
        leaves = [randn((2, 40, 256), i).requires_grad_() for i in (1, 2)]
        outs = []
        for _ in range(2):
            out = apply(*leaves)
            out.float().square().sum().backward()
            outs += [out.detach(), *(t.grad.clone() for t in (*leaves, *modules.parameters()))]
        modules.zero_grad()
        return outs

    want = passes(call)
    assert all(torch.equal(a, b) for a, b in zip(passes(call), want))
    assert all(torch.equal(a, b) for a, b in zip(passes(lambda *t: checkpoint(call, *t, use_reentrant=reentrant)), want))
    assert not torch.equal(want[0], want[len(want) // 2])


@pytest.mark.parametrize("reentrant", [True, False])
def test_numbered_masks_refuse_recomputation(cuda, reentrant):
    x = randn((4, 64), 1).requires_grad_()
    m, n = FusedDropout(0.5, seed=0).cuda(), FusedResidualRMSNorm(64, dropout=0.5, dropout_seed=0).cuda()
    for call in (m, lambda t: n(t, t)[1]):
        out = checkpoint(call, x, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="seed"):
            out.float().square().sum().backward()
    (g,) = torch.autograd.grad(m(x).sum(), x)  # without recomputation as before
    assert torch.isfinite(g).all() and m.seed.item() == 2


def test_masks_of_modules_and_calls(cuda):
    x = torch.ones(512, 512, device="cuda")

    def masks():
        modules = [FusedDropout(0.5).cuda(), FusedDropout(0.5).cuda()]
        res = [FusedResidualRMSNorm(512, dropout=0.5).cuda() for _ in range(2)]
        zero = torch.zeros_like(x)
        return [m != 0 for _ in range(2) for m in (*(d(x) for d in modules), *(r(x, zero)[0] for r in res))]

    torch.manual_seed(5)
    drawn = masks()
    for i, a in enumerate(drawn):
        for b in drawn[:i]:
            # 2^18 fair coins twice: five standard deviations
            assert abs((a == b).float().mean().item() - 0.5) < 5 * 0.5 / 512
    torch.manual_seed(5)
    assert all(torch.equal(a, b) for a, b in zip(drawn, masks()))


def test_captured_steps_draw_anew(cuda):
    """Every replay drops other elements, in the forward pass and in its gradient the same ones, and goes on from torch's seed."""
    m, n = FusedDropout(0.5).cuda(), FusedResidualRMSNorm(64, dropout=0.5).cuda()
    x = torch.ones(64, 64, device="cuda", requires_grad=True)
    zero = torch.zeros(64, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out, h = m(x), n(x, zero)[0]
        return out, h, torch.autograd.grad(out.sum(), x)[0], torch.autograd.grad(h.sum(), x)[0]

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()

    def replays(count=3):
        torch.manual_seed(11)
        seen = []
        for _ in range(count):
            graph.replay()
            torch.cuda.synchronize()
            out, h, dout, dh = (t.detach().clone() for t in captured)
            assert torch.equal(out != 0, dout != 0) and torch.equal(h != 0, dh != 0)
            seen += [out != 0, h != 0]
        return seen

    seen = replays()
    for i, a in enumerate(seen):
        for b in seen[:i]:
            assert abs((a == b).float().mean().item() - 0.5) < 5 * 0.5 / 64
    assert all(torch.equal(a, b) for a, b in zip(replays(), seen))
