"""Device memory of the rotation by several axes: the outputs, and joined table rows only where the call makes them."""

import pytest
import torch

from triton_ops import RoPEAxes, _lib, fused_qk_norm_rope, fused_rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("sections,order,tokens,joined", [
    ((16, 24, 24), "blocks", 20000, False), ((24, 20, 20), "cycle", 64, False), ((24, 20, 20), "cycle", 20000, True),
])
def test_allocated(cuda, monkeypatch, extension, sections, order, tokens, joined):
    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    axes = RoPEAxes(sections, order)
    q, k = (torch.randn(1, tokens, h, 128, device="cuda").bfloat16().requires_grad_() for h in (8, 2))
    cos, sin = torch.rand(2, 96, 128, device="cuda")
    at = torch.randint(96, (3, 1, tokens), device="cuda")

    heads = 2 * q.numel() + 2 * k.numel()
    rows = 2 * tokens * 64 * 4 if joined else 0

    def allocated(call):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["requested_bytes.all.allocated"]
        out = call()
        return torch.cuda.memory_stats()["requested_bytes.all.allocated"] - before, out

    for op in (lambda: fused_rope(q, k, cos, sin, at, axes=axes),
               lambda: fused_qk_norm_rope(q, k, None, None, cos, sin, at, axes=axes)):
        size, out = allocated(op)
        assert size == heads + rows
        given = [t.detach() for t in out]
        size, _ = allocated(lambda: torch.autograd.grad(out, [q, k], given, retain_graph=True))
        assert size == heads + rows
