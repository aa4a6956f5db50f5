"""What fused_lora keeps of its fp32 sums and low-rank values, and what autograd hears of its writes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("rank", [2, 20, 40, 100, 256])
@pytest.mark.parametrize("dtype, bits, t", [("bf16", 24, 3), ("bf16", 24, 300), ("bf16", 16, 500), ("f16", 22, 3), ("f16", 22, 500)])
def test_low_rank_values_keep_their_bits(cuda, dtype, bits, t, rank):
    """Two low-rank values below 2^bits that differ by less than 128, one subtracted from the other.

    Every product, partial sum and result is exact in fp32 and in the operands' type, so the outputs have to be equal.
    A holds a value in four parts of six bits, x the parts' weights. The two values are the first and the last of the
    rank, so that from rank 40 on they enter different tensor instructions."""
    from triton_ops import fused_lora

    g = torch.Generator().manual_seed(rank + t)
    m, k, n = 3, 40, 40
    first = torch.randint(2 ** (bits - 1), 2**bits - 128, (m,), generator=g) | 1
    other = first + torch.randint(1, 128, (m,), generator=g)
    x = torch.zeros(t, k)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 2.0**18, 2.0**12, 2.0**6, 1.0
    scale = 1.0
    if dtype == "f16":  # its largest value is 65504: a sixteenth of everything, and 16 as the adapter's factor
        x /= 16
        scale = 16.0
    a = torch.zeros(m, rank, k)
    for r, v in ((0, first), (rank - 1, other)):
        for i, shift in enumerate((18, 12, 6, 0)):
            a[:, r, i] = (v >> shift) % 64
    b = torch.zeros(m, n, rank)
    b[:, ::2, 0], b[:, ::2, rank - 1] = -1.0, 1.0
    b[:, 1::2, 0], b[:, 1::2, rank - 1] = 1.0, -1.0
    ids = torch.arange(t) % m
    want = (other - first)[ids][:, None].double() * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    x, a, b = (v.to(DT[dtype]).cuda() for v in (x, a, b))
    got = fused_lora(x, a, b, ids.cuda(), torch.full((m,), scale, device="cuda"))
    assert torch.equal(got.double().cpu(), want)


@pytest.mark.parametrize("rank", [8, 64, 128, 256])
@pytest.mark.parametrize("t", [9, 500])
def test_fp32_sums_are_rounded_not_cut(cuda, t, rank):
    """Low-rank values of 4096 positive terms: errors that all have one sign would add up.

    Bound relative to v, in units of 2^-24: the 16 terms of a chunk within one instruction chain, 6 steps of at most
    two units: 12; the chunks of half of K one after the other, each addition off by at most one unit of what is there
    by then, which grows evenly: K / 64; the halves, warps and CTAs: 12 more additions; operands of two tf32 values
    with the smallest product left out: three times 2^-22, 12; the same for v times one: 4 (B is one at one place).
    """
    from triton_ops import fused_lora

    k, n = 4096, 32
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = 0.5 + torch.rand(t, k, device="cuda", generator=g)
    a = 0.5 + torch.rand(1, rank, k, device="cuda", generator=g)
    b = torch.zeros(1, n, rank, device="cuda")
    at = torch.arange(n, device="cuda") * 7 % rank
    b[0, torch.arange(n), at] = 1.0
    got = fused_lora(x, a, b, torch.zeros(t, dtype=torch.int64, device="cuda"))
    want = (x.double() @ a[0].double().t())[:, at]
    assert ((got.double() - want).abs() <= (k / 64 + 40) * 2.0**-24 * want).all()


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("t", [9, 500])
def test_autograd_hears_of_a_write(cuda, monkeypatch, extension, t):
    """`out` may be a tensor that another operation keeps for its backward pass: that pass has to refuse."""
    from triton_ops import _lib, fused_lora

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    x, a, b = (torch.ones(s, device="cuda") for s in ((t, 16), (2, 4, 16), (2, 8, 4)))
    ids = torch.zeros(t, dtype=torch.int64, device="cuda")
    w = torch.ones(t, 8, device="cuda", requires_grad=True)
    y = torch.ones(t, 8, device="cuda")
    z = w * y
    fused_lora(x, a, b, ids, base=y)  # writes a tensor of its own
    torch.autograd.grad(z.sum(), w, retain_graph=True)
    view = y[:, :]
    fused_lora(x, a, b, ids, base=view, out=view)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z.sum(), w)
    with torch.inference_mode():
        y = torch.ones(t, 8, device="cuda")
        want = fused_lora(x, a, b, ids, base=y)
        assert torch.equal(fused_lora(x, a, b, ids, base=y, out=y), want)
    assert torch.equal(fused_lora(x, a, b, ids, out=y), want - 1)  # a tensor of inference mode keeps no version
