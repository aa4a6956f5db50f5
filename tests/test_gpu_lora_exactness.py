"""What fused_lora keeps of its fp32 low-rank values, on cases with exact answers.

Every product, partial sum and result below is exact in fp32 and in the operands' type: the outputs have to be equal,
not near.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("rank", [2, 20, 40, 100, 256])
@pytest.mark.parametrize("dtype, bits, t", [("bf16", 24, 3), ("bf16", 24, 300), ("bf16", 16, 500), ("f16", 22, 3), ("f16", 22, 500)])
def test_low_rank_values_keep_their_bits(cuda, dtype, bits, t, rank):
    """Two low-rank values below 2^bits that differ by less than 128, one subtracted from the other.

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
