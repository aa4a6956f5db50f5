"""What fused_lora keeps of its fp32 sums and low-rank values, and what autograd hears of its writes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("rank", [2, 13, 16, 20, 40, 100, 256])
@pytest.mark.parametrize("dtype, bits, t", [("bf16", 24, 3), ("bf16", 24, 300), ("bf16", 24, 500), ("f16", 22, 3), ("f16", 22, 500)])
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
    by then, which grows evenly: K / 64; the halves, warps and CTAs: 12 more additions; each operand's lower tf32 value
    2^-22, and the products of two of them left out, at most 2^-20 and 2^-22 on average over the terms: 12; the same for v
    times one: 4 (B is one at one place).
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


@pytest.mark.parametrize("rank", [2, 30, 60, 120])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_sums_have_no_drift(cuda, dtype, rank):
    """The mean error of sums of 4096 positive terms in 16-bit types, in units of 2^-24 of the sum.

    Each row's sum S (products of 16 bits, 27 bits in all) is subtracted from itself: x holds its first 24 bits in three
    further columns, which the last rank adds up exactly. Rounded additions and rounded split values are off by as
    much either way; what is left of the mean is cut inside a step, at most eight instructions of at most two units of
    the step's own sum: 16, and 2 for the mean of the rest over 8192 rows. Sums kept in the instructions lose half an
    ulp, on average, of what is there at each of 128 (or with two CTAs a tile 64): 48 units (24)."""
    from triton_ops import fused_lora

    t, k, n = 8192, 4096, 16
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = torch.zeros(t, k + 32, device="cuda")
    x[:, :k] = 1 + torch.randint(128, (t, k), device="cuda", generator=g) / 128
    a = torch.zeros(1, rank, k + 32, device="cuda")
    a[0, 0, :k] = 1 + torch.randint(128, (k,), device="cuda", generator=g) / 128
    a[0, rank - 1, k:] = 1.0
    total = x.double() @ a[0, 0].double()
    step = 2.0 ** (torch.floor(torch.log2(total)) - 23)
    whole = torch.round(total / step).long()
    for i, shift in enumerate((16, 8, 0)):  # eight bits each: values of both types
        x[:, k + i] = ((whole >> shift) % 256 * 2**shift).double().mul(step).float()
    b = torch.zeros(1, n, rank, device="cuda")
    b[0, :, 0], b[0, :, rank - 1] = 1.0, -1.0
    dt = DT[dtype]
    got = fused_lora(x.to(dt), a.to(dt), b.to(dt), torch.zeros(t, dtype=torch.int64, device="cuda"))
    want = total - whole.double() * step
    assert abs(((got.double() - want[:, None]) / total[:, None]).mean().item()) <= 18 * 2.0**-24


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


@pytest.mark.parametrize("rank", [1, 12, 32, 48, 128, 200])
@pytest.mark.parametrize("t", [3, 40, 600])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_infinities_where_the_formula_has_them(cuda, dtype, t, rank):
    """Infinities of x, A, B, the factors and base give infinities and NaN where the formula does, and nowhere else."""
    from triton_ops import fused_lora

    g = torch.Generator().manual_seed(100 * rank + t)
    m, k, n, inf = 4, 24, 72, float("inf")
    # quarters between 1 and 2, of both signs: exact in each type, no zero beside an infinity
    x, a, b, base = ((1 + torch.randint(4, s, generator=g) / 4) * (1 - 2 * torch.randint(2, s, generator=g).float())
                     for s in ((t, k), (m, rank, k), (m, n, rank), (t, n)))
    scaling = torch.tensor([1.0, -0.5, 2.0, 1.5])
    ids = torch.arange(t) % m
    b[0, 5, 0], b[0, 6, rank - 1], b[1, 64, rank // 2] = inf, -inf, inf
    if rank > 1:
        b[0, 7, 0], b[0, 7, 1] = inf, -inf
    a[2, rank // 2, 3] = -inf
    b[2, 70, rank // 2] = inf
    x[t - 1, 7] = inf
    base[t // 2, 8], base[0, 9] = inf, float("nan")
    for numbers in (x, a, b):  # where fp32 is split: values that a tf32 holds, and values that it does not
        numbers.mul_(1.0 + (2.0**-20 if dtype == "f32" and t != 40 else 0.0))
    ref = base.double() + torch.stack([(b[i].double() * (a[i].double() * x[r].double()).sum(-1)).sum(-1) * scaling[i]
                                       for r, i in enumerate(ids.tolist())])
    to = DT[dtype]
    got = fused_lora(x.to(to).cuda(), a.to(to).cuda(), b.to(to).cuda(), ids.cuda(), scaling.cuda(),
                     base=base.to(to).cuda()).double().cpu()
    # Where fp32 operands are no tf32 values, a low-rank value whose terms cancel to zero is one only within its sum's
    # rounding: times an infinity it is a NaN, or an infinity if the sum is not quite zero. Both are right.
    if dtype == "f32" and t != 40:
        for r, i in enumerate(ids.tolist()):
            v = (a[i].double() * x[r].double()).sum(-1)
            either = ((v == 0) & torch.isinf(b[i])).any(-1)
            assert not torch.isfinite(got[r, either]).any()
            got[r, either] = ref[r, either]
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(torch.isinf(got), torch.isinf(ref)) and torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])
    fine = torch.isfinite(ref)
    # |v| <= 1.75^2 k and |B|, |scaling| <= 2: magnitudes of at most 16 k rank; v of 16 bits: 2^-16 of them (its sum is
    # exact); fp32: 2^-19 for both products; and the result's rounding
    slack = rank * k * 16 * (2.0**-19 if dtype == "f32" else 2.0**-16)
    assert ((got - ref).abs() <= ref.abs() * torch.finfo(to).eps / 2 * 1.01 + slack)[fine].all()


def test_the_largest_fp32_values(cuda):
    """Finite operands that round past the largest tf32."""
    from triton_ops import fused_lora

    big = torch.finfo(torch.float32).max
    for t in (3, 500):
        x, a, b = torch.full((t, 8), big, device="cuda"), torch.zeros(1, 1, 8, device="cuda"), torch.ones(1, 4, 1, device="cuda")
        a[0, 0, 2] = 0.25
        got = fused_lora(x, a, b, torch.zeros(t, dtype=torch.int64, device="cuda"))
        assert ((got.double() - big / 4).abs() <= big / 4 * 2.0**-21).all()


@pytest.mark.parametrize("t", [3, 500])
def test_any_nan_is_a_nan(cuda, t):
    """Also one whose bits past those of a tf32 are all that sets it apart from an infinity."""
    from triton_ops import fused_lora

    x, a, b = (torch.ones(s, device="cuda") for s in ((t, 8), (1, 4, 8), (1, 8, 4)))
    ids = torch.zeros(t, dtype=torch.int64, device="cuda")
    for bits in (0x7F800001, 0x7FC00000, 0x7FFFFFFF, -0x7FFFFF):  # the last: 0xff800001
        for v, at, where in ((x, (1, 3), (slice(1, 2), slice(None))), (a, (0, 2, 5), (slice(None), slice(None))),
                             (b, (0, 6, 1), (slice(None), slice(6, 7)))):
            with_nan = v.clone()
            with_nan.view(torch.int32)[at] = bits
            got = fused_lora(*(with_nan if u is v else u for u in (x, a, b)), ids)
            want = torch.zeros(t, 8, dtype=torch.bool, device="cuda")
            want[where] = True
            assert torch.equal(torch.isnan(got), want)
