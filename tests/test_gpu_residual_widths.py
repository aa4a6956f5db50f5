"""fused_residual_rmsnorm on the GPU where a row's width, or the number of elements, changes the way it is worked on.

The bounds are those that test_gpu_residual.py derives.
"""

import pytest
import torch
from test_gpu_residual import compare, formulas, make, randn, run

from triton_ops.kernels.dropout import dropout_keep_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,stream", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("branch_norm", [True, False])
def test_rows_that_end_inside_a_warp(cuda, dtype, stream, branch_norm):
    """1, 7, 17 and 31 lanes of the last warp with columns, the last of them with all or some; every sum wanted."""
    lane = 8 if dtype == "f32" else 16  # columns a thread
    for lanes in (1, 7, 17, 31):
        for warps, odd in ((1, 0), (3, 0), (6, 5), (9, 0), (10, 1)):
            hidden = (32 * warps + lanes) * lane - odd
            shape = (2, 5, hidden)
            t = make(shape, dtype, stream, branch_weight="f32" if branch_norm else None, gate="f32", shift="f32", per="gate",
                     seed=hidden)
            keep = dropout_keep_reference(shape, 0.2, 7, 0, "cuda")
            gh, gy = randn(shape, stream, 11), randn(shape, dtype, 12)
            both = run(t, branch_norm, 0.7, 0.2, 7, gh, gy)
            compare(t, both, formulas(t, branch_norm, 0.7, keep, 0.2, gh, gy), f"{hidden} wide")
            # one gradient alone: without the second norm a row may have no sum that joins its threads
            for one in (dict(gh=gh), dict(gy=gy)):
                compare(t, run(t, branch_norm, 0.7, 0.2, 7, **one), formulas(t, branch_norm, 0.7, keep, 0.2, **one), f"{hidden} wide")
            again = run(t, branch_norm, 0.7, 0.2, 7, gh, gy)
            assert all(torch.equal(again[k], both[k]) for k in both if both[k] is not None)


# Both sides of each border between the kernels: a row in one group's registers with 16 columns a thread up to 8192, forward
# aligned 32 up to 16384; gradients of 4 bytes a column that are not aligned up to 4096; wider ones read a row again.
@pytest.mark.parametrize("dtype,stream,hidden", [
    ("bf16", "bf16", 8192), ("bf16", "bf16", 8200), ("bf16", "bf16", 8191), ("bf16", "bf16", 8193),
    ("f16", "f16", 16384), ("f16", "f16", 16392), ("bf16", "f32", 16384), ("bf16", "f32", 16388),
    ("bf16", "f32", 4095), ("bf16", "f32", 4097), ("bf16", "f32", 8192), ("bf16", "f32", 8196), ("f16", "f32", 8191), ("f16", "f32", 8193),
    ("f32", "f32", 8192), ("f32", "f32", 8196), ("f32", "f32", 16384), ("f32", "f32", 16388),
    ("f32", "f32", 4095), ("f32", "f32", 4097), ("f32", "f32", 8191), ("f32", "f32", 8193),
])
def test_borders_between_kernels(cuda, dtype, stream, hidden):
    shape = (2, 3, hidden)
    t = make(shape, dtype, stream, branch_weight="f32", gate="f32", shift="f32", per="gate")
    keep = dropout_keep_reference(shape, 0.1, 7, 0, "cuda")
    gh, gy = randn(shape, stream, 11), randn(shape, dtype, 12)
    compare(t, run(t, True, 0.7, 0.1, 7, gh, gy), formulas(t, True, 0.7, keep, 0.1, gh, gy), "border")


def kept_rows(rows, hidden, p, seed):
    """What is kept in some rows of a long tensor, from the generator's words at their elements."""
    low = 0xFFFFFFFF
    element = rows[:, None] * hidden + torch.arange(hidden, device=rows.device)
    block = element // 4
    words = [block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)]
    key = [seed & low, seed >> 32]
    for _ in range(10):
        even, odd = words[0] * 0xD2511F53, words[2] * 0xCD9E8D57
        words = [((odd >> 32) & low) ^ words[1] ^ key[0], odd & low, ((even >> 32) & low) ^ words[3] ^ key[1], even & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    word = torch.stack(words, -1).gather(-1, (element % 4)[..., None])[..., 0]
    return word >= round(p * 2**32)


def test_kept_rows_are_those_of_the_reference(cuda):
    rows = torch.tensor([0, 3, 4], device="cuda")
    assert torch.equal(kept_rows(rows, 33, 0.3, 2**33 + 5), dropout_keep_reference((5, 33), 0.3, 2**33 + 5, 0, "cuda")[rows])


@pytest.mark.parametrize("hidden", [8192, 8191, 20001])
def test_both_directions_past_2_31_elements(cuda, hidden):
    """With dropout: rows at the start, around 2^31 elements and at the end; aligned, not aligned, read again."""
    rows = 2**31 // hidden + 300
    g = torch.Generator(device="cuda").manual_seed(1)
    x, res, gh, gy = (torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in range(4))
    t = {"x": x, "residual": res, "branch_weight": 1 + 0.1 * randn((hidden,), "f32", 2), "gate": None, "weight": None, "shift": None}
    got = run(t, True, 1.0, 0.3, 2**40 + 7, gh, gy)
    border = 2**31 // hidden
    at = torch.tensor([0, 1, 77, border - 2, border - 1, border, border + 1, border + 200, rows - 2, rows - 1], device="cuda")
    part = {k: v if v is None or v.dim() == 1 else v[at] for k, v in t.items()}
    want = formulas(part, True, 1.0, kept_rows(at, hidden, 0.3, 2**40 + 7), 0.3, gh[at], gy[at])
    del want["branch_weight"]  # of these rows alone
    compare(part, {k: v[at] for k, v in got.items() if k in want}, want, "past 2^31")


@pytest.mark.parametrize("dtype,shape,per", [
    ("f32", (1, 148, 4096), False), ("bf16", (1, 4440, 4096), False), ("bf16", (1, 3000, 1001), False), ("f32", (1, 1200, 5329), False),
    ("bf16", (1, 1500, 12288), False), ("bf16", (16, 1025, 1152), True), ("f16", (40, 300, 136), True), ("f32", (700, 7, 64), True),
])
def test_sums_over_rows(cuda, dtype, shape, per):
    """Parameters' gradients, of sums whose terms are exact: one rounding for each row that a CTA adds, not one for each row.

    A launch gives each of 148 SMs, or its share of them for each sequence, a run of rows; that run's rows are added in
    fp32 (by up to 16 groups, and these to one another), the runs in fp64.
    """
    batch, seq, hidden = shape
    run_rows = -(-seq // max(1, 148 // batch)) if per else -(-batch * seq // 148)
    share = (run_rows + 4) * 2.0**-24
    sign = randn(shape, "f32", 1).sign()
    sign[sign == 0] = 1
    gy = randn(shape, dtype, 2)
    axis = 1 if per else (0, 1)
    own = (batch, hidden) if per else (hidden,)

    def check(got, terms, factor=0.0):
        ref = terms.sum(axis)
        assert ((got.double() - ref).abs() <= share * terms.abs().sum(axis) + (factor + 2.0**-24) * ref.abs()).all()

    t = {"x": torch.zeros(shape, device="cuda", dtype=gy.dtype), "residual": sign.to(gy.dtype),
         "weight": torch.ones(own, device="cuda"), "shift": torch.zeros(own, device="cuda")}
    got = run(t, gy=gy)
    check(got["shift"], gy.double())
    # rows of ones and minus ones: their norm is one factor, rsqrtf's (2 ulp) of a mean that has less than 2^-18 of error
    check(got["weight"], gy.double() * sign.double() / (1 + 1e-5) ** 0.5, 2.0**-18)
    gate = {"x": sign.to(gy.dtype), "residual": t["residual"], "gate": torch.ones(own, device="cuda")}
    check(run(gate, gh=gy, norm=False)["gate"], gy.double() * sign.double())
