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
