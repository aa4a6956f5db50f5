"""What the rotation's host side keeps between calls (no GPU)."""

from triton_ops import RoPEAxes
from triton_ops.kernels.rope import _pair_axes


def test_pairs_axes_are_kept_once():
    axes = RoPEAxes((2, 1, 3), "cycle")
    assert _pair_axes(axes) is _pair_axes(RoPEAxes([2, 1, 3], "cycle")) and _pair_axes(axes).tolist() == [0, 1, 2, 0, 2, 2]
    assert not hasattr(_pair_axes.__wrapped__, "cache_info")
