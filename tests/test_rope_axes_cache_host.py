"""What the rotation's host side keeps between calls (no GPU)."""

import pytest

from triton_ops import RoPEAxes, RoPEScaling
from triton_ops.kernels.rope import _pair_axes, _turns, rope_frequencies


def test_pairs_axes_are_kept_once():
    axes = RoPEAxes((2, 1, 3), "cycle")
    assert _pair_axes(axes) is _pair_axes(RoPEAxes([2, 1, 3], "cycle")) and _pair_axes(axes).tolist() == [0, 1, 2, 0, 2, 2]
    assert not hasattr(_pair_axes.__wrapped__, "cache_info")


def test_checks_do_not_depend_on_earlier_calls():
    """A plain tuple is no RoPEAxes, nor RoPEScaling, also where one that equals it was used before."""
    axes, scaling = RoPEAxes((2, 1, 3)), RoPEScaling("linear", 2.0)
    for cached in (rope_frequencies, _turns):
        cached(12, 10000.0, scaling, axes)
        with pytest.raises(TypeError):
            cached(12, 10000.0, scaling, tuple(axes))
        with pytest.raises(AttributeError):
            cached(12, 10000.0, tuple(scaling), axes)
