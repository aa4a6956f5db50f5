"""Scratch of the rotation by several axes: asked for where a call puts its tokens' table rows together, and only there."""

import ctypes

from triton_ops import RoPEAxes, _lib


def asked(sections, order="blocks", batch=1, seq=8192, heads=(32, 8), dim=128, pairs=0, dtype=_lib.BF16, table=_lib.F32, count=None):
    of = (ctypes.c_uint8 * sum(sections))(*RoPEAxes(sections, order).axis_of_pairs())
    axes = _lib.Axes(count or len(sections), 0, ctypes.addressof(of), None, 0)
    return _lib.load().tfo_rope_axes_call_workspace_bytes(batch, seq, *heads, dim, 2 * sum(sections), pairs, dtype, table,
                                                          ctypes.byref(axes))


def most(tokens, pairs, table=_lib.F32):
    return _lib.load().tfo_rope_axes_workspace_bytes(tokens, 2 * pairs, table)


def test_many_tokens_of_shared_vectors():
    assert asked((24, 20, 20), "cycle") == most(8192, 64) == 2 * 8192 * 64 * 4
    assert asked((24, 20, 20), "cycle", batch=2, seq=4096, table=_lib.BF16) == most(8192, 64, _lib.BF16) == 2 * 8192 * 64 * 2
    assert asked((24, 20, 20)) == asked((24, 20, 20), heads=(32, 0)) == most(8192, 64)  # 24 is three vectors, 44 is not a whole number
    assert asked((12, 10, 10), pairs=1, dim=64) == most(8192, 32)
    # no vectors of 16 bytes, but of 8
    assert asked((18, 14, 12), dim=88) == most(8192, 44)


def test_no_use():
    assert asked((16, 24, 24)) == 0 and asked((16, 24, 24), seq=1 << 20) == 0  # whole vectors of 8 pairs
    assert asked((8, 28, 28), pairs=1, seq=29999) == 0  # of 4 pairs
    assert asked((24, 20, 20), dtype=_lib.F32) == 0  # of 4 pairs
    for seq in (1, 64, 500):  # tokens below the streaming kernel's
        assert asked((24, 20, 20), "cycle", seq=seq) == 0
    assert asked((9, 8), "cycle", dim=36) == 0  # heads that are not whole vectors
    assert asked((24, 20, 20), "cycle", heads=(0, 0)) == asked((24, 20, 20), "cycle", seq=0) == 0


def test_wrong_arguments():
    assert asked((24, 20, 20), "cycle", dim=64) == asked((24, 20, 20), "cycle", dtype=7) == asked((24, 20, 20), "cycle", table=7) == 0
    assert asked((24, 20, 20), "cycle", count=2) == asked((24, 20, 20), "cycle", count=5) == 0
    assert _lib.load().tfo_rope_axes_call_workspace_bytes(1, 8192, 32, 8, 128, 128, 0, _lib.BF16, _lib.F32, None) == 0
