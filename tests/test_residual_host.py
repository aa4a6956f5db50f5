"""Host logic of the residual stream, dropout and positions of several axes without a GPU."""

import ctypes

import pytest
import torch

from triton_ops import FusedDropout, FusedResidualRMSNorm, RoPEAxes, RoPEScaling, _lib, fused_dropout, fused_residual_rmsnorm
from triton_ops.exceptions import DeviceError, ShapeMismatchError
from triton_ops.kernels.dropout import dropout_keep_reference
from triton_ops.kernels.residual import residual_rmsnorm_reference
from triton_ops.kernels.rope import rope_frequencies


def test_axes_of_pairs():
    assert RoPEAxes((2, 1, 3)).axis_of_pairs() == (0, 0, 1, 2, 2, 2)
    assert RoPEAxes((2, 1, 3), "cycle").axis_of_pairs() == (0, 1, 2, 0, 2, 2)
    turns = RoPEAxes((24, 20, 20), "cycle").axis_of_pairs()
    assert all(turns[i] == i % 3 for i in range(60)) and turns[60:] == (0, 0, 0, 0)
    assert RoPEAxes([1, 2]) == RoPEAxes((1, 2)) and hash(RoPEAxes([1, 2])) == hash(RoPEAxes((1, 2)))
    for wrong in (((3,),), ((1, 2, 3, 4, 5),), ((0, 4),), ((4, 4), "rows"), ((4, 4), "blocks", "mine")):
        with pytest.raises(ValueError):
            RoPEAxes(*wrong)
    with pytest.raises(ValueError):
        RoPEAxes((4, 4))._replace(order="rows")


def test_axes_frequencies():
    plain, _ = rope_frequencies(12, 10000.0)
    assert rope_frequencies(12, 10000.0, None, RoPEAxes((2, 1, 3)))[0] == plain
    own, gain = rope_frequencies(12, 10000.0, None, RoPEAxes((2, 1, 3), "cycle", "own"))
    three = rope_frequencies(6, 10000.0)[0]
    assert own == (1.0, 1.0, three[0], rope_frequencies(4, 10000.0)[0][1], three[1], three[2]) and gain == 1.0
    assert rope_frequencies(8, 100.0, RoPEScaling("linear", 2.0, attention_factor=3.0), RoPEAxes((2, 2), "blocks", "own")) == \
        ((0.5, 0.05, 0.5, 0.05), 3.0)
    with pytest.raises(ShapeMismatchError):
        rope_frequencies(16, 10000.0, None, RoPEAxes((2, 1, 3)))
    with pytest.raises(TypeError):
        rope_frequencies(12, 10000.0, None, (2, 1, 3))


def test_generator_known_answers():
    """The published answer of the generator for a counter and key of zeros."""
    for word, i in ((0x6627E8D5, 0), (0xE169C58D, 1), (0xBC57AC4C, 2), (0x9B00DBD8, 3)):
        assert dropout_keep_reference((4,), word / 2**32, 0)[i]
        assert not dropout_keep_reference((4,), (word + 1) / 2**32, 0)[i]


def test_reference_is_the_formula():
    x = torch.tensor([[3.0, 4.0]], dtype=torch.float64)
    res = torch.tensor([[1.0, -1.0]], dtype=torch.float64)
    h, y = residual_rmsnorm_reference(x, res, torch.tensor([2.0, 1.0]).double(), torch.tensor([1.0, 0.5]).double(), branch_norm=True,
                                      shift=torch.tensor([0.0, 1.0]).double(), scale=2.0, eps=0.0)
    r = 12.5**0.5
    want = torch.tensor([[1 + 2 * 3 / r, -1 + 4 / r]], dtype=torch.float64)
    assert torch.allclose(h, want)
    assert torch.allclose(y, want / want.pow(2).mean().sqrt() * torch.tensor([2.0, 1.0]) + torch.tensor([0.0, 1.0]))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(DeviceError):
        fused_residual_rmsnorm(x, x)
    with pytest.raises(DeviceError):
        fused_dropout(x, 0.5, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            FusedDropout(p)
        with pytest.raises(ValueError):
            FusedResidualRMSNorm(8, dropout=p)
    m = FusedResidualRMSNorm(8, branch_norm=True, layer_scale=0.5)
    assert {k for k, _ in m.named_parameters()} == {"weight", "branch_weight", "gate"}
    assert (m.gate == 0.5).all() and dict(m.named_buffers())["seed"].dtype == torch.int64


def test_c_abi_refusals():
    """Argument errors are reported without touching a GPU."""
    lib = _lib.load()
    drop = _lib.DropoutParams(0.5, None, 1, 0)

    def dropout(x=16, res=None, out=16, n=8, d=drop, xt=0, ot=0):
        return lib.tfo_dropout(x, res, out, n, None if d is None else ctypes.byref(d), xt, ot, None)

    assert dropout(n=0) == _lib.OK
    assert dropout(xt=3) == dropout(ot=1) == dropout(ot=2) == dropout(res=16, xt=2, ot=0) == _lib.ERR_DTYPE
    assert dropout(n=-1) == dropout(d=None) == dropout(x=None) == dropout(out=None) == _lib.ERR_INVALID
    for p in (-0.1, 1.1, float("nan")):
        assert dropout(d=_lib.DropoutParams(p, None, 1, 0)) == _lib.ERR_INVALID
    assert dropout(d=_lib.DropoutParams(0.5, 4, 1, 0)) == _lib.ERR_INVALID  # a seed off its border

    def params(**more):
        p = (_lib.RowParam * 4)()
        for i, name in enumerate(("branch_weight", "gate", "weight", "shift")):
            p[i] = more.get(name, _lib.RowParam(None, 0, 2, None))
        return p

    def forward(x=16, res=16, p=None, h=16, rstd=None, rows=4, per=2, hidden=8, norm=1, d=None, xt=0, rt=0):
        return lib.tfo_residual_rmsnorm(x, hidden, res, hidden, params() if p is None else p, h, None, rstd, rows, per, hidden,
                                        norm, 1.0, 1e-6, d, xt, rt, None)

    def backward(rstd=16, rows=4, per=2, p=None, ws=None, size=0):
        return lib.tfo_residual_rmsnorm_backward(16, 8, 16, 8, 16, 8, 16, 8, params() if p is None else p, rstd, 16, 16, rows, per,
                                                 8, 1, 1.0, None, 0, 0, ws, size, None)

    assert forward(rows=0, x=None) == backward(rows=0) == _lib.OK
    assert forward(xt=3) == forward(xt=2, rt=0) == forward(xt=0, rt=1) == _lib.ERR_DTYPE
    assert forward(p=params(gate=_lib.RowParam(16, 0, 3, None))) == _lib.ERR_DTYPE
    assert forward(x=None) == forward(res=None) == forward(h=None) == forward(rstd=4) == _lib.ERR_INVALID
    assert forward(hidden=0) == forward(hidden=2**24 + 1) == forward(rows=-1) == forward(per=3) == forward(per=0) == _lib.ERR_INVALID
    assert forward(rows=2**31, per=1) == forward(d=ctypes.byref(_lib.DropoutParams(2.0, None, 1, 0))) == _lib.ERR_INVALID
    assert forward(norm=0, p=params(branch_weight=_lib.RowParam(16, 0, 2, None))) == _lib.ERR_INVALID
    assert backward(rstd=None) == backward(rstd=4) == backward(per=3) == _lib.ERR_INVALID

    def strided(x=8, res=8):
        return lib.tfo_residual_rmsnorm(16, x, 16, res, params(), 16, None, None, 4, 2, 8, 1, 1.0, 1e-6, None, 0, 0, None)

    def strided_backward(x=8, res=8, dh=8, dy=8):
        return lib.tfo_residual_rmsnorm_backward(16, dh, 16, dy, 16, x, 16, res, params(), 16, 16, 16, 4, 2, 8, 1, 1.0, None, 0, 0,
                                                 None, 0, None)

    assert strided(x=-8) == strided(res=-1) == _lib.ERR_INVALID
    for wrong in (dict(x=-8), dict(res=-8), dict(dh=-8), dict(dy=-8)):
        assert strided_backward(**wrong) == _lib.ERR_INVALID

    def heads(axes):
        s = (ctypes.c_int64 * 3)(64, 64, 8)
        return lib.tfo_rope_axes(16, s, None, None, 16, 16, 8, 4, 16, _lib.POS_I64, 4, 1, 16, None, 1, 4, 1, 0, 8, 8, 0, 0, 0, 2, axes,
                                 None)

    for count, which in ((1, (0, 0, 0, 0)), (5, (0, 1, 2, 3)), (2, (0, 1, 2, 1))):
        of = (ctypes.c_uint8 * 4)(*which)
        assert heads(ctypes.byref(_lib.Axes(count, 4, ctypes.addressof(of)))) == _lib.ERR_INVALID
    assert heads(ctypes.byref(_lib.Axes(2, 4, None))) == _lib.ERR_INVALID
    turns = (ctypes.c_double * 4)(*(0.1,) * 4)
    of = (ctypes.c_uint8 * 4)(0, 1, 0, 1)
    assert lib.tfo_rope_tables_axes(None, _lib.POS_NONE, 4, turns, 4, 1.0, 16, 16, 2,
                                    ctypes.byref(_lib.Axes(2, 4, ctypes.addressof(of))), None) == _lib.ERR_INVALID
