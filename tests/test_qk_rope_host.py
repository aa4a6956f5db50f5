"""Host logic of the query/key path without a GPU: frequencies, refusals, C-ABI argument checks."""

import ctypes
import math

import pytest
import torch

from triton_ops import RoPEScaling, _lib, validation
from triton_ops.exceptions import DeviceError, ShapeMismatchError, UnsupportedDtypeError
from triton_ops.kernels.rope import rope_frequencies


def test_frequencies():
    freq, gain = rope_frequencies(8, 10000.0)
    assert gain == 1.0 and freq == tuple(10000.0 ** (-i / 4) for i in range(4))
    half, _ = rope_frequencies(8, 10000.0, RoPEScaling("linear", 2.0))
    assert half == tuple(f / 2 for f in freq)
    ntk, _ = rope_frequencies(8, 10000.0, RoPEScaling("ntk", 4.0))
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], freq[-1] / 4, rel_tol=1e-12)
    # far above / below the borders a pair is kept / slowed by the factor
    for kind in ("yarn", "wavelength"):
        s = RoPEScaling(kind, 8.0, 8192)
        got, gain = rope_frequencies(128, 10000.0, s)
        plain, _ = rope_frequencies(128, 10000.0)
        assert got[0] == plain[0] and math.isclose(got[-1], plain[-1] / 8, rel_tol=1e-12)
        assert all(p / 8 * (1 - 1e-12) <= g <= p for g, p in zip(got, plain))
        assert list(got) == sorted(got, reverse=True)
        assert math.isclose(gain, 1 + 0.1 * math.log(8.0) if kind == "yarn" else 1.0)
        for i, (g, p) in enumerate(zip(got, plain)):
            if kind == "wavelength":
                turns = 8192 * p / (2 * math.pi)
                if turns >= 4:
                    assert g == p
                elif turns <= 1:
                    assert math.isclose(g, p / 8, rel_tol=1e-12)
    assert rope_frequencies(8, 10000.0, RoPEScaling("linear", 2.0, attention_factor=0.25))[1] == 0.25


@pytest.mark.parametrize("args", [("cubic",), ("linear", 0.0), ("linear", float("nan")), ("yarn", 2.0),
                                  ("wavelength", 2.0), ("yarn", 2.0, 4096, 1.0, 1.0),
                                  ("wavelength", 2.0, 4096, 32.0, 1.0, 4.0, 4.0)])
def test_scaling_refusals(args):
    with pytest.raises(ValueError):
        RoPEScaling(*args)


def test_scaling_is_a_checked_value():
    s = RoPEScaling("yarn", 8.0, original_max_position=4096)
    assert s == RoPEScaling("yarn", 8.0, 4096) and hash(s) == hash(RoPEScaling("yarn", 8.0, 4096))
    assert s.factor == 8.0 and s._replace(factor=2.0) == RoPEScaling("yarn", 2.0, 4096)
    with pytest.raises(ValueError):
        s._replace(factor=-1.0)
    with pytest.raises(AttributeError):
        s.factor = 3.0


def test_frequency_refusals():
    for rot in (0, 3, 514):
        with pytest.raises(ShapeMismatchError):
            rope_frequencies(rot)
    with pytest.raises(ShapeMismatchError):
        rope_frequencies(2, 10000.0, RoPEScaling("ntk", 2.0))
    with pytest.raises(ValueError):
        rope_frequencies(8, 1.0)


def test_ops_refuse_cpu_tensors():
    from triton_ops import fused_qk_norm_rope, fused_rope, rope_tables

    q, t = torch.zeros(1, 2, 2, 8), torch.zeros(2, 8)
    with pytest.raises(DeviceError):
        fused_rope(q, None, t, t)
    with pytest.raises(DeviceError):
        fused_qk_norm_rope(q, q, None, None, t, t)
    with pytest.raises(DeviceError):
        rope_tables(torch.zeros(3, dtype=torch.int64), 8)


def test_argument_checks(monkeypatch):
    """The checks behind the ops, on CPU tensors (the device check set aside)."""
    monkeypatch.setattr(validation, "_check_cuda", lambda t, n: None)
    q, t = torch.zeros(2, 4, 3, 8), torch.zeros(4, 8)
    check = validation.validate_rope_heads
    cos, sin, pos = check(q, q[:, :, :1], t[None, :, None], t, torch.zeros(4, dtype=torch.int32))
    assert cos.shape == sin.shape == (4, 8) and pos.shape == (2, 4) and pos.stride() == (0, 1)
    assert check(q, None, t, t.half(), None)[0].dtype == torch.float32
    strided = torch.zeros(4, 16)[:, ::2]
    assert check(q, None, strided, t, None)[0].stride() == (8, 1)
    for args, error in (
        ((q.double(), None, t, t, None), UnsupportedDtypeError),
        ((q, q.half(), t, t, None), UnsupportedDtypeError),
        ((q, q[:1], t, t, None), ShapeMismatchError),
        ((q, q[0], t, t, None), ShapeMismatchError),
        ((q[0, 0], None, t, t, None), ShapeMismatchError),
        ((q, None, t[:3], t[:3], None), ShapeMismatchError),
        ((q, None, t[0], t[0], None), ShapeMismatchError),
        ((q, None, torch.zeros(4, 10), torch.zeros(4, 10), None), ShapeMismatchError),
        ((q, None, torch.zeros(4, 0), torch.zeros(4, 0), None), ShapeMismatchError),
        ((q, None, t, t, torch.zeros(2, 4)), UnsupportedDtypeError),
        ((q, None, t, t, torch.zeros(3, 4, dtype=torch.int64)), ShapeMismatchError),
        ((q, None, t[:0], t[:0], torch.zeros(2, 4, dtype=torch.int64)), ShapeMismatchError),
        ((q.transpose(2, 3), None, torch.zeros(4, 2), torch.zeros(4, 2), None), ValueError),
        ((q, None, t.clone().requires_grad_(), t, None), ValueError),
        ((torch.zeros(1, 1, 1, 1026), None, t, t, None), ShapeMismatchError),
    ):
        with pytest.raises(error):
            check(*args)
    with pytest.raises(ShapeMismatchError):
        validation.validate_head_weight(q, torch.ones(7), "q_weight")
    with pytest.raises(ValueError):
        validation.validate_head_weight(q, torch.ones(16)[::2], "q_weight")


def strides(*s):
    return (ctypes.c_int64 * 3)(*s)


def test_entry_points_report_bad_arguments():
    lib = _lib.load()
    st = strides(8, 8, 8)

    def rope(batch=1, seq=2, hq=1, hk=0, dim=8, rot=8, dtype=2, table=2, rows=2, pos=None, pos_dtype=0, q=16):
        return lib.tfo_rope(q, st, None, st, 16, 16, 8, rows, pos, pos_dtype, 0, 0, 16, None, batch, seq, hq, hk, dim,
                            rot, 0, 0, dtype, table, None)

    assert rope(batch=0) == _lib.OK and rope(hq=0) == _lib.OK  # nothing to do, nothing launched
    assert rope(dtype=3) == _lib.ERR_DTYPE and rope(table=4) == _lib.ERR_DTYPE and rope(pos_dtype=3) == _lib.ERR_DTYPE
    for bad in ({"rot": 7}, {"rot": 10}, {"rot": 0}, {"dim": 0}, {"dim": 1025}, {"batch": -1}, {"rows": 1},
                {"pos_dtype": 1}, {"q": None}, {"hk": 1}, {"hq": 1 << 17}):
        assert rope(**bad) == _lib.ERR_INVALID, bad
    turns = (ctypes.c_double * 4)()
    assert lib.tfo_rope_tables(None, 0, 0, turns, 4, 1.0, None, None, 2, None) == _lib.OK
    assert lib.tfo_rope_tables(None, 0, 3, turns, 257, 1.0, 16, 16, 2, None) == _lib.ERR_INVALID
    assert lib.tfo_rope_tables(None, 2, 3, turns, 4, 1.0, 16, 16, 2, None) == _lib.ERR_INVALID
    assert lib.tfo_rope_tables(None, 0, 3, turns, 4, 1.0, 16, 16, 3, None) == _lib.ERR_DTYPE
    assert b"f16, bf16 or f32" in lib.tfo_last_error()

    def backward(ws=0, w=16, dw=16, wd=2):
        return lib.tfo_qk_norm_rope_backward(16, st, None, st, 16, st, None, st, w, None, 16, 16, 8, 2, None, 0, 0, 0, 16,
                                             None, dw, None, 1, 2, 1, 0, 8, 8, 0, 1e-6, 2, wd, 2, 2, None, ws, None)

    assert backward() == _lib.ERR_INVALID  # no workspace for the weight sums
    assert backward(w=None) == _lib.ERR_INVALID
    assert backward(wd=3) == _lib.ERR_DTYPE
    assert lib.tfo_qk_norm_rope_backward_workspace_bytes(128) >= 4 * 128
    assert lib.tfo_qk_norm_rope_backward_workspace_bytes(0) == 0


def test_lora_argument_checks(monkeypatch):
    from triton_ops import fused_lora

    x, a, b, ids = torch.zeros(3, 8), torch.zeros(2, 4, 8), torch.zeros(2, 6, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(DeviceError):
        fused_lora(x, a, b, ids)
    monkeypatch.setattr(validation, "_check_cuda", lambda t, n: None)
    check = validation.validate_lora_inputs
    assert check(x, a, b, ids, None, None, None) == (3, 2, 4, 8, 6)
    for args, error in (
        ((x, a.half(), b, ids, None, None, None), UnsupportedDtypeError),
        ((x, a, b, ids.float(), None, None, None), UnsupportedDtypeError),
        ((x, a[:, :, :7], b, ids, None, None, None), ShapeMismatchError),
        ((x, a, b[:1], ids, None, None, None), ShapeMismatchError),
        ((x, a, b, ids[:2], None, None, None), ShapeMismatchError),
        ((x, a, b, ids, torch.ones(3), None, None), ShapeMismatchError),
        ((x, a, b, ids, None, torch.zeros(3, 5), None), ShapeMismatchError),
        ((x, a, b, ids, None, None, torch.zeros(2, 6)), ShapeMismatchError),
        ((x, torch.zeros(2, 257, 8), torch.zeros(2, 6, 257), ids, None, None, None), ShapeMismatchError),
        ((x.clone().requires_grad_(), a, b, ids, None, None, None), ValueError),
    ):
        with pytest.raises(error):
            check(*args)


def test_the_factors_of_adapters_stay_fp32():
    from triton_ops import FP8LoRALinear

    m = FP8LoRALinear(16, 8, max_adapters=2, rank=4)
    m.set_adapter(1, torch.ones(4, 16), torch.ones(8, 4), 1 / 3)
    factors = m.scaling.clone()
    for convert in (m.half, m.bfloat16, lambda: m.to("cpu", torch.float16)):
        convert()
        assert m.scaling.dtype == torch.float32 and torch.equal(m.scaling, factors)
    assert m.lora_a.dtype == m.lora_b.dtype == torch.float16
    assert m.state_dict()["scaling"].dtype == torch.float32


def test_lora_entry_point_reports_bad_arguments():
    lib = _lib.load()

    def lora(tokens=2, adapters=1, rank=4, k=8, n=8, dtype=2, ids_dtype=2, x=16, ws=None, bytes_=0, base=None):
        return lib.tfo_lora(x, 8, 16, 16, 16, ids_dtype, None, base, 0, 16, 8, tokens, adapters, rank, k, n, dtype, ws,
                            bytes_, None)

    assert lora(tokens=0) == _lib.OK and lora(n=0) == _lib.OK
    assert lora(dtype=3) == _lib.ERR_DTYPE and lora(ids_dtype=0) == _lib.ERR_DTYPE
    for bad in ({"rank": 257}, {"rank": 0}, {"k": 0}, {"adapters": 0}, {"adapters": 16385}, {"tokens": -1}, {"x": None},
                {"tokens": 400}, {"tokens": 400, "ws": 8, "bytes_": 1 << 40}, {"n": 9}, {"base": 16}):
        assert lora(**bad) == _lib.ERR_INVALID, bad
    assert lib.tfo_lora_workspace_bytes(400, 4) >= 400 * 4
    assert lib.tfo_lora_workspace_bytes(400, 0) == 0
