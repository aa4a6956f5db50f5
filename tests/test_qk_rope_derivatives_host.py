"""Host logic of the query/key path without a GPU: what torch's default device and derivatives have to do with it."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def test_the_frequencies_lie_in_host_memory_whatever_the_default_device():
    """The library reads them on the host."""
    from triton_ops.kernels.rope import _turns

    with torch.device("meta"):
        array, turns, _ = _turns(34, 12345.0, None)
    assert turns.device.type == "cpu" and turns.dtype == torch.float64 and turns.is_contiguous()
    assert turns.tolist() == list(array) and len(array) == 17
    assert _turns(34, 12345.0, None)[1].device.type == "cpu"


def test_forward_mode_is_refused(monkeypatch):
    """The checks behind the ops, on CPU tensors (the device check set aside): no tangent is lost without a word."""
    from triton_ops import validation

    monkeypatch.setattr(validation, "_check_cuda", lambda t, n: None)
    q, k, t, w = torch.ones(2, 4, 3, 8), torch.ones(2, 4, 1, 8), torch.ones(4, 8), torch.ones(8)
    x, a, b, ids = torch.ones(3, 8), torch.ones(2, 4, 8), torch.ones(2, 6, 4), torch.zeros(3, dtype=torch.int64)
    scaling, base = torch.ones(2), torch.ones(3, 6)

    def calls(q, k, cos, sin, w, x, a, b, scaling, base):
        validation.validate_rope_heads(q, k, cos, sin, None)
        validation.validate_head_weight(q, w, "q_weight")
        validation.validate_lora_inputs(x, a, b, ids, scaling, base, None)

    plain = (q, k, t, t.clone(), w, x, a, b, scaling, base)
    calls(*plain)
    with forward_ad.dual_level(), torch.no_grad():
        calls(*plain)
        for i in range(len(plain)):
            dual = forward_ad.make_dual(plain[i], torch.ones_like(plain[i]))
            with pytest.raises(ValueError, match="tangent"):
                calls(*plain[:i], dual, *plain[i + 1:])
