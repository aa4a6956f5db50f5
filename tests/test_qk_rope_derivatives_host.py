"""Host logic of the query/key path without a GPU: what torch's default device and derivatives have to do with it."""

import torch


def test_the_frequencies_lie_in_host_memory_whatever_the_default_device():
    """The library reads them on the host."""
    from triton_ops.kernels.rope import _turns

    with torch.device("meta"):
        array, turns, _ = _turns(34, 12345.0, None)
    assert turns.device.type == "cpu" and turns.dtype == torch.float64 and turns.is_contiguous()
    assert turns.tolist() == list(array) and len(array) == 17
    assert _turns(34, 12345.0, None)[1].device.type == "cpu"
