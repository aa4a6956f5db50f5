"""rope_tables, fused_rope and fused_qk_norm_rope on the GPU: torch's default device, derivatives, small angles."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extension", [True, False])
def test_tables_under_a_default_device(cuda, monkeypatch, extension):
    """The frequencies are read on the host, also when the first call with them comes under another default device."""
    from triton_ops import RoPEScaling, _lib, rope_tables

    if not extension:
        monkeypatch.setattr(_lib, "ext", lambda: None)
    at = torch.tensor([0, 1, 77, 4096], device="cuda")
    base = 4321.0 + extension  # a key of its own
    for scaling in (None, RoPEScaling("yarn", 4.0, 2048)):
        with torch.device("cuda"):
            inside = [*rope_tables(at, 48, base, scaling), *rope_tables(5, 48, base, scaling)]
        outside = [*rope_tables(at, 48, base, scaling), *rope_tables(5, 48, base, scaling)]
        assert all(torch.equal(a, b) for a, b in zip(inside, outside))
        assert torch.equal(inside[2][0], inside[0][0]) and inside[2].device == at.device


def test_the_extension_takes_frequencies_from_the_host_alone(cuda):
    from triton_ops import _lib

    at = torch.arange(3, device="cuda")
    turns = torch.rand(4, dtype=torch.float64)
    assert _lib.ext().rope_tables(at, turns, 1.0, _lib.F32) is not None
    for other in (turns.cuda(), turns.float(), torch.rand(8, dtype=torch.float64)[::2]):
        assert _lib.ext().rope_tables(at, other, 1.0, _lib.F32) is None
