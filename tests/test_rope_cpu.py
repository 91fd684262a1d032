"""CPU: the rotation table."""

import pytest
import torch

from pa_b200 import ops


@pytest.mark.parametrize("rot", [2, 16, 128])
def test_table_holds_cosines_then_sines(rot):
    t = ops.rope_table(9, rot, base=500.0, device="cpu")
    assert t.shape == (9, rot) and t.dtype == torch.float32
    i = torch.arange(rot // 2, dtype=torch.float64)
    ang = torch.arange(9, dtype=torch.float64)[:, None] * 500.0 ** (-2 * i / rot)
    assert float((t[:, :rot // 2] - ang.cos()).abs().max()) <= 2.0 ** -24
    assert float((t[:, rot // 2:] - ang.sin()).abs().max()) <= 2.0 ** -24


@pytest.mark.parametrize("rot", [15, 1, 0, -2])
def test_odd_and_empty_rotations_are_refused(rot):
    """An odd rot_dim gave a table of rot_dim + 1 columns with other frequencies."""
    with pytest.raises(RuntimeError, match="even"):
        ops.rope_table(4, rot, device="cpu")
