"""Arguments of the norm and dropout functions that must be refused before anything is launched."""

import pytest
import torch

from mhc import ops

ROWS = [2 ** 64, 2 ** 64 + 5, 2 ** 63, -2 ** 63 - 1, -2 ** 64]


@pytest.mark.parametrize("row_offset", ROWS)
def test_row_offset_past_64_bits(row_offset, monkeypatch):
    """Such a number would reach the library with its upper bits cut off, as another row."""
    def launched(*a, **k):
        raise AssertionError("launched")

    for name in ("counter_dropout_forward", "add_rms_norm_forward", "add_residual_dropout_forward"):
        monkeypatch.setattr(ops, name, launched)
    x, H, post = torch.randn(3, 16), torch.randn(1, 3, 4, 16), torch.rand(1, 4)
    rng = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.counter_dropout(x, 0.5, rng, row_offset),
                 lambda: ops.fused_add_rms_norm(x, None, None, dropout_p=0.5, rng=rng, row_offset=row_offset),
                 lambda: ops.fused_add_residual(H, x.view(1, 3, 16), post, dropout_p=0.5, rng=rng, row_offset=row_offset),
                 lambda: ops.add_residual_from_state(H, H, torch.rand(1, 4, 4), x.view(1, 3, 16), post, False, 0.5, rng, row_offset)):
        with pytest.raises(ValueError, match="row_offset"):
            call()
