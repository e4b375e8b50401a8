"""Host-side checks of the rotations and the shared-prefix attention that need
no GPU."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape,index,want", [
    ((4, 3, 8), (slice(None),), True),
    ((4, 3, 16), (slice(None), slice(None), slice(0, 8)), False),
    ((4, 3, 16), (slice(0, 0), slice(None), slice(0, 8)), True),
    ((4, 6, 8), (slice(None), slice(None, None, 2)), False),
    ((4, 6, 8), (slice(0, 0), slice(None, None, 2)), True),
    ((4, 3, 16), (slice(None), slice(0, 0), slice(0, 8)), True),
    ((4, 1, 16), (slice(None), slice(None), slice(0, 8)), True),
])
def test_layouts_that_a_rotation_takes(shape, index, want):
    """What is copied first has to pass afterwards, or the call never ends."""
    from engine import layer_ops

    x = torch.zeros(shape)[index]
    assert layer_ops._has_head_rows(x) is want
    assert layer_ops._has_head_rows(x.contiguous())
