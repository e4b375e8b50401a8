"""Edges of the rotations: positions outside the table, empty and overlapping
tensors, in-place calls.  Formula and tolerances as in ``test_rotary_gpu``.
"""

from __future__ import annotations

import pytest
import torch

from engine import layer_ops
from test_rotary_gpu import DEV, _cache, _check, _inputs

pytestmark = pytest.mark.gpu

# (head_dim, rotary width, sections): sections that end inside a 16-byte piece
# of every type, on a piece's end, a partly turned head, the element-wise kernel
SPLITS = [(64, 64, (31, 1)), (64, 64, (1, 31)), (128, 128, (3, 0, 50, 11)), (64, 32, (8, 8)), (64, 32, (5, 11)),
          (10, 10, (2, 3))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rotary,sections", SPLITS)
def test_a_bad_position_spoils_its_own_pairs_alone(dtype, d, rotary, sections):
    axes, half, reach = len(sections), rotary // 2, 50
    q, k, _, table, pos = _inputs(2 * axes + 1, 3, 2, d, dtype, axes, reach, d, rotary)
    want = layer_ops.rope_axes(q, k, table, pos, sections)
    bad = pos.clone()
    for a in range(axes):  # one bad position in each row but the last
        bad[a, 2 * a] = reach
        bad[a, 2 * a + 1] = -1
    got = layer_ops.rope_axes(q, k, table, bad, sections)
    first = 0
    lost = torch.zeros((2 * axes + 1, d), dtype=torch.bool, device=DEV)
    for a, n in enumerate(sections):
        for lo in (first, first + half):
            lost[2 * a:2 * a + 2, lo:lo + n] = True
        first += n
    for x, y in zip(got, want):
        spoiled = lost[:, None].expand_as(x)
        assert torch.isnan(x[spoiled]).all()
        assert torch.equal(x[~spoiled], y[~spoiled])
    # the append stores such a row nowhere; its query comes out the same
    kv = _cache(2, d, dtype, [2 * axes + 1])
    slots = kv.reserve([0], [0], [2 * axes + 1])
    turned = kv.append_rotary(0, slots, k, k, table, bad, sections, query=q)
    with pytest.raises(RuntimeError, match="0x4"):
        kv.check_errors()
    assert torch.equal(turned.nan_to_num(9.0), got[0].nan_to_num(9.0))
    rows = kv._k[0].view(-1, 2, d)[slots.long()]
    assert (rows[:-1] == 0).all() and torch.equal(rows[-1], want[1][-1])
