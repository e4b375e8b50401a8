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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rotary,sections", SPLITS)
@pytest.mark.parametrize("heads", [(3, 2), (0, 2)])
def test_the_c_entry_reports_a_bad_position_of_any_axis(dtype, d, rotary, sections, heads):
    import ctypes

    from engine import _lib

    axes = len(sections)
    q, k, _, table, pos = _inputs(3, 3, 2, d, dtype, axes, 50, d, rotary)
    q, k, pos = q.contiguous(), k.contiguous(), pos.contiguous()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    a = _lib.SdlRopeArgs()
    if heads[0]:
        a.q = a.q_out = q.data_ptr()
        a.q_row_stride = a.q_out_row_stride = 3 * d
    a.k = a.k_out = k.data_ptr()
    a.k_row_stride = a.k_out_row_stride = 2 * d
    a.table, a.table_rows, a.positions, a.pos_stride, a.pos64 = table.data_ptr(), 50, pos.data_ptr(), 3, 1
    a.err, a.axes, a.num_tokens, a.head_dim, a.rotary = err.data_ptr(), axes, 3, d, rotary
    a.Hq, a.Hkv, a.dtype = heads[0], heads[1], _lib.dtype_code(dtype)
    for i, n in enumerate(sections):
        a.sections[i] = n
    _lib.check(_lib.load().sdl_rope_axes(ctypes.byref(a), _lib.stream_handle(DEV)), "sdl_rope_axes")
    assert int(err) == 0
    for axis, n in enumerate(sections):
        for row, value in ((0, 50), (2, -1)):
            kept = pos[axis, row].clone()
            pos[axis, row] = value
            err.zero_()
            _lib.check(_lib.load().sdl_rope_axes(ctypes.byref(a), _lib.stream_handle(DEV)), "sdl_rope_axes")
            assert int(err) == (0x4 if n else 0)  # an axis without pairs turns nothing
            pos[axis, row] = kept


@pytest.mark.parametrize("heads", [1, 2, 5])
def test_empty_calls_of_sliced_tensors(heads):
    """No tokens, with the strides of a slice; no heads."""
    q, k, v, table, pos = _inputs(4, heads, 2, 64, torch.bfloat16, 1, 50, 1, rotary=32)
    wide = torch.zeros((4, heads, 128), dtype=q.dtype, device=DEV)[..., :64]
    pair = torch.zeros((4, 2, 128), dtype=q.dtype, device=DEV)[:, :, ::2]
    kv = _cache(2, 64, torch.bfloat16, [4])
    slots = kv.reserve([0], [0], [4])[:0]
    for a in (wide[:0], q[:0], wide.transpose(0, 1)[:, :0].transpose(0, 1)):
        for b in (pair[:0], k[:0]):
            out = layer_ops.rope_axes(a, b, table, pos[:0])
            assert out[0].shape == (0, heads, 64) and out[1].shape == (0, 2, 64)
            given = torch.empty_like(q[:0]), torch.empty_like(k[:0])
            assert layer_ops.rope_axes(a, b, table, pos[:0], out=given)[0] is given[0]
            assert kv.append_rotary(0, slots, b, b, table, pos[:0], query=a).shape == (0, heads, 64)
            assert kv.append_rotary(0, slots, b, pair[:0], table, pos[:0]) is None
    none = wide[:, :0]
    turned, other = layer_ops.rope_axes(none, k, table, pos)
    assert turned.shape == (4, 0, 64)
    _check(other, k, table, pos, None)
    kv.check_errors()
