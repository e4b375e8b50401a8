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


def test_outputs_that_overlap_inputs_or_each_other_are_refused():
    T, hq, hkv, d = 6, 4, 2, 64
    q, k, v, table, pos = _inputs(T, hq, hkv, d, torch.bfloat16, 1, 50, 1)
    want = layer_ops.rope_axes(q, k, table, pos)
    kv = _cache(hkv, d, torch.bfloat16, [T])
    slots = kv.reserve([0], [0], [T])
    flat = torch.zeros(8192, dtype=q.dtype, device=DEV)
    nq, nk = q.numel(), k.numel()

    def at(first, like):
        return flat[first:first + like.numel()].view(like.shape)

    fresh = at(0, q).copy_(q), at(nq, k).copy_(k)
    free = at(4096, q), at(4096 + nq, k)
    for shift in (8, 64, 256):
        with pytest.raises(ValueError, match="overlap"):
            layer_ops.rope_axes(fresh[0], fresh[1], table, pos, out=(at(shift, q), free[1]))
        with pytest.raises(ValueError, match="overlap"):
            layer_ops.rope_axes(fresh[0], fresh[1], table, pos, out=(free[0], at(nq + shift, k)))
        with pytest.raises(ValueError, match="overlap"):
            layer_ops.rope_axes(fresh[0], None, table, pos, out=(at(shift, q), None))
        with pytest.raises(ValueError, match="overlap"):
            layer_ops.rope_axes(fresh[0], fresh[1], table, pos, out=(free[0], at(4096 + shift, k)))
        for inputs in ((fresh[0], k, v), (q, fresh[1], v), (q, k, fresh[1])):
            out = at(shift, q) if inputs[0] is not q else at(nq + shift, q)
            with pytest.raises(ValueError, match="overlap"):
                kv.append_rotary(0, slots, inputs[1], inputs[2], table, pos, query=inputs[0], query_out=out)
    # an output at the other input's place, and both at one place
    same = at(0, k).copy_(k)
    with pytest.raises(ValueError, match="overlap"):
        layer_ops.rope_axes(same, k, table, pos, out=(free[1], same))
    with pytest.raises(ValueError, match="overlap"):
        layer_ops.rope_axes(k, k, table, pos, out=(free[1], free[1]))
    for out in ((same, free[1]), (free[1], same), (same, same)):  # one tensor as q and k
        with pytest.raises(ValueError, match="overlap"):
            layer_ops.rope_axes(same, same, table, pos, out=out)
    with pytest.raises(ValueError, match="overlap"):
        kv.append_rotary(0, slots, same, v, table, pos, query=same, query_out=same)
    # apart, in place, and in place in the columns of one projection, each twice
    fresh[0].copy_(q), fresh[1].copy_(k)
    for _ in range(2):
        got = layer_ops.rope_axes(fresh[0], fresh[1], table, pos, out=free)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        block = torch.cat((q.reshape(T, -1), k.reshape(T, -1), v.reshape(T, -1)), 1)
        qb, kb = block[:, :hq * d].view(T, hq, d), block[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
        layer_ops.rope_axes(qb, kb, table, pos, out=(qb, kb))
        assert torch.equal(qb, want[0]) and torch.equal(kb, want[1])
        assert torch.equal(block[:, (hq + hkv) * d:], v.reshape(T, -1))
    kv.check_errors()


@pytest.mark.parametrize("dtype,d,rotary", [(torch.bfloat16, 64, 0), (torch.float32, 64, 32), (torch.float16, 10, 0)])
def test_append_rotary_turns_the_query_in_place(dtype, d, rotary):
    """``query_out`` the query itself: padding rows come out zero, the others
    as in a new tensor."""
    T, hq, hkv = 9, 6, 2
    q, k, v, table, pos = _inputs(T, hq, hkv, d, dtype, 1, 50, 4, rotary)
    kv = _cache(hkv, d, dtype, [T])
    slots = kv.reserve([0], [0], [T]).clone()
    slots[[2, 7]] = -1
    want = kv.append_rotary(0, slots, k, v, table, pos, query=q)
    pools = kv._k.clone(), kv._v.clone()
    assert (want[[2, 7]] == 0).all()
    kv._k.zero_(), kv._v.zero_()
    for query in (q.clone(), torch.cat((q, q), 1)[:, :hq]):  # rows back to back, and strided
        got = kv.append_rotary(0, slots, k, v, table, pos, query=query, query_out=query)
        assert got is query and torch.equal(query, want)
        assert torch.equal(kv._k, pools[0]) and torch.equal(kv._v, pools[1])
    kv.check_errors()


def test_wide_slots_do_not_wrap():
    """64-bit slots are those of 32 bits; one past 32 bits lies outside the
    pool, as any other too large, and is not another row's."""
    T = 5
    q, k, v, table, pos = _inputs(T, 4, 2, 64, torch.bfloat16, 1, 50, 1)
    kv = _cache(2, 64, torch.bfloat16, [T])
    slots = kv.reserve([0], [0], [T])
    kv.append_rotary(0, slots, k, v, table, pos)
    want = kv._k.clone(), kv._v.clone()
    kv._k.zero_(), kv._v.zero_()
    kv.append_rotary(0, slots.long(), k, v, table, pos)
    assert torch.equal(kv._k, want[0]) and torch.equal(kv._v, want[1])
    kv.check_errors()
    for far in (2 ** 32, 2 ** 32 + int(slots[1]), 2 ** 31, 2 ** 62):
        kv._k.zero_(), kv._v.zero_()
        wide = slots.long()
        wide[3] = far
        kv.append_rotary(0, wide, k, v, table, pos)
        with pytest.raises(RuntimeError, match="0x10"):
            kv.check_errors()
        live = [0, 1, 2, 4]
        at = slots[live].long()
        assert torch.equal(kv._v[0].view(-1, 2, 64)[at], v[live])
        kv._v[0].view(-1, 2, 64)[at] = 0
        assert (kv._v == 0).all()
    kv._v.zero_()
    wide = slots.long()
    wide[3] = -2 ** 33 + int(slots[0])  # negative: padding
    turned = kv.append_rotary(0, wide, k, v, table, pos, query=q)
    assert (turned[3] == 0).all()
    kv.check_errors()
    for dtype in (torch.float32, torch.bool, torch.bfloat16):
        with pytest.raises(TypeError, match="slots"):
            kv.append_rotary(0, slots.to(dtype), k, v, table, pos)
