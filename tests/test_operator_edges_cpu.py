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


def _bytes(t):
    """Addresses of every byte of ``t``, with repetitions."""
    import itertools

    out = []
    for at in itertools.product(*(range(n) for n in t.shape)):
        a = t.data_ptr() + t.element_size() * sum(i * st for i, st in zip(at, t.stride()))
        out += range(a, a + t.element_size())
    return out


def test_shared_memory_is_found_byte_by_byte():
    import random

    from engine import _lib

    rng = random.Random(5)
    buf = torch.zeros(400, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    alone = {True: 0, False: 0}

    def view():
        base = buf if rng.random() < 0.7 else buf.view(torch.float32)
        while True:
            shape = [rng.randint(0 if rng.random() < 0.1 else 1, 4) for _ in range(rng.randint(1, 4))]
            stride = [rng.choice([0, 1, 2, 3, 4, 5, 8, 12, 16, 24, 40]) for _ in shape]
            if rng.random() < 0.7:
                stride[-1] = 1
            at = rng.randint(0, 60)
            if at + sum(max(0, n - 1) * st for n, st in zip(shape, stride)) < base.numel():
                return base.as_strided(shape, stride, at)

    for _ in range(1500):
        a, b = view(), view()
        x, y = _bytes(a), _bytes(b)
        assert _lib.overlaps_itself(a) is (len(set(x)) < len(x)), (a.shape, a.stride())
        assert _lib.share_memory(a, b) is bool(set(x) & set(y)), (a.shape, a.stride(), b.shape, b.stride())
        alone[_lib.overlaps_itself(a)] += 1
        seen[_lib.share_memory(a, b)] += 1
    assert min(seen.values()) > 200 and min(alone.values()) > 200
    # column blocks of one wider tensor interleave and share nothing
    wide = torch.zeros(50, 24)
    assert not _lib.share_memory(wide[:, :8], wide[:, 8:16])
    assert _lib.share_memory(wide[:, :9], wide[:, 8:16])
    q = wide[:, :8]
    assert _lib.same_elements(q, q.view(50, 8)) and not _lib.same_elements(q, wide[:, 8:16])
    assert not _lib.same_elements(q, wide.view(torch.int32)[:, :8])


def test_rows_past_32_bits_are_refused():
    """Counts are 32 bits wide below: 2^31 + 1 rows are not one row."""
    import ctypes

    from engine import _lib, layer_ops
    from test_shared_prefix_cpu import _rope

    table = torch.empty((10, 2, 64), device="meta")
    for tokens in (2 ** 31 - 64, 2 ** 31, 2 ** 32 + 1):
        pos = torch.empty(tokens, dtype=torch.int64, device="meta")
        with pytest.raises(ValueError, match="rows"):
            layer_ops._rope_args(table, pos, None, tokens, 64, table.device)
    pos = torch.empty(2 ** 31 - 65, dtype=torch.int64, device="meta")
    assert layer_ops._rope_args(table, pos, None, 2 ** 31 - 65, 64, table.device).num_tokens == 2 ** 31 - 65
    for fn in ("sdl_rope_axes", "sdl_kv_append_rotary"):
        for tokens in (2 ** 31 - 64, 2 ** 31 - 1):
            assert getattr(_lib.load(), fn)(ctypes.byref(_rope(num_tokens=tokens)), None) == 2  # SDL_ERR_UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(B=256, chunk=128, Hq=32, Hkv=8, max_limit=32768),
    dict(B=256, chunk=128, Hq=32, Hkv=8, max_limit=32768, prefix_len=0),
    dict(B=512, chunk=1, Hq=64, Hkv=8, max_limit=40000, key_count=512 * 100),
    dict(B=512, chunk=64, Hq=32, Hkv=8, max_limit=32768, out_dtype=0),          # mma.sync
    dict(B=2000, chunk=64, Hq=4, Hkv=2, head_dim=64, max_limit=32768, dtype=0, out_dtype=0, key_count=2000 * 64),
], ids=str)
def test_the_workspace_of_many_rows_is_bounded(kw):
    """Own ranges take 1 GiB of partials, or one range of all keys; prefix
    ranges one for rows as many as these, or a few."""
    import ctypes

    from engine import _lib
    from test_shared_prefix_cpu import _attn

    x = _attn(**dict(dict(width=4096, capacity=100000), **kw))
    need = _lib.load().sdl_prefix_attention_workspace_bytes(ctypes.byref(x))
    a = x.attn
    one = a.B * a.chunk * a.Hq * (a.head_dim + 2) * 4
    assert 0 < need <= max(one, 2 ** 30) + 4 * one, need / one


def test_the_workspace_of_ordinary_calls_is_as_it_was():
    """Ranges of 512 own keys (mma.sync, 64 decode rows) where they are few."""
    import ctypes

    from engine import _lib
    from test_shared_prefix_cpu import _attn

    x = _attn(B=64, max_limit=32768, width=4096, prefix_len=0, kernel=2)
    need = _lib.load().sdl_prefix_attention_workspace_bytes(ctypes.byref(x))
    assert need == 64 * 12 * 64 * (128 + 2) * 4
