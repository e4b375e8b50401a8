"""Edges of the attention over a shared prefix: bounds below a sequence's
length, masked values at the type's ends, outputs that overlap, plans of very
many rows.  Definition and tolerances as in ``test_shared_prefix_gpu``.
"""

from __future__ import annotations

import pytest
import torch

from engine.attention import SharedPrefixBatch, paged_attention_shared_prefix, prefix_attention_kernel
from test_shared_prefix_gpu import BF, DEV, F32, HF, PLANTS, _build, _check, _exact, _planted, _query

pytestmark = pytest.mark.gpu


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _exact_bounded(q, kv, P, starts, bound):
    """``_exact`` where row j attends min(starts[b] + j + 1, bound) own keys."""
    rows = [_exact(q[:, j:j + 1], kv, 0, P, [max(-1, min(s + j, bound - 1)) for s in starts])
            for j in range(q.shape[1])]
    return tuple(torch.cat(x, 1) for x in zip(*rows))


# (kernel, chunk, d, page size, type): CUDA cores narrow and wide and of another
# head_dim (a lane per dim in the merge), mma.sync, tcgen05 with own items of
# both kinds, the plan's own choice
FORMS = [(1, 4, 64, 4, F32), (1, 30, 64, 16, F32), (1, 4, 20, 16, HF), (2, 4, 128, 16, BF), (2, 9, 64, 16, HF),
         (3, 4, 128, 16, BF), (3, 33, 128, 16, HF), (0, 4, 128, 16, BF), (0, 40, 64, 16, BF)]


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("split", [0, 16, 1000])
def test_a_bound_below_a_length_cuts_the_keys_and_is_reported(form, split):
    kernel, chunk, d, bs, dtype = form
    P, owns = 64, [130, 80]
    kv, g = _build(P, owns, 2, d, bs, dtype, 3)
    q = _query(g, 2, chunk, 8, d, dtype)
    starts = [n - chunk for n in owns]
    w = dtype if dtype != F32 else None

    def call(starts, bound, valid=None):
        return paged_attention_shared_prefix(q, kv, 0, SharedPrefixBatch(0, P, _i32(1, 2), _i32(*starts), bound, valid),
                                             kernel=kernel, own_split=split)

    for use, bound in ((starts, 111), (starts, 129), (starts, 1), (starts, 0), ([2 ** 31 - 1, starts[1]], 130),
                       ([2 ** 31 - 3, -chunk], 100)):
        got = call(use, bound)
        _check(got, _exact_bounded(q, kv, P, use, bound), w)
        with pytest.raises(RuntimeError, match="0x4"):
            kv.check_errors()
    for use, bound in ((starts, 130), (starts, 200), ([-2 ** 31, starts[1]], 80), ([-chunk, -chunk], 0)):
        _check(call(use, bound), _exact_bounded(q, kv, P, use, bound), w)
        kv.check_errors()
    # rows past valid_rows are not written and not reported
    got = call(starts, starts[0] + 2, _i32(2, chunk))
    exact = _exact_bounded(q, kv, P, starts, starts[0] + 2)
    _check(got[0, :2], tuple(x[0, :2] for x in exact), w)
    _check(got[1], tuple(x[1] for x in exact), w)
    kv.check_errors()


@pytest.mark.parametrize("d,hq", [(128, 12), (64, 6)])
def test_a_bound_below_a_length_where_the_merge_attends(d, hq):
    """Sequences with at most a page of own keys, many of them."""
    B, chunk = 170, 2
    kv, g = _build(50, [8] * B, 2, d, 16, BF, 2)
    q = _query(g, B, chunk, hq, d, BF)
    rows = torch.arange(1, B + 1, dtype=torch.int32, device=DEV)
    for P in (50, 0):
        for starts, bound, bad in (([6] * B, 5, True), ([6] * B, 8, False), ([2 ** 31 - 1] + [6] * (B - 1), 8, True),
                                   ([6] * B, 0, True)):
            batch = SharedPrefixBatch(0, P, rows, _i32(*starts), bound)
            _check(paged_attention_shared_prefix(q, kv, 0, batch), _exact_bounded(q, kv, P, starts, bound), BF)
            if bad:
                with pytest.raises(RuntimeError, match="0x4"):
                    kv.check_errors()
            else:
                kv.check_errors()


def _large(dtype):
    """A value of which 2^-126 would still move a row."""
    return 60000.0 if dtype == HF else 2.0 ** 126


@pytest.mark.parametrize("case", PLANTS, ids=str)
def test_a_large_value_behind_a_row_weighs_nothing(case):
    """The largest values of a chunk's later rows do not reach the earlier
    ones, in any column of a tile."""
    kernel, P, before, chunk, d, bs, dtype = case
    kv, batch, q, exact, places = _planted(case, False)
    w = dtype if dtype != F32 else None
    for pos, page, at in places:
        kept = kv._v[0, page, at, 1].clone()
        kv._v[0, page, at, 1] = _large(dtype)
        got = paged_attention_shared_prefix(q, kv, 0, batch, kernel=kernel)
        kv._v[0, page, at, 1] = kept
        first = pos - before
        _check(got[0, :first], tuple(x[0, :first] for x in exact), w) if first else None
        _check(got[0, :, :4], tuple(x[0, :, :4] for x in exact), w)
        _check(got[1], tuple(x[1] for x in exact), w)
    kv.check_errors()


@pytest.mark.parametrize("case", PLANTS, ids=str)
@pytest.mark.parametrize("prefix", [True, False])
@pytest.mark.parametrize("score", [-16.0, float("-inf")])
def test_a_large_value_of_a_key_far_below_weighs_nothing(case, prefix, score):
    """A key whose weight lies below fp32's range, or whose score is -inf."""
    kernel, P, before, chunk, d, bs, dtype = case
    kv, batch, q, exact, places = _planted(case, prefix)
    w = dtype if dtype != F32 else None
    q[..., 4:, :] = q[..., 4:, :].abs() + 0.5  # of kv head 1: scores of -16 sum q / sqrt(d) < -100
    for pos, page, at in places:
        kept = kv._k[0, page, at, 1].clone(), kv._v[0, page, at, 1].clone()
        kv._k[0, page, at, 1] = score
        kv._v[0, page, at, 1] = _large(dtype)
        got = paged_attention_shared_prefix(q, kv, 0, batch, kernel=kernel)
        kv._v[0, page, at, 1] = 0.0
        kv._k[0, page, at, 1] = -16.0  # the scores' rounding bound needs a finite one
        want = _exact(q, kv, 0, P, [before, before])
        kv._k[0, page, at, 1], kv._v[0, page, at, 1] = kept
        _check(got, want, w)
    kv.check_errors()


@pytest.mark.parametrize("kernel", [0, 1])
def test_outputs_that_overlap_are_refused(kernel):
    kv, g = _build(40, [10, 20], 2, 64, 16, BF, 1)
    starts, shape = [8, 18], (2, 2, 4, 64)
    batch = SharedPrefixBatch.from_lists(kv, 0, 40, [1, 2], starts, 2)
    q = _query(g, 2, 2, 4, 64, BF)
    exact = _exact(q, kv, 0, 40, starts)

    def call(query, out):
        return paged_attention_shared_prefix(query, kv, 0, batch, out=out, kernel=kernel)

    flat = torch.zeros(4096, dtype=BF, device=DEV)
    for stride in ((512, 128, 64, 1), (256, 256, 64, 1), (512, 256, 32, 1)):
        with pytest.raises(ValueError, match="overlap"):
            call(q, flat.as_strided(shape, stride))
    n = q.numel()
    for shift in (8, 64, 256, 512):  # the query shifted by a piece, a head, a chunk row, a sequence
        query = flat[:n].view(shape)
        query.copy_(q)
        with pytest.raises(ValueError, match="overlap"):
            call(query, flat[shift:shift + n].view(shape))
        with pytest.raises(ValueError, match="overlap"):
            call(flat[shift:shift + n].view(shape), query)
    query = flat[:n].view(shape)
    with pytest.raises(ValueError, match="overlap"):
        call(query, flat.view(F32)[:n].view(shape))  # of another type at the same place
    # the query itself, the memory behind it, and column blocks of the query's own rows
    query.copy_(q)
    _check(call(query, query), exact, BF if kernel == 0 else None)
    query.copy_(q)
    _check(call(query, flat[n:2 * n].view(shape)), exact, BF if kernel == 0 else None)
    wide = torch.zeros((2, 2, 8 * 64), dtype=BF, device=DEV)
    query, out = (wide[..., i * 256:(i + 1) * 256].view(shape) for i in range(2))
    query.copy_(q)
    for _ in range(2):
        _check(call(query, out), exact, BF if kernel == 0 else None)
    # a query that is copied first (its heads are not unit-stride) may lie where the output goes
    turned = flat[:n].view(2, 2, 64, 4).transpose(2, 3)
    turned.copy_(q)
    _check(call(turned, flat[:n].view(shape)), exact, BF if kernel == 0 else None)
    kv.check_errors()


def test_the_named_kernel_is_the_one_that_runs():
    """For queries that the call copies first: of another type, off 16-byte
    boundaries, with strided dims."""
    P, owns, chunk = 300, [40, 30, 20, 9], 5
    kv, g = _build(P, owns, 2, 128, 16, BF, 8)
    starts = [n - chunk for n in owns]
    batch = SharedPrefixBatch.from_lists(kv, 0, P, [1, 2, 3, 4], starts, chunk)
    q = _query(g, 4, chunk, 12, 128, BF)
    want = paged_attention_shared_prefix(q, kv, 0, batch)
    assert prefix_attention_kernel(q, kv, batch) == "tcgen05"
    assert torch.equal(want, paged_attention_shared_prefix(q, kv, 0, batch, kernel=3))
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape).copy_(q)
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)
    rows = torch.zeros((4, chunk, 12, 130), dtype=BF, device=DEV)[..., :128].copy_(q)
    for same in (q.float(), odd, turned, rows):
        assert prefix_attention_kernel(same, kv, batch) == "tcgen05"
        assert torch.equal(paged_attention_shared_prefix(same, kv, 0, batch), want)
    kv.check_errors()


def test_tensors_set_on_a_batch_in_use_are_checked():
    kv, g = _build(60, [40, 30], 2, 64, 16, BF, 3)
    q = _query(g, 2, 1, 4, 64, BF)
    batch = SharedPrefixBatch.from_lists(kv, 0, 60, [1, 2], [39, 29], 1)
    exact = _exact(q, kv, 0, 60, [39, 29])
    _check(paged_attention_shared_prefix(q, kv, 0, batch), exact, BF)
    for name, value in (("starts", torch.tensor([39, 29], device=DEV)), ("starts", _i32(39)), ("rows", _i32(1)),
                        ("rows", _i32(1, 7, 2, 7)[::2]), ("valid_rows", _i32(1, 1, 1)),
                        ("valid_rows", torch.ones(2, device=DEV)), ("starts", _i32(39, 29)[:, None])):
        kept = getattr(batch, name)
        setattr(batch, name, value)
        with pytest.raises(ValueError, match="int32"):
            paged_attention_shared_prefix(q, kv, 0, batch)
        setattr(batch, name, kept)
    batch.starts = torch.tensor([39, 29], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention_shared_prefix(q, kv, 0, batch)
    batch.starts = _i32(39, 29)
    _check(paged_attention_shared_prefix(q, kv, 0, batch), exact, BF)
    kv.check_errors()


@pytest.mark.parametrize("kernel", [0, 2])
def test_own_ranges_that_grow_for_many_rows(kernel):
    """A bound whose partials would pass the workspace's: 32768 rows of up to
    40000 own keys, of which one sequence has many."""
    B, P, hq, hkv, d = 512, 70, 64, 8, 128
    owns = [1 + i % 90 for i in range(B)]
    owns[300] = 20011
    kv, g = _build(P, owns, hkv, d, 16, BF, 6, extra=2600)
    q = _query(g, B, 1, hq, d, BF)
    starts = [n - 1 for n in owns]
    rows = torch.arange(1, B + 1, dtype=torch.int32, device=DEV)
    batch = SharedPrefixBatch(0, P, rows, _i32(*starts), 40000)
    got = paged_attention_shared_prefix(q, kv, 0, batch, kernel=kernel)
    _check(got, _exact(q, kv, 0, P, starts), BF)
    kv.check_errors()


@pytest.mark.parametrize("case", PLANTS, ids=str)
def test_rows_of_nothing_but_infinitely_low_scores_are_zero(case):
    kernel, P, before, chunk, d, bs, dtype = case
    kv, batch, q, exact, _ = _planted(case, True)
    q[..., 4:, :] = q[..., 4:, :].abs() + 0.5
    kv._k[:, :, :, 1] = float("-inf")  # every key of kv head 1
    kv._v[:, :, :, 1].nan_to_num_(2.0)
    got = paged_attention_shared_prefix(q, kv, 0, batch, kernel=kernel)
    assert (got[:, :, 4:] == 0).all()
    _check(got[:, :, :4], tuple(x[:, :, :4] for x in exact), dtype if dtype != F32 else None)
    kv.check_errors()
