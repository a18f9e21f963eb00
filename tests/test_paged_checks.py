"""CPU: what paged attention would refuse is known before rows are appended for it: no workspace size for such a call.

No pointer here is ever dereferenced."""
import pytest

from test_paged_args import CACHE_FAULTS, INVALID, P, _attend, ext

FAR = 1 << 40


# Strides that no tensor map takes: not positive where they are stepped along, 2^40 bytes or more.
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("strides", [(0, 1 << 12, 128), (-(1 << 16), 1 << 12, 128), (1 << 16, 0, 128), (1 << 16, -128, 128),
                                     (1 << 16, 1 << 12, 0), (1 << 16, 1 << 12, -128), (FAR, 1 << 12, 128), (1 << 16, FAR, 128)])
def test_strides_that_no_tensor_map_takes(dtype, strides):
    for rows in (1, 32):
        assert _attend(dtype=dtype, strides=strides, rows=rows) == INVALID
        assert _attend(dtype=dtype, strides=strides, rows=rows, run=False) == 0
        assert _attend(dtype=dtype, rows=rows, run=False) > 0


def test_strides_of_dimensions_of_one_do_not_matter():
    assert _attend(strides=(0, 0, 128), pages=1, heads=1, run=False) > 0


@pytest.mark.parametrize("bad", [b for b, _ in CACHE_FAULTS] + [dict(q=P + 8), dict(q=0), dict(o=P + 2), dict(heads_q=5), dict(rows=0),
                                                               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan"))])
@pytest.mark.parametrize("rows", [1, 400])
def test_a_call_that_would_be_refused_has_no_workspace_size(bad, rows):
    assert _attend(**{"rows": rows, **bad}, run=False) == 0


def _split_bytes(entries, heads, rows, capacity, d):
    return ext._lib.fal_fwd_kvcache_workspace_bytes(entries, heads, rows, capacity, d)


# 32 768 positions: 32 entries of 2 heads of 128, or 64 heads of one, are put in order at a time, and what is left is
# a launch of few thread blocks.
@pytest.mark.parametrize("dtype", [0, 1])
def test_the_keys_of_what_is_left_for_the_last_launch_are_dealt_out_too(dtype):
    def size(**change):
        return _attend(**{**dict(dtype=dtype, rows=400, batch=32, heads=2, heads_q=4, per_entry=2048, run=False), **change})
    alone = _split_bytes(1, 4, 400, 32768, 128)
    assert alone > 0 == _split_bytes(32, 4, 400, 32768, 128)
    assert size(batch=33) - size(batch=32) == alone
    assert size(batch=64) == size(batch=32)
    wide = dict(batch=1, d=128, rows=1100)
    assert _split_bytes(1, 64, 1100, 32768, 128) == 0 < _split_bytes(1, 2, 1100, 32768, 128)
    assert size(heads=66, heads_q=66, **wide) - size(heads=64, heads_q=64, **wide) == _split_bytes(1, 2, 1100, 32768, 128)
