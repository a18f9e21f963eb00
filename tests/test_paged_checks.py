"""CPU: what paged attention would refuse is known before rows are appended for it: no workspace size for such a call.

No pointer here is ever dereferenced."""
import pytest

from test_paged_args import CACHE_FAULTS, INVALID, P, _attend

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
