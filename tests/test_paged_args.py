"""CPU: argument checks of the paged cache's C entries, their workspace sizes, and what the Python entries refuse.

No pointer here is ever dereferenced: every call ends in a check (or, with good arguments, at the missing GPU)."""
import ctypes

import pytest
import torch

ext = pytest.importorskip("flash_attn_legacy_cuda")
import flash_attn_legacy as fal  # noqa: E402

INVALID, BAD_HEAD_DIM, TOO_SMALL = -1, -2, -3
NO_GPU = {-4, -6}
P = 256  # an aligned address


def _cache(dtype=0, k_pages=P, scales=P, tail=P, table=P, lens=P, strides=(1 << 16, 1 << 12, 128), tail_strides=(1 << 16, 1 << 12, 128),
           pages=100, page=16, per_entry=10, batch=2, heads=2, d=128):
    if dtype == 0:
        scales = tail = 0
    return (k_pages, P, scales, scales, tail, tail, table, lens, *strides * 2, *tail_strides * 2, per_entry, dtype, pages, page,
            per_entry, batch, heads, d, 0)


def _append(q=P, k=P, q_out=P, cos=P, sin=P, new=P, heads_q=4, rows=3, rotary_dim=64, positions=160, q_stride=128, **cache):
    return ext._lib.fal_paged_append_run(ext._PAGED_APPEND_ARGS.pack(
        *_cache(**cache), q, k, P, q_out, cos, sin, new, *(1 << 12, q_stride, 1 << 9) * 3, heads_q, rows, rotary_dim, 0, 0, positions, 0, 0))


def _attend(q=P, o=P, heads_q=4, rows=1, scale=0.1, ws=P, nbytes=1 << 40, run=True, **cache):
    block = ext._PAGED_ATTN_ARGS.pack(*_cache(**cache), q, o, 1 << 12, 128, 1 << 9, heads_q, rows, scale, 0, ws, nbytes, 0, 0)
    return ext._lib.fal_paged_attn_run(block) if run else ext._lib.fal_paged_attn_workspace_bytes(block)


CACHE_FAULTS = [({"k_pages": 0}, INVALID), ({"k_pages": P + 8}, INVALID), ({"table": 0}, INVALID), ({"lens": 0}, INVALID),
                ({"dtype": 3}, INVALID), ({"dtype": -1}, INVALID), ({"dtype": 1, "scales": 0}, INVALID), ({"dtype": 2, "tail": 0}, INVALID),
                ({"dtype": 1, "tail": P + 2}, INVALID), ({"strides": (1 << 16, 1 << 12, 132)}, INVALID),
                ({"dtype": 1, "strides": (1 << 16, 1 << 12, 136)}, INVALID), ({"dtype": 1, "tail_strides": (1 << 16, 4, 128)}, INVALID),
                ({"pages": 0}, INVALID), ({"page": 8}, INVALID), ({"page": 48}, INVALID), ({"page": 512}, INVALID), ({"per_entry": 0}, INVALID),
                ({"per_entry": 1 << 27}, INVALID), ({"batch": 0}, INVALID), ({"batch": 65536}, INVALID), ({"heads": 0}, INVALID),
                ({"d": 80}, BAD_HEAD_DIM)]


@pytest.mark.parametrize("bad,code", CACHE_FAULTS)
def test_both_entries_check_the_cache(bad, code):
    assert _append(**bad) == code
    assert _attend(**bad) == code


@pytest.mark.parametrize("bad", [{"k": 0}, {"k": P + 4}, {"new": 0}, {"rows": 0}, {"q": 0}, {"q_out": 0}, {"heads_q": 0}, {"heads_q": -1},
                                 {"cos": 0}, {"sin": 0}, {"sin": P + 4}, {"rotary_dim": 24}, {"rotary_dim": 0}, {"rotary_dim": 144},
                                 {"positions": 159}, {"q_stride": 129}])
def test_append_checks_its_rows(bad):
    assert _append(**bad) == INVALID


@pytest.mark.parametrize("bad,code", [({"q": 0}, INVALID), ({"o": 0}, INVALID), ({"o": P + 2}, INVALID), ({"heads_q": 5}, INVALID),
                                      ({"rows": 0}, INVALID), ({"scale": 0.0}, INVALID), ({"scale": float("nan")}, INVALID), ({"ws": 0}, INVALID),
                                      ({"ws": P + 4}, INVALID), ({"nbytes": 10}, TOO_SMALL), ({"rows": 500, "nbytes": 10}, TOO_SMALL)])
def test_attention_checks_its_queries_and_workspace(bad, code):
    assert _attend(**bad) == code


def test_null_blocks_and_blocks_of_zeros_are_refused():
    for run, layout in ((ext._lib.fal_paged_append_run, ext._PAGED_APPEND_ARGS), (ext._lib.fal_paged_attn_run, ext._PAGED_ATTN_ARGS)):
        assert run(bytes(layout.size)) == INVALID
        assert run(ctypes.c_char_p(None)) == INVALID
    assert ext._lib.fal_paged_attn_workspace_bytes(bytes(ext._PAGED_ATTN_ARGS.size)) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="good arguments with addresses that nothing is at")
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_good_arguments_end_at_the_missing_gpu(dtype):
    assert _append(dtype=dtype) in NO_GPU
    assert _append(dtype=dtype, q=0, q_out=0, heads_q=0, cos=0, sin=0, rotary_dim=0, positions=0) in NO_GPU
    for rows in (1, 5, 400):
        assert _attend(dtype=dtype, rows=rows) in NO_GPU


def test_the_workspace_of_many_rows_stays_bounded():
    one = _attend(rows=400, run=False)
    assert one >= 2 * 2 * 2 * 160 * 128 * 2  # all entries' K and V rows as fp16
    # 32 entries of 131 072 positions: as many at a time as 1 GiB holds; then fewer heads, at the least one
    kv = 131072 * 128 * 2 * 2
    for heads, at_once in ((8, 8 * 2), (64, 16)):
        got = _attend(rows=400, heads=heads, heads_q=heads, batch=32, per_entry=8192, run=False)
        assert at_once * kv <= got <= 1.1 * at_once * kv
    got = _attend(rows=400, d=256, per_entry=1 << 22, page=256, run=False)
    assert got >= (1 << 30) * 256 * 2 * 2


def test_python_entries_want_gpu_tensors_of_their_types():
    q, kv = torch.zeros(2, 1, 4, 64).half(), torch.zeros(2, 1, 2, 64).half()
    pages = torch.zeros(4, 16, 2, 64).half()
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        fal.flash_attn_with_paged_kvcache(q, pages, pages.clone(), table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        fal.paged_cache_append(kv, kv, pages, pages.clone(), table, lens)
    with pytest.raises(AssertionError):
        fal.flash_attn_with_paged_kvcache(q.float(), pages, pages, table, lens)
    with pytest.raises(AssertionError):
        fal.paged_cache_append(kv.bfloat16(), kv, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="inference only"):
        fal.paged_cache_append(kv.clone().requires_grad_(), kv, pages, pages, table, lens)
