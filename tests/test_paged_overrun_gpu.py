"""GPU: a call whose new tokens run over the end of an entry's block table.  The tokens that fit see what they would see in a
longer table, those without a place give 0, and the status word reports it."""
import math

import pytest
import torch

from paged_reference import assert_close, attention, rotate
from test_paged_gpu import DTYPES, _filled, _lens, _rows, _tables

pytestmark = pytest.mark.gpu


def _run_over(ext, fal, dtype, rows, hq, hkv, d, page, width, lens, rotated, layout, native, monkeypatch):
    gen = torch.Generator().manual_seed(rows + width)
    capacity = width * page
    cache = _filled(gen, DTYPES[dtype], [min(n, capacity) for n in lens], page, hkv, d, extra=rows)
    cache.table = cache.table[:, :width].contiguous()
    cos, sin = _tables(capacity, d)
    got = cache.on_gpu(layout)
    q, k, v = (_rows(gen, len(lens), rows, h, d) for h in (hq, hkv, hkv))
    turning = dict(rotary_cos=cos.cuda(), rotary_sin=sin.cuda()) if rotated else {}
    ext.reset_device_status()
    if not native:
        monkeypatch.setattr(ext, "paged_attend_plain", ext._general)
        monkeypatch.setattr(ext, "paged_append_plain", ext._general)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens), k=k.cuda(), v=v.cuda(),
                                          cache_layout=layout, **turning, **got).cpu()
    over = any(n >= 0 and n + rows > capacity for n in lens)
    assert ext.device_status() == (2000 if over else 0)
    ext.reset_device_status()
    for e, n in enumerate(lens):
        fit = 0 if n < 0 else max(min(rows, capacity - n), 0)
        assert not o[e, fit:].any()
        if fit == 0:
            continue
        turn = (lambda x: rotate(x[e, :fit], n, cos, sin, False)) if rotated else (lambda x: x[e, :fit])
        cache.append(e, turn(k), v[e, :fit])
        kd, vd = cache.dense(e, n + fit)
        want, mag = attention(turn(q), kd, vd, 1 / math.sqrt(d))
        assert_close(o[e, :fit], want, mag, n + fit, vd.abs().max().item())
    cache.check(got, layout)


@pytest.fixture()
def ext():
    import flash_attn_legacy_cuda as m
    m.reset_device_status()
    yield m
    m.reset_device_status()


@pytest.fixture()
def fal():
    import flash_attn_legacy as m
    return m


# Entries that run over in the middle, by one, by all but one, that are full or beyond it, unused, that just fit; up to 32 tokens
# and more, in one tile and several, keys of a block dealt to several thread blocks (2 048 positions), one token.
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("rows,hq,hkv,d,page,width,lens,layout", [
    (20, 4, 2, 64, 16, 3, [40, 10, -1, 48, 47, 29, 28, 3, 60], "bshd"),
    (1, 8, 2, 128, 32, 4, [127, 128, 5, -3, 0], "bhsd"),
    (5, 16, 1, 128, 16, 70, [1117, 1119, 1120, 1115, 600], "bshd"),
    (32, 2, 1, 256, 16, 5, [60, 48, 49, 80], "bhsd"),
    (40, 4, 2, 64, 32, 3, [70, 56, 57, 96, -1, 95, 10], "bshd"),
    (150, 4, 4, 128, 16, 20, [200, 170, 171, 320, 319, 0], "bhsd"),
    (300, 2, 2, 64, 64, 8, [300, 212, 213, 511, 100], "bshd"),
    (60, 2, 1, 128, 64, 32, [2030, 1988, 1000, 2048, -1], "bshd"),
    (70, 2, 2, 256, 128, 3, [350, 384, 20], "bshd")])
def test_tokens_that_fit_see_their_own_positions(ext, fal, monkeypatch, dtype, native, rotated, rows, hq, hkv, d, page, width, lens, layout):
    _run_over(ext, fal, dtype, rows, hq, hkv, d, page, width, lens, rotated, layout, native, monkeypatch)


@pytest.mark.parametrize("rows", [6, 50])
def test_tokens_without_a_place_give_zeros_whatever_the_cache_holds(ext, fal, rows):
    gen = torch.Generator().manual_seed(3)
    cache = _filled(gen, torch.float16, [30, 2000], 16, 2, 64, extra=rows)
    cache.table = cache.table[:, :125].contiguous()  # 2 000 positions
    got = cache.on_gpu("bshd")
    got["v_pages"][cache.table[1, 0].item(), 3] = math.inf
    got["v_pages"][cache.table[1, 124].item(), 15] = math.nan
    q, k, v = (_rows(gen, 2, rows, h, 64).cuda() for h in (4, 2, 2))
    o = fal.flash_attn_with_paged_kvcache(q, block_table=cache.table.cuda(), cache_seqlens=_lens([30, 2000]), k=k, v=v, **got)
    assert not o[1].any() and not o[0].isnan().any()


@pytest.mark.parametrize("rows", [2, 40])
def test_captured_steps_run_into_the_end_of_their_table(ext, fal, rows):
    """Lengths moved on inside the graph, beyond the capacity: each replay as the eager call."""
    gen = torch.Generator().manual_seed(4)
    width = rows // 4 + 4
    room = 2 * rows - rows // 2
    lens = [width * 16 - room, 20]
    cache = _filled(gen, torch.int8, lens, 16, 2, 64, extra=4 * rows)
    cache.table = cache.table[:, :width].contiguous()
    at, table = _lens(lens), cache.table.cuda()
    q, k, v = (_rows(gen, 2, rows, h, 64).cuda() for h in (4, 2, 2))
    got, eager = cache.on_gpu("bshd"), cache.on_gpu("bshd")
    inside = at.clone()
    fal.flash_attn_with_paged_kvcache(q, block_table=table, cache_seqlens=at, k=k, v=v, **{n: t.clone() for n, t in got.items()})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = fal.flash_attn_with_paged_kvcache(q, block_table=table, cache_seqlens=inside, k=k, v=v, **got)
        inside += rows
    dropped = []
    for _ in range(4):
        graph.replay()
        want = fal.flash_attn_with_paged_kvcache(q, block_table=table, cache_seqlens=at, k=k, v=v, **eager)
        at += rows
        assert torch.equal(o, want)
        for n in got:
            assert torch.equal(got[n].view(torch.uint8), eager[n].view(torch.uint8))
        dropped.append(int((o[0] == 0).all(dim=-1).all(dim=-1).sum()))
    assert dropped == [min(max((i + 1) * rows - room, 0), rows) for i in range(4)] and dropped[0] == 0 and dropped[-1] == rows


# Tables so long that the entries, or the KV heads of one, are put in order a few at a time: as each of them alone.
@pytest.mark.parametrize("dtype", ["fp16", "int8"])
@pytest.mark.parametrize("hq,hkv,d,width,ends", [(4, 2, 64, 2048, [-30, None, -7, 5000, 0, -40, 600]), (8, 4, 128, 4096, [-30, None, 300])])
def test_entries_a_few_at_a_time(ext, fal, dtype, hq, hkv, d, width, ends):
    gen = torch.Generator().manual_seed(width)
    page, rows, pool = 256, 40, 24
    capacity, batch = page * width, len(ends)
    lens = torch.tensor([-2 if n is None else n + capacity if n <= 0 else n for n in ends], dtype=torch.int32).cuda()
    # every position has a page, most of them several times; the pages that new rows go to are an entry's own
    table = torch.randint(0, pool, (batch, width), generator=gen, dtype=torch.int32)
    for e, n in enumerate(lens.tolist()):
        if n >= 0:
            for i in range(n // page, min(n // page + 2, width)):
                table[e, i] = pool + 2 * e + i % 2
    table = table.cuda()
    shape = (pool + 2 * batch, page, hkv, d)
    caches = {}
    for n in ("k", "v"):
        x = _rows(gen, *shape).cuda()
        if dtype == "fp16":
            caches[n + "_pages"] = x
        else:
            caches[n + "_pages"] = (x.float() * 28).clamp(-127, 127).to(torch.int8)
            caches[n + "_scales"] = (torch.rand(shape[0], hkv, generator=gen) / 50 + 0.01).cuda()
            caches[n + "_tail"] = _rows(gen, batch, page, hkv, d).cuda()
    q, k, v = (_rows(gen, batch, rows, h, d).cuda() for h in (hq, hkv, hkv))
    start = {n: t.clone() for n, t in caches.items()}
    o = fal.flash_attn_with_paged_kvcache(q, block_table=table, cache_seqlens=lens, k=k, v=v, softmax_scale=0.5, **caches)
    assert ext.device_status() == 2000
    for e in range(batch):
        one = slice(e, e + 1)
        alone = {n: (t[one].clone() if n.endswith("tail") else t.clone()) for n, t in start.items()}
        used = max(min(int(lens[e]) + rows + page - 1, capacity) // page, 1)  # (a table no longer than the entry needs)
        want = fal.flash_attn_with_paged_kvcache(q[one], block_table=table[one, :used], cache_seqlens=lens[one], k=k[one], v=v[one],
                                                 softmax_scale=0.5, **alone)
        # each: its output's rounding and its weights', 2^-11 of values below 6 each
        assert float((o[one].double() - want.double()).abs().max()) <= 2 * 2 * 2.0 ** -11 * 6
        placed = 0 if ends[e] is None else min(rows, capacity - int(lens[e]))
        assert not o[e, placed:].any() and bool(o[e, :placed].any(dim=-1).all())
