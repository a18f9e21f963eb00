"""GPU: paged caches against plain models -- append with rotation bit for bit, attention over the pages to rounding."""
import math

import pytest
import torch

from paged_reference import Cache, assert_close, attention, rotate

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


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


def _rows(gen, *shape):
    return torch.randn(*shape, generator=gen).half()


def _tables(positions, rotary_dim):
    half = rotary_dim // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half) / half)[None]
    return angle.cos().float(), angle.sin().float()


def _filled(gen, dtype, lens, page, hkv, d, extra=0, spare=2):
    """A cache with lens[b] rows in entry b (negative: unused) and room for `extra` more."""
    width = (max(max(lens), 0) + extra) // page + 2
    pages = sum((max(n, 0) + extra + page - 1) // page for n in lens) + spare
    cache = Cache(gen, dtype, pages, page, hkv, d, len(lens), width)
    for e, n in enumerate(lens):
        if n >= 0:
            cache.reserve(e, n + extra)
            cache.append(e, _rows(gen, n, hkv, d), _rows(gen, n, hkv, d))
    return cache


def _lens(lens):
    return torch.tensor(lens, dtype=torch.int32).cuda()


# Chunks that start and end on, before and behind a page border, whole pages, several pages, one row; entries that are empty,
# that are full and that are unused; every head_dim; both rotations, all or half of the columns.
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d,page,layout", [(4, 2, 128, 16, "bshd"), (2, 1, 64, 32, "bhsd"), (3, 3, 32, 64, "bshd"),
                                                 (8, 2, 96, 16, "bhsd"), (2, 2, 256, 128, "bshd"), (5, 1, 128, 256, "bhsd")])
@pytest.mark.parametrize("rows", [1, 5, 16, 33, 300])
def test_append_writes_what_the_model_writes(ext, fal, dtype, hq, hkv, d, page, layout, rows):
    gen = torch.Generator().manual_seed(d + rows)
    lens = [0, 1, page - 1, page, 2 * page + 7, -1, 3 * page - rows % page]
    cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d, extra=rows)
    interleaved, rotary_dim = rows % 2 == 1, d if rows % 3 else d // 2
    cos, sin = _tables(cache.table.shape[1] * page, rotary_dim)
    if rows == 33:
        cos, sin = cos.half(), sin.half()
    got = cache.on_gpu(layout)
    q, k, v = (_rows(gen, len(lens), rows, h, d) for h in (hq, hkv, hkv))
    q_out, new = fal.paged_cache_append(k.cuda(), v.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens), q=q.cuda(),
                                        rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=interleaved,
                                        cache_layout=layout, **got)
    for e, n in enumerate(lens):
        if n >= 0:
            cache.append(e, rotate(k[e], n, cos, sin, interleaved), v[e])
            assert torch.equal(q_out[e].cpu(), rotate(q[e], n, cos, sin, interleaved))
        else:
            assert not q_out[e].any()
    cache.check(got, layout)
    assert new.tolist() == [n + rows if n >= 0 else n for n in lens]
    assert ext.device_status() == 0


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_8_bit_pages_do_not_depend_on_how_the_rows_came_in(fal, dtype):
    gen = torch.Generator().manual_seed(9)
    page, hkv, d, total = 16, 2, 64, 75
    k, v = _rows(gen, 2, total, hkv, d).cuda(), _rows(gen, 2, total, hkv, d).cuda()
    ends = []
    for steps in ([total], [1] * total, [3, 20, 1, 51], [16, 16, 43]):
        cache = _filled(torch.Generator().manual_seed(4), DTYPES[dtype], [0, 0], page, hkv, d, extra=total)
        got, lens, at = cache.on_gpu("bshd"), _lens([0, 0]), 0
        for n in steps:
            _, lens = fal.paged_cache_append(k[:, at:at + n], v[:, at:at + n], block_table=cache.table.cuda(), cache_seqlens=lens, **got)
            at += n
        left = total % page
        got["k_tail"], got["v_tail"] = got["k_tail"][:, :left], got["v_tail"][:, :left]
        ends.append([got[n].view(torch.uint8) for n in sorted(got) if not n.endswith("tail")] + [got["k_tail"], got["v_tail"]])
    for other in ends[1:]:
        assert all(torch.equal(a, b) for a, b in zip(ends[0], other))


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_what_8_bit_pages_make_of_special_values(fal, dtype):
    """Zeros, the smallest and the largest fp16 numbers, ties, an infinity, a NaN: one head each of one page."""
    page, d = 16, 32
    specials = [0.0, 2.0 ** -24, 65504.0, 1.0, math.inf, math.nan]
    gen = torch.Generator().manual_seed(1)
    k = (torch.rand(1, page, len(specials), d, generator=gen) - 0.5).half()
    for h, x in enumerate(specials):
        k[0, :, h] = 0 if x == 0 else (k[0, :, h] * (x if math.isfinite(x) else 1)).half()
        k[0, 3, h, 5] = x
        if x == 1.0:
            k[0, 4, h, :8] = torch.tensor([0.5, -0.5, 63.5 / 127, 0.25, 1.3125 * 2 / 7, 0.75, -1.0, 2.0 ** -9]).half()
    cache = Cache(gen, DTYPES[dtype], 2, page, len(specials), d, 1, 1)
    cache.reserve(0, page)
    got = cache.on_gpu("bshd")
    fal.paged_cache_append(k.cuda(), k.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens([0]), **got)
    cache.append(0, k[0], k[0])
    for n in ("k_pages", "v_pages"):
        assert torch.equal(got[n].cpu().view(torch.uint8), cache.tensors[n].view(torch.uint8))
    scales, want = got["k_scales"].cpu(), cache.tensors["k_scales"]
    assert torch.equal(scales.isnan(), want.isnan()) and torch.equal(scales.nan_to_num(), want.nan_to_num())
    assert scales[cache.table[0, 0]].isnan().tolist() == [not math.isfinite(x) for x in specials]


# Lengths around page, slice and split borders, empty and unused entries; one and several query tokens, up to where the
# split-K pass hands over to the forward kernel and beyond; one, several and many query heads per KV head.
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d,page,layout", [(8, 2, 128, 16, "bshd"), (16, 1, 64, 64, "bhsd"), (3, 3, 32, 32, "bshd"),
                                                 (20, 1, 96, 16, "bhsd"), (4, 2, 256, 128, "bshd"), (6, 6, 128, 256, "bhsd")])
@pytest.mark.parametrize("rows,lens", [(1, [1, 15, 16, 17, 255, 256, 257, 0, -1]), (1, [2049]), (1, [700, 9, 4100]),
                                       (3, [3, 1, 16, 300, 0, -1, 35]), (16, [16, 40, 513, 7]), (130, [130, 200, 1000, 0, 64, -5])])
def test_attention_over_pages(ext, fal, dtype, hq, hkv, d, page, layout, rows, lens):
    gen = torch.Generator().manual_seed(hq * d + rows)
    cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d)
    q = _rows(gen, len(lens), rows, hq, d)
    scale = 1 / math.sqrt(d)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens),
                                          cache_layout=layout, **cache.on_gpu(layout)).cpu()
    for e, n in enumerate(lens):
        k, v = cache.dense(e, max(n, 0))
        want, mag = attention(q[e], k, v, scale)
        assert_close(o[e], want, mag, n, v.abs().max().item() if n > 0 else 0.0)
        first = max(rows - max(n, 0), 0)
        assert not o[e, :first].any()  # queries before the first position
    assert ext.device_status() == 0


# Many more entries than a block has threads, one of them long; with and without unused ones at the ends.
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("batch,rows", [(129, 1), (300, 1), (257, 3)])
def test_many_entries(ext, fal, dtype, batch, rows):
    gen = torch.Generator().manual_seed(batch)
    hq, hkv, d, page = 4, 2, 64, 16
    lens = [int(x) for x in torch.randint(0, 50, (batch,), generator=gen)]
    lens[0], lens[batch // 2], lens[128], lens[-1] = -1, 3000, 77, 0
    cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d)
    q = _rows(gen, batch, rows, hq, d)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens), **cache.on_gpu("bshd")).cpu()
    for e, n in enumerate(lens):
        k, v = cache.dense(e, max(n, 0))
        want, mag = attention(q[e], k, v, 1 / math.sqrt(d))
        assert_close(o[e], want, mag, n, v.abs().max().item() if n > 0 else 0.0)
    assert ext.device_status() == 0


# Long entries, cut into many parts whose borders fall anywhere; every number of query rows that has a kernel of its own, full and
# partial; lengths that end in the pages and in the tail.
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d,rows", [(8, 1, 128, 1), (8, 1, 64, 2), (7, 1, 128, 3), (4, 1, 128, 8), (4, 1, 64, 24), (2, 1, 256, 8),
                                           (5, 1, 256, 5), (3, 1, 96, 10), (2, 2, 32, 24)])
def test_long_entries_and_every_number_of_rows(ext, fal, dtype, hq, hkv, d, rows):
    gen = torch.Generator().manual_seed(d + rows)
    lens = [9000, 4097, 2500]
    cache = _filled(gen, DTYPES[dtype], lens, 64, hkv, d)
    q = _rows(gen, 3, rows, hq, d)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens), softmax_scale=0.3,
                                          **cache.on_gpu("bshd")).cpu()
    for e, n in enumerate(lens):
        k, v = cache.dense(e, n)
        want, mag = attention(q[e], k, v, 0.3)
        assert_close(o[e], want, mag, n, v.abs().max().item())
    assert ext.device_status() == 0


def test_scores_of_every_size_and_order(fal):
    """The largest score last, first, or the same throughout; scores far above and below what exponentials of 32 bits hold."""
    hq, hkv, d, page, n = 2, 1, 64, 16, 400
    for dtype in (torch.float16, torch.int8):
        for slope in (-0.5, 0.0, 0.5, 4.0):
            for offset in (0.0, -60.0, 60.0):
                gen = torch.Generator().manual_seed(1)
                cache = Cache(gen, dtype, 30, page, hkv, d, 1, 26)
                cache.reserve(0, n)
                k = torch.zeros(n, hkv, d)
                k[:, 0, 0] = (torch.arange(n) - n / 2) * slope / 16 + offset  # (times q's 8: steps of slope / 2)
                cache.append(0, k.half(), _rows(gen, n, hkv, d))
                q = torch.zeros(1, 1, hq, d).half()
                q[..., 0] = 8
                o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens([n]), softmax_scale=1.0,
                                                      **cache.on_gpu("bshd")).cpu()
                kd, vd = cache.dense(0, n)
                want, mag = attention(q[0], kd, vd, 1.0)
                assert_close(o[0], want, mag, n, vd.abs().max().item())


# Block tables so long that the pages of a part of the entries, or of the KV heads of one entry, are put in order at a time.
@pytest.mark.parametrize("dtype", ["fp16", "int8"])
@pytest.mark.parametrize("batch,hq,hkv,d,width", [(70, 4, 2, 64, 128), (2, 8, 8, 128, 2048)])
def test_many_tokens_behind_long_block_tables(ext, fal, dtype, batch, hq, hkv, d, width):
    gen = torch.Generator().manual_seed(width)
    lens = [int(x) for x in torch.randint(0, 300, (batch,), generator=gen)]
    lens[-1] = 513
    cache = _filled(gen, DTYPES[dtype], lens, 256, hkv, d)
    table = torch.full((batch, width), -1, dtype=torch.int32)
    table[:, :cache.table.shape[1]] = cache.table
    q = _rows(gen, batch, 33, hq, d)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=table.cuda(), cache_seqlens=_lens(lens), **cache.on_gpu("bshd")).cpu()
    for e, n in enumerate(lens):
        k, v = cache.dense(e, n)
        want, mag = attention(q[e], k, v, 1 / math.sqrt(d))
        assert_close(o[e], want, mag, n, v.abs().max().item() if n > 0 else 0.0)
    assert ext.device_status() == 0


# Pages whose values differ by many powers of two, pages of zeros, of the smallest fp16 numbers and of the largest; each query sees
# another part of them, and is off by no more than the largest value that it sees allows.
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 7, 24, 32, 33, 130, 400])
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 128, 16), (2, 2, 64, 32), (2, 1, 256, 16), (3, 1, 96, 64)])
def test_pages_of_every_size_of_values(ext, fal, dtype, rows, hq, hkv, d, page):
    gen = torch.Generator().manual_seed(rows + d)
    n = 411
    cache = Cache(gen, DTYPES[dtype], n // page + 3, page, hkv, d, 1, n // page + 1)
    cache.reserve(0, n)
    pages = n // page + 1

    def sizes(powers):
        x = torch.tensor(powers)[torch.randint(0, len(powers), (pages, hkv), generator=gen)]
        return x.repeat_interleave(page, 0)[:n, :, None]
    k = (_rows(gen, n, hkv, d).float() * sizes([0.0, 2.0 ** -24, 2.0 ** -10, 1.0, 4.0])).half()
    v = (_rows(gen, n, hkv, d).float() * sizes([0.0, 2.0 ** -22, 2.0 ** -14, 2.0 ** -7, 1.0, 2.0 ** 7, 2.0 ** 12])).half()
    cache.append(0, k, v)
    q = _rows(gen, 1, rows, hq, d)
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens([n]),
                                          **cache.on_gpu("bshd")).cpu()
    kd, vd = cache.dense(0, n)
    want, mag = attention(q[0], kd, vd, 1 / math.sqrt(d))
    seen = vd.abs().amax(dim=2).cummax(dim=0).values[n - rows:].repeat_interleave(hq // hkv, dim=1)[:, :, None]
    assert_close(o[0], want, mag, n, seen)
    assert ext.device_status() == 0


def test_values_behind_the_length_do_not_matter(fal):
    """NaN and infinities in the rest of the last page, of other pages and of the tail, for every path."""
    gen = torch.Generator().manual_seed(14)
    for dtype in DTYPES:
        for rows in (1, 5, 32, 40):
            cache = _filled(gen, DTYPES[dtype], [41, 100], 32, 2, 64)
            got = cache.on_gpu("bshd")
            args = dict(block_table=cache.table.cuda(), cache_seqlens=_lens([41, 100]))
            q = _rows(gen, 2, rows, 4, 64).cuda()
            o = fal.flash_attn_with_paged_kvcache(q, **args, **got)
            for n, t in got.items():
                if dtype == "fp16" or n.endswith("tail"):
                    t.masked_fill_(t.isnan(), math.inf)  # (the model leaves NaN there)
            assert torch.equal(fal.flash_attn_with_paged_kvcache(q, **args, **got), o) and not o.isnan().any()


def test_a_run_of_steps_as_a_server_makes_them(ext, fal):
    """A prompt, chunks and tokens, appended and attended to in one call each, against the whole text in 64 bits."""
    for dtype in DTYPES:
        gen = torch.Generator().manual_seed(11)
        hq, hkv, d, page, total = 8, 2, 64, 32, 230
        q, k, v = (_rows(gen, 2, total, h, d) for h in (hq, hkv, hkv))
        cos, sin = _tables(256, d)
        cache = _filled(gen, DTYPES[dtype], [0, 0], page, hkv, d, extra=256)
        cache.table = cache.table[:, :8].contiguous()
        got, lens = cache.on_gpu("bshd"), _lens([0, 0])
        table, at = cache.table.cuda(), 0
        for n in [150, 40, 1, 1, 5, 30, 1, 1, 1]:
            args = [x[:, at:at + n].cuda() for x in (q, k, v)]
            o = fal.flash_attn_with_paged_kvcache(args[0], block_table=table, cache_seqlens=lens, k=args[1], v=args[2],
                                                  rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), **got).cpu()
            for e in range(2):
                cache.append(e, rotate(k[e, at:at + n], at, cos, sin, False), v[e, at:at + n])
                kd, vd = cache.dense(e, at + n)
                want, mag = attention(rotate(q[e, at:at + n], at, cos, sin, False), kd, vd, 1 / math.sqrt(d))
                assert_close(o[e], want, mag, at + n, vd.abs().max().item())
            at += n
            lens = lens + n
        cache.check(got, "bshd")
        assert ext.device_status() == 0


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_captured_steps_replayed_side_by_side(fal, dtype):
    """Two graphs of one stream, replayed on two streams at once, lengths moved on inside: each as the same steps made eagerly."""
    gen = torch.Generator().manual_seed(2)
    hq, hkv, d, page, steps = 8, 2, 128, 16, 20
    cos, sin = (t.cuda() for t in _tables(64 * page, d))
    sides, graphs = [], []
    for i in range(2):
        lens = [500 + i, 9, 30]
        cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d, extra=steps + 1)
        s = {"got": cache.on_gpu("bshd"), "table": cache.table.cuda(), "lens": _lens(lens),
             "in": [_rows(gen, 3, 1, h, d).cuda() for h in (hq, hkv, hkv)]}
        s["eager"] = {"got": {n: t.clone() for n, t in s["got"].items()}, "lens": s["lens"].clone()}
        sides.append(s)

    def step(s, got, lens):
        q, k, v = s["in"]
        o = fal.flash_attn_with_paged_kvcache(q, block_table=s["table"], cache_seqlens=lens, k=k, v=v, rotary_cos=cos,
                                              rotary_sin=sin, **got)
        lens += 1
        return o

    want = []
    for s in sides:
        for _ in range(steps):
            o = step(s, s["eager"]["got"], s["eager"]["lens"])
        want.append(o)
    capture = torch.cuda.Stream()
    for s in sides:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=capture):
            s["out"] = step(s, s["got"], s["lens"])
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(steps):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, o in zip(sides, want):
        assert torch.equal(s["out"], o) and torch.equal(s["lens"], s["eager"]["lens"])
        for n, t in s["got"].items():
            assert torch.equal(t.view(torch.uint8), s["eager"]["got"][n].view(torch.uint8)), n


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_views_and_another_stream(fal, dtype):
    """q, k, v as slices of one projection, a table that is part of a larger one, pages of one allocation, off the default stream."""
    gen = torch.Generator().manual_seed(3)
    hq, hkv, d, page, rows, lens = 4, 2, 64, 16, 6, [20, 45]
    cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d, extra=rows)
    plain = cache.on_gpu("bshd")
    views = {n: t.clone() for n, t in plain.items()}  # (the append moves scales and tails on)
    both = torch.stack([plain["k_pages"].view(torch.uint8), plain["v_pages"].view(torch.uint8)], dim=1).contiguous()
    views["k_pages"], views["v_pages"] = both[:, 0].view(DTYPES[dtype]), both[:, 1].view(DTYPES[dtype])
    x = _rows(gen, 2, rows, hq + 2 * hkv, d).cuda()
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]
    wide = torch.full((4, cache.table.shape[1] + 5), -7, dtype=torch.int32).cuda()
    wide[1:3, 2:-3] = cache.table.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        o = fal.flash_attn_with_paged_kvcache(q, block_table=wide[1:3, 2:-3], cache_seqlens=_lens(lens), k=k, v=v, **views)
    stream.synchronize()
    want = fal.flash_attn_with_paged_kvcache(q.contiguous(), block_table=cache.table.cuda(), cache_seqlens=_lens(lens).long(),
                                             k=k.contiguous(), v=v.contiguous(), **plain)
    assert torch.equal(o, want)
    for n in plain:
        assert torch.equal(views[n].contiguous().view(torch.uint8), plain[n].view(torch.uint8))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_without_a_place_are_dropped_and_reported(ext, fal, dtype):
    """Entry 0 runs into the end of its table, entry 1 into a table entry that names no page, entry 2 into a page number that is too large."""
    gen = torch.Generator().manual_seed(5)
    hkv, d, page, rows = 2, 64, 16, 20
    cache = _filled(gen, DTYPES[dtype], [40, 10, 10, 3], page, hkv, d, extra=rows)
    cache.table = cache.table[:, :3].contiguous()  # 48 positions
    cache.table[1, 1], cache.table[2, 1] = -1, 10 ** 6
    got = cache.on_gpu("bshd")
    k, v, q = (_rows(gen, 4, rows, hkv, d) for _ in range(3))
    out, lens = fal.paged_cache_append(k.cuda(), v.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens([40, 10, 10, 3]), q=q.cuda(), **got)
    assert ext.device_status() == 2000
    assert lens.tolist() == [48, 30, 30, 23]
    assert not out[0, 8:].any() and torch.equal(out[0, :8].cpu(), q[0, :8]) and torch.equal(out[1:].cpu(), q[1:])
    cache.append(0, k[0, :8], v[0, :8])
    cache.table[2, 1] = -1
    for e in (1, 2, 3):
        cache.append(e, k[e], v[e])
    cache.check(got, "bshd")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [1, 40])
def test_a_position_without_a_page_counts_as_zeros(ext, fal, dtype, rows):
    gen = torch.Generator().manual_seed(6)
    hq, hkv, d, page, lens = 4, 2, 64, 16, [100, 70]
    cache = _filled(gen, DTYPES[dtype], lens, page, hkv, d)
    q = _rows(gen, 2, rows, hq, d)
    table = cache.table.clone()
    table[0, 2], table[1, 0] = -1, 4096
    args = dict(cache_seqlens=_lens(lens), **cache.on_gpu("bshd"))
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=table.cuda(), **args).cpu()
    assert ext.device_status() == 3000
    for e, (n, gone) in enumerate(zip(lens, (2, 0))):
        k, v = cache.dense(e, n)
        k[gone * page:(gone + 1) * page] = 0
        v[gone * page:(gone + 1) * page] = 0
        want, mag = attention(q[e], k, v, 1 / math.sqrt(d))
        assert_close(o[e], want, mag, n, v.abs().max().item())


def test_a_page_with_a_nan_shows_in_what_sees_it_only(fal):
    gen = torch.Generator().manual_seed(7)
    cache = _filled(gen, torch.int8, [64, 64], 16, 2, 64)
    got = cache.on_gpu("bshd")
    got["v_scales"][cache.table[1, 2].item(), 1] = math.nan
    o = fal.flash_attn_with_paged_kvcache(_rows(gen, 2, 1, 4, 64).cuda(), block_table=cache.table.cuda(),
                                          cache_seqlens=_lens([64, 64]), **got)
    assert o.isnan().any(dim=-1)[:, 0].tolist() == [[False] * 4, [False, False, True, True]]


def test_positions_beyond_32_bits_of_elements(fal):
    """Pages whose elements lie more than 2^31 from the pool's start."""
    gen = torch.Generator().manual_seed(8)
    hkv, d, page = 8, 128, 256
    pages = 2 ** 31 // (page * hkv * d) + 4
    for dtype in (torch.float16, torch.int8):
        small = _filled(gen, dtype, [600], page, hkv, d, extra=8, spare=0)
        got = small.on_gpu("bshd")
        large = {n: t.clone() for n, t in got.items()}
        for n in ("k_pages", "v_pages"):
            large[n] = torch.zeros((pages, page, hkv, d), dtype=dtype, device="cuda")
            large[n][-3:] = got[n]
            if dtype == torch.int8:
                scales = torch.zeros((pages, hkv), device="cuda")
                scales[-3:] = got[n[0] + "_scales"]
                large[n[0] + "_scales"] = scales
        q, k, v = (_rows(gen, 1, 3, h, d).cuda() for h in (16, hkv, hkv))
        for rows in (3, 1):
            args = dict(cache_seqlens=_lens([600]), k=k[:, :rows], v=v[:, :rows])
            a = fal.flash_attn_with_paged_kvcache(q[:, :rows], block_table=small.table.cuda(), **args, **got)
            far = torch.where(small.table >= 0, small.table + pages - 3, small.table).cuda()
            b = fal.flash_attn_with_paged_kvcache(q[:, :rows], block_table=far, **args, **large)
            assert torch.equal(a, b) and torch.equal(large["k_pages"][-3:].view(torch.uint8), got["k_pages"].view(torch.uint8))
        del large


def test_refusals(fal):
    gen = torch.Generator().manual_seed(10)
    good = _filled(gen, torch.int8, [20, 30], 16, 2, 64, extra=4)
    got = good.on_gpu("bshd")
    q, k, v = (_rows(gen, 2, 1, h, 64).cuda() for h in (4, 2, 2))
    base = dict(block_table=good.table.cuda(), cache_seqlens=_lens([20, 30]), **got)
    cos, sin = (t.cuda() for t in _tables(good.table.shape[1] * 16, 64))

    def attend(**change):
        return fal.flash_attn_with_paged_kvcache(**{"q": q, **base, **change})

    attend()
    attend(k=k, v=v, rotary_cos=cos, rotary_sin=sin)
    wrong = [dict(k_tail=None), dict(k_scales=None), dict(k_scales=got["k_scales"].half()), dict(v_scales=got["v_scales"][:, :1]),
             dict(k_tail=got["k_tail"][:1]), dict(v_tail=got["v_tail"].float()), dict(k_pages=got["k_pages"].half()),
             dict(k_pages=got["k_pages"].view(torch.uint8), v_pages=got["v_pages"].view(torch.uint8)),
             dict(v_pages=got["v_pages"][:-1]), dict(k_pages=got["k_pages"][:, :8], v_pages=got["v_pages"][:, :8]),
             dict(block_table=base["block_table"][:1]), dict(block_table=base["block_table"].t()), dict(cache_seqlens=_lens([1, 2, 3])),
             dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(softmax_scale=-1.0), dict(block_table=base["block_table"].cpu()),
             dict(k=k, v=v[:, :, :1]), dict(k=k, v=v, rotary_cos=cos), dict(k=k, v=v, rotary_cos=cos[:20], rotary_sin=sin[:20]),
             dict(k=k, v=v, rotary_cos=cos[:, :12].contiguous(), rotary_sin=sin[:, :12].contiguous()),
             dict(k=k, v=v, rotary_cos=cos.double(), rotary_sin=sin.double()), dict(q=q.clone().requires_grad_()),
             dict(k=k.clone().requires_grad_(), v=v), dict(q=q[:, :0]), dict(k=got["k_tail"][:, :1], v=v)]
    for change in wrong:
        with pytest.raises(RuntimeError):
            attend(**change)
    for change in (dict(q=q.float()), dict(rotary_cos=cos, rotary_sin=sin), dict(k=k), dict(v=v), dict(k=k.float(), v=v.float())):
        with pytest.raises(AssertionError):
            attend(**change)
    with pytest.raises(ValueError):
        attend(cache_layout="bhnd")
    with torch.no_grad():
        attend(q=q.clone().requires_grad_())
    # a refused call has not appended anything
    before = {n: t.clone() for n, t in got.items()}
    for change in (dict(softmax_scale=0.0), dict(q=q[:, :, :3].contiguous())):
        with pytest.raises(RuntimeError):
            attend(k=k, v=v, **change)
    torch.cuda.synchronize()
    assert all(torch.equal(t.view(torch.uint8), before[n].view(torch.uint8)) for n, t in got.items())


def test_both_host_paths_give_the_same(ext, fal, monkeypatch):
    """The native function takes these calls, and Python makes them to the same bits where there is none."""
    gen = torch.Generator().manual_seed(12)
    if ext._host is None:
        pytest.skip("no native host path was built")
    ext.device_status()
    for dtype in DTYPES:
        ends = []
        for native in (True, False):
            gen = torch.Generator().manual_seed(12)
            cache = _filled(gen, DTYPES[dtype], [30, 7], 16, 2, 64, extra=9)
            got = cache.on_gpu("bhsd")
            q, k, v = (_rows(gen, 2, 9, h, 64).cuda() for h in (4, 2, 2))
            cos, sin = (t.cuda() for t in _tables(cache.table.shape[1] * 16, 32))
            calls = []
            for n in ("paged_append_plain", "paged_attend_plain"):
                real = getattr(ext._host, n[:-6])
                monkeypatch.setattr(ext, n, (lambda *a, real=real: calls.append(real(*a)) or calls[-1]) if native else ext._general)
            versions = {n: t._version for n, t in got.items()}
            o = fal.flash_attn_with_paged_kvcache(q[:, :4], block_table=cache.table.cuda(), cache_seqlens=_lens([30, 7]), k=k[:, :4], v=v[:, :4],
                                                  rotary_cos=cos, rotary_sin=sin, rotary_interleaved=True, softmax_scale=0.2, cache_layout="bhsd", **got)
            turned, lens = fal.paged_cache_append(k[:, 4:], v[:, 4:], block_table=cache.table.cuda(), cache_seqlens=_lens([34, 11]), q=q[:, 4:],
                                                  rotary_cos=cos, rotary_sin=sin, cache_layout="bhsd", **got)
            o2 = fal.flash_attn_with_paged_kvcache(turned, block_table=cache.table.cuda(), cache_seqlens=lens, cache_layout="bhsd", **got)
            assert len(calls) == (3 if native else 0) and all(c is not None for c in calls)
            assert all(t._version > versions[n] for n, t in got.items())
            ends.append([o, turned, lens, o2, *(t.view(torch.uint8) for t in got.values())])
        assert all(torch.equal(a, b) for a, b in zip(*ends))
