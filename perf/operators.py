"""The paged key/value cache calls whose speed matters to a server, as cases that a harness can time.

Three operators: the append of new rows to a paged cache with the position rotation applied on the way
(`paged_cache_append`), attention of new tokens over fp16 pages, and attention over pages held in 8 bits with a scale
for each page and head (`flash_attn_with_paged_kvcache`, both).  With `own` they are called as a user's program calls
them; without, the same results are computed by elementary tensor operations in 32 bits.

Cache layout: pages [num_pages, page, Hkv, d] ("bshd") or [num_pages, Hkv, page, d] ("bhsd"); block_table int32
[B, pages per entry]; position p of entry b is row p % page of page block_table[b, p // page].  8-bit pages hold codes
and have fp32 scales [num_pages, Hkv]; the rows of an entry's last, unfinished page are fp16 rows of its tail
[B, page, Hkv, d] (or [B, Hkv, page, d]) until the page is full.

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU, made from the seed
    run(state)           one pass, and everything it computes
    work(case)           bytes and floating-point operations a pass cannot do without
    exact(case, seed)    the results in 64 bits
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "flash-attention-legacy_b200"))

own = False
DEVICE = "cuda"
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
TORCH = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _case(name, kind, dtype, batch, heads, kv_heads, head_dim, page, new, min_len, max_len, **more):
    """kind: attend (the cache holds the new rows), append, step (append, then attend).  min_len, max_len: positions in the
    cache before the new ones.  rotary: rotated columns of a head."""
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "new": new, "min_len": min_len, "max_len": max_len, "len_seed": 1,
            "layout": "bshd", "rotary": head_dim if kind != "attend" else 0, "interleaved": False, **more}


def listed():
    return [
        # One chat session being answered from fp16 pages: launches and host work are what a step costs.
        _case("decode_fp16_single", "attend", "fp16", 1, 32, 8, 128, 16, 1, 1998, 1998),
        # A serving step: 64 sequences of 1 024 to 32 512 cached tokens, one new token each.
        _case("decode_fp16_serving", "attend", "fp16", 64, 32, 8, 128, 16, 1, 1024, 32511),
        # A small batch of half-width heads with the cache in 8 bits, head-major pages.
        _case("decode_int8_b8", "attend", "int8", 8, 32, 4, 64, 64, 1, 2048, 2048, layout="bhsd"),
        # The serving step with the cache in 8 bits.
        _case("decode_int8_serving", "attend", "int8", 64, 32, 8, 128, 32, 1, 1024, 32511),
        # Every query head with a KV head of its own, the widest heads, ragged lengths.
        _case("decode_e4m3_wide", "attend", "e4m3", 16, 16, 16, 256, 128, 1, 100, 9000),
        # Five drafted tokens checked at once behind eight texts.
        _case("verify_int8", "attend", "int8", 8, 32, 8, 128, 64, 5, 500, 12000),
        # A prompt chunk behind caches filled to different lengths (chunked prefill of a serving loop).
        _case("chunk_int8", "attend", "int8", 4, 32, 8, 128, 64, 1024, 512, 7000),
        # The token of one chat session goes to its page, q and k rotated.
        _case("append_token_fp16", "append", "fp16", 1, 32, 8, 128, 16, 1, 1999, 1999),
        # The tokens of a serving step go to 8-bit pages; some of them fill a page.
        _case("append_token_int8", "append", "int8", 64, 32, 8, 128, 16, 1, 1024, 32000),
        # Prompts of no particular length, pairs of neighbouring columns rotated, half of a head's columns.
        _case("append_prompt_fp16", "append", "fp16", 4, 40, 8, 128, 16, 2987, 0, 900, rotary=64, interleaved=True),
        # A prompt chunk is rotated and rounded to 8 bits.
        _case("append_prompt_int8", "append", "int8", 4, 32, 8, 128, 64, 1024, 100, 6000),
        # What a server does for every token: rotate, append, attend, in one call.
        _case("step_fp16_b16", "step", "fp16", 16, 32, 8, 128, 32, 1, 500, 6000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "attend", "append", "append", "step"])
        dtype = rng.choice(["fp16", "int8", "int8", "e4m3"]) if kind != "step" else "fp16"
        heads, kv_heads = rng.choice([(8, 8), (16, 16), (32, 8), (32, 8), (32, 4), (16, 2), (40, 8), (8, 1), (16, 1), (24, 8)])
        head_dim = rng.choice([64, 64, 128, 128, 128, 32, 96, 256])
        page = rng.choice([16, 16, 32, 64, 128, 256])
        if kind == "append":
            new = rng.choice([1, _log_int(rng, 2, 4096)])
        else:
            new = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 2048)])
        longest = _log_int(rng, 64, 33000)
        c = _case("", kind, dtype, _log_int(rng, 1, 96), heads, kv_heads, head_dim, page, new,
                  rng.randint(0, longest), longest, len_seed=rng.randint(0, 9999), layout=rng.choice(["bshd", "bhsd"]),
                  interleaved=rng.random() < 0.4)
        del c["name"]
        if kind != "attend":
            c["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2])
        rows = c["batch"] * (longest + new) * kv_heads * head_dim
        cost = work(c)
        if (c["batch"] * new * heads * head_dim <= 1 << 26
                and (kind == "append" or rows <= (64 * 32768 * 8 * 128 if kind == "attend" and new == 1 else 1 << 28))
                and all(cost[x] <= max(work(y)[x] for y in listed()) for x in cost)):
            return c


def _lengths(c):
    """Positions of every entry before the new ones: from the case alone, the longest among them."""
    r = random.Random(c["len_seed"])
    return [c["max_len"]] + [r.randint(c["min_len"], c["max_len"]) for _ in range(c["batch"] - 1)]


def work(c):
    lens, new, d, hq, hkv, page = _lengths(c), c["new"], c["head_dim"], c["heads"], c["kv_heads"], c["page"]
    size = 2 if c["dtype"] == "fp16" else 1
    queries, rows = 2 * c["batch"] * new * hq * d, 2 * c["batch"] * new * hkv * d
    total, flops = 0.0, 0.0
    if c["kind"] != "attend":
        total += 2 * queries + 2 * rows + 8 * sum(new * (c["rotary"] // 2) for _ in lens)
        for n in lens:
            sealed = ((n + new) // page - n // page) if size == 1 else 0
            waiting = ((n + new) % page if sealed else new) if size == 1 else new
            total += 2 * hkv * d * (sealed * page + 2 * waiting) + (8 * sealed * hkv)
            if sealed:
                total += 2 * hkv * d * 2 * (n % page)
        flops += 6.0 * c["batch"] * new * (hq + hkv) * (c["rotary"] // 2)
    if c["kind"] != "append":
        for n in lens:
            n += new
            inside = n // page * page if size == 1 else n
            total += 2 * hkv * d * (inside * size + (n - inside) * 2) + (8 * (inside // page) * hkv if size == 1 else 0)
            flops += 4.0 * hq * d * (new * (n - new) + new * (new + 1) / 2)
        total += 2 * queries
    return {"bytes": total, "flops": flops}


def _quantised(x, dtype):
    """Codes and scales of fp16 rows [pages, page, H, d], each page and head by its own largest magnitude."""
    x = x.float()
    most = x.abs().amax(dim=(1, 3))
    scale = most / torch.full_like(most, CODE_MAX[dtype])
    scale = torch.where(torch.isfinite(most), scale, torch.full_like(scale, math.nan))
    ok = (torch.isfinite(most) & (most > 0))[:, None, :, None]
    y = x * CODE_MAX[dtype] / torch.where(most > 0, most, torch.ones_like(most))[:, None, :, None]
    y = torch.where(ok, y, torch.zeros_like(y))
    return (y.round() if dtype == "int8" else y).to(TORCH[dtype]), scale


def _to_layout(t, layout):
    return t if layout == "bshd" else t.transpose(1, 2).contiguous()


def _rows_first(t, layout):
    return t if layout == "bshd" else t.transpose(1, 2)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    b, new, hq, hkv, d, page = c["batch"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens = _lengths(c)

    def rows(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float16)

    width = (max(lens) + new) // page + 2
    first = [0] * b if c["kind"] != "append" else [n // page for n in lens]
    need = [(n + new + page - 1) // page - f for n, f in zip(lens, first)]
    pages = sum(need) + 1
    order = (torch.randperm(pages - 1, generator=g, device=DEVICE) + 1).to(torch.int32)
    # Pages that nobody needs any more (an append does not look at them) are page 0; behind an entry's length: no page.
    table = torch.full((b, width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for e in range(b):
        table[e, :first[e]] = 0
        table[e, first[e]:first[e] + need[e]] = order[at:at + need[e]]
        at += need[e]
    s = {"case": c, "block_table": table}
    kept = [n + new if c["kind"] == "attend" else n for n in lens]
    s["cache_seqlens"] = torch.tensor(kept, dtype=torch.int32, device=DEVICE)
    for name in ("k", "v"):
        shape = (pages, page, hkv, d) if c["layout"] == "bshd" else (pages, hkv, page, d)
        store = torch.empty(shape, dtype=TORCH[c["dtype"]], device=DEVICE)
        scales = torch.empty((pages, hkv), dtype=torch.float32, device=DEVICE)
        step = max(1, (1 << 26) // (page * hkv * d))
        for i in range(0, pages, step):
            x = rows(min(step, pages - i), page, hkv, d)
            if c["dtype"] == "fp16":
                store[i:i + step] = _to_layout(x, c["layout"])
            else:
                codes, scales[i:i + step] = _quantised(x, c["dtype"])
                store[i:i + step] = _to_layout(codes, c["layout"])
        s[name + "_pages"] = store
        if c["dtype"] != "fp16":
            s[name + "_scales"] = scales
            s[name + "_tail"] = _to_layout(rows(b, page, hkv, d), c["layout"])
    s["q"] = rows(b, new, hq, d)
    if c["kind"] != "attend":
        s["k"], s["v"] = rows(b, new, hkv, d), rows(b, new, hkv, d)
        half = c["rotary"] // 2
        speed = 10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
        angle = torch.arange(width * page, device=DEVICE, dtype=torch.float64)[:, None] * speed[None, :]
        s["rotary_cos"], s["rotary_sin"] = angle.cos().float(), angle.sin().float()
    return s


def _rotated(x, positions, s):
    """x [B, L, H, d] rotated by its rows' positions [B, L], in 32 bits, rounded once to fp16."""
    c = s["case"]
    half = c["rotary"] // 2
    cos, sin = (s[n][positions][:, :, None, :] for n in ("rotary_cos", "rotary_sin"))
    x = x.float()
    if c["interleaved"]:
        x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).flatten(-2)
    else:
        x1, x2 = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1).half()


def _append(s):
    c, table, lens = s["case"], s["block_table"].long(), s["cache_seqlens"].long()
    b, new, page = c["batch"], c["new"], c["page"]
    entry = torch.arange(b, device=DEVICE)[:, None]
    positions = lens[:, None] + torch.arange(new, device=DEVICE)[None, :]
    q, k = _rotated(s["q"], positions, s), _rotated(s["k"], positions, s)
    for name, x in (("k", k), ("v", s["v"])):
        store = _rows_first(s[name + "_pages"], c["layout"])
        if c["dtype"] == "fp16":
            store[table[entry, positions // page], positions % page] = x
            continue
        # a window of pages from the one that the first new row belongs to
        tail = _rows_first(s[name + "_tail"], c["layout"])
        windows = (page - 1 + new) // page + 1
        window = torch.zeros((b, windows * page, *x.shape[2:]), dtype=torch.float16, device=DEVICE)
        window[:, :page] = tail
        window[entry, (lens % page)[:, None] + torch.arange(new, device=DEVICE)] = x
        end = lens % page + new
        codes, scales = _quantised(window.view(b * windows, page, *x.shape[2:]), c["dtype"])
        index = torch.arange(windows, device=DEVICE)[None, :]
        full = index < (end // page)[:, None]
        ids = table[entry, torch.minimum(lens[:, None] // page + index, torch.full_like(entry, table.shape[1] - 1))]
        ids = torch.where(full, ids, torch.zeros_like(ids)).flatten()  # page 0 takes what belongs to no page, and gets its own back
        full = full.flatten()
        bits = store.view(torch.uint8)
        bits[ids] = torch.where(full[:, None, None, None], codes.view(torch.uint8), bits[0])
        s[name + "_scales"][ids] = torch.where(full[:, None], scales, s[name + "_scales"][0])
        row = torch.arange(page, device=DEVICE)
        waits = row[None, :] < (end % page)[:, None]
        last = window[entry, (end // page * page)[:, None] + row]
        tail.copy_(torch.where(waits[:, :, None, None], last, tail))
    return q, (lens + new).int()


def _values(s):
    """What the cache holds, as fp16 rows: fp16 pages as they are, 8-bit ones as codes times scales, and the rows that wait."""
    c, got = s["case"], {}
    for name in ("k", "v"):
        pages = s[name + "_pages"]
        if c["dtype"] != "fp16":
            scale = s[name + "_scales"]
            scale = scale[:, None, :, None] if c["layout"] == "bshd" else scale[:, :, None, None]
            pages = torch.mul(pages if c["dtype"] == "int8" else pages.float(), scale,
                              out=torch.empty(pages.shape, dtype=torch.float16, device=DEVICE))
            got[name + "_tail"] = s[name + "_tail"]
        got[name + "_pages"] = pages
    return got


def _dense(s, name, lens, most):
    """[B, most, Hkv, d] rows of every entry in 32 bits, whatever lies behind its length."""
    c = s["case"]
    page = c["page"]
    ids = s["block_table"][:, :(most + page - 1) // page].long().clamp(min=0)
    bits = torch.float16 if c["dtype"] == "fp16" else torch.int8
    x = _rows_first(s[name + "_pages"], c["layout"]).view(bits)[ids].view(TORCH[c["dtype"]]).float()
    if c["dtype"] != "fp16":
        x = x * s[name + "_scales"][ids][:, :, None, :, None]
        tail = _rows_first(s[name + "_tail"], c["layout"]).float()
        waits = torch.arange(ids.shape[1], device=DEVICE)[None, :] == (lens // page)[:, None]
        x = torch.where(waits[:, :, None, None, None], tail[:, None], x)
    return x.flatten(1, 2)[:, :most]


def _attend(s, q, lens):
    c = s["case"]
    b, new, hq, hkv, d = c["batch"], c["new"], c["heads"], c["kv_heads"], c["head_dim"]
    lens = lens.long()
    most = c["max_len"] + new
    k = _dense(s, "k", lens, most)
    x = q.float().view(b, new, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    scores = (x @ k.permute(0, 2, 3, 1)).view(b, hkv, hq // hkv, new, most) / math.sqrt(d)
    del k
    place = torch.arange(most, device=DEVICE)
    limit = lens[:, None] - new + torch.arange(new, device=DEVICE)[None, :]
    scores.masked_fill_((place[None, None, :] > limit[:, :, None])[:, None, None], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(dim=-1, keepdim=True)
    v = _dense(s, "v", lens, most)
    o = p.view(b, hkv, -1, most) @ v.permute(0, 2, 1, 3)
    return o.view(b, hkv, hq // hkv, new, d).permute(0, 3, 1, 2, 4).reshape(b, new, hq, d).half()


def _cache(s):
    return {n: s[n] for n in ("k_scales", "v_scales", "k_tail", "v_tail") if n in s}


def run(s):
    c = s["case"]
    if own:
        from flash_attn_legacy import flash_attn_with_paged_kvcache, paged_cache_append
        pages = (s["k_pages"], s["v_pages"], s["block_table"], s["cache_seqlens"])
        if c["kind"] == "attend":
            return flash_attn_with_paged_kvcache(s["q"], *pages, cache_layout=c["layout"], **_cache(s))
        turn = {"rotary_cos": s["rotary_cos"], "rotary_sin": s["rotary_sin"], "rotary_interleaved": c["interleaved"],
                "cache_layout": c["layout"]}
        if c["kind"] == "append":
            q, lens = paged_cache_append(s["k"], s["v"], *pages, q=s["q"], **turn, **_cache(s))
            return {"q": q, "lens": lens, **_values(s)}
        out = flash_attn_with_paged_kvcache(s["q"], *pages, k=s["k"], v=s["v"], **turn, **_cache(s))
        return {"out": out, **_values(s)}
    if c["kind"] == "attend":
        return _attend(s, s["q"], s["cache_seqlens"])
    q, lens = _append(s)
    if c["kind"] == "append":
        return {"q": q, "lens": lens, **_values(s)}
    return {"out": _attend(s, q, lens), **_values(s)}


# ---- the same from the definition, in 64 bits, entry by entry and page by page ----
def _exact_turn(x, start, s):
    """x [L, H, d] in 64 bits; the angles are those of the tables the operator is given."""
    c = s["case"]
    half, n = c["rotary"] // 2, x.shape[0]
    cos = s["rotary_cos"][start:start + n].double().unsqueeze(1)
    sin = s["rotary_sin"][start:start + n].double().unsqueeze(1)
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    y = x.double().clone()
    a, z = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * cos - z * sin
    y[..., second] = a * sin + z * cos
    return y


def _exact_codes(x, dtype):
    """The values that rows x [page, H, d] stand for in 8 bits."""
    most = x.abs().amax(dim=0).amax(dim=-1)[None, :, None]
    y = torch.where(most > 0, x * CODE_MAX[dtype] / most, torch.zeros_like(x))
    if dtype == "int8":
        y = y.round()
    else:  # three bits behind the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = (y / step).round() * step
    return y * most / CODE_MAX[dtype]


def _exact_pages(s):
    """The cache's values in 64 bits; pages first, then rows."""
    c, got = s["case"], {}
    for name in ("k", "v"):
        x = s[name + "_pages"]
        if c["layout"] == "bhsd":
            x = x.transpose(1, 2)
        x = x.to(torch.float32).double()
        if c["dtype"] != "fp16":
            x = x * s[name + "_scales"].double()[:, None, :, None]
            tail = s[name + "_tail"]
            got[name + "_tail"] = (tail.transpose(1, 2) if c["layout"] == "bhsd" else tail).double().clone()
        got[name + "_pages"] = x
    return got


def _exact_append(s, cache):
    c, page = s["case"], s["case"]["page"]
    queries = []
    for e, n in enumerate(s["cache_seqlens"].tolist()):
        queries.append(_exact_turn(s["q"][e], n, s))
        # (a cache row is an fp16 number by definition)
        for name, x in (("k", _exact_turn(s["k"][e], n, s).half().double()), ("v", s["v"][e].double())):
            if c["dtype"] == "fp16":
                for i in range(0, c["new"]):
                    if i == 0 or (n + i) % page == 0:
                        count = min(page - (n + i) % page, c["new"] - i)
                        at = (n + i) % page
                        cache[name + "_pages"][int(s["block_table"][e, (n + i) // page]), at:at + count] = x[i:i + count]
                continue
            tail = cache[name + "_tail"]
            x = torch.cat([tail[e, :n % page], x])
            start = n // page
            while x.shape[0] >= page:
                cache[name + "_pages"][int(s["block_table"][e, start])] = _exact_codes(x[:page], c["dtype"])
                x, start = x[page:], start + 1
            tail[e, :x.shape[0]] = x
    return torch.stack(queries)


def _exact_attend(s, cache, q, lens):
    c, page = s["case"], s["case"]["page"]
    group, out = c["heads"] // c["kv_heads"], []
    for e, n in enumerate(lens):
        ids = s["block_table"][e, :(n + page - 1) // page].long()
        rows = []
        for name in ("k", "v"):
            x = cache[name + "_pages"][ids] if isinstance(cache, dict) else cache(name, ids)
            x = x.reshape(-1, *x.shape[2:])[:n]
            if c["dtype"] != "fp16" and n % page:
                tail = s[name + "_tail"] if not isinstance(cache, dict) else None
                if tail is None:
                    tail = cache[name + "_tail"][e]
                else:
                    tail = (tail[e].transpose(0, 1) if c["layout"] == "bhsd" else tail[e]).double()
                x = torch.cat([x[:n - n % page], tail[:n % page]])
            rows.append(x.transpose(0, 1))
        k, v = rows
        heads = []
        for h in range(c["kv_heads"]):
            x = q[e][:, h * group:(h + 1) * group].double().transpose(0, 1) / math.sqrt(c["head_dim"])
            w = x @ k[h].T
            hidden = torch.arange(n, device=DEVICE)[None, :] - (n - c["new"]) > torch.arange(c["new"], device=DEVICE)[:, None]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
            heads.append((w @ v[h]).transpose(0, 1))
        out.append(torch.cat(heads, dim=1))
    return torch.stack(out)


def exact(c, seed):
    s = prepare(c, seed)
    new, lens = c["new"], s["cache_seqlens"].tolist()

    def layout(cache):
        return {n: _to_layout(x, c["layout"]) for n, x in cache.items()}

    def fetch(name, ids):  # only the pages of one entry in 64 bits: a large cache would not fit
        x = s[name + "_pages"]
        x = x.view(torch.int8 if c["dtype"] == "e4m3" else x.dtype)[ids].view(x.dtype).to(torch.float32).double()
        x = x.transpose(1, 2) if c["layout"] == "bhsd" else x
        return x if c["dtype"] == "fp16" else x * s[name + "_scales"][ids].double()[:, None, :, None]

    if c["kind"] == "attend":
        return _exact_attend(s, fetch, s["q"], lens)
    cache = _exact_pages(s)
    q = _exact_append(s, cache)
    if c["kind"] == "append":
        return {"q": q, "lens": None, **layout(cache)}
    # (queries are fp16 numbers between the two operators)
    return {"out": _exact_attend(s, cache, q.half(), [n + new for n in lens]), **layout(cache)}
