"""Plain models of a paged cache and of attention over it, on the CPU, for the tests of the paged operators."""
import math

import torch

CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rotate(x, start, cos, sin, interleaved):
    """x [L,H,d] fp16 at positions start ...: 32-bit products and sums, rounded once."""
    half = cos.shape[1]
    c, s = (t[start:start + x.shape[0], None].float() for t in (cos, sin))
    y = x.float().clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y.half()


def quantise(rows, dtype):
    """rows [page,H,d] fp16 -> (codes, scales [H] fp32), the quotients in 64 bits."""
    most = rows.float().abs().amax(dim=(0, 2))
    scale = most / torch.full_like(most, CODE_MAX[dtype])
    ok = torch.isfinite(most) & (most > 0)
    y = rows.double() * CODE_MAX[dtype] / torch.where(ok, most, torch.ones_like(most)).double()[None, :, None]
    y = torch.where(ok[None, :, None], y, torch.zeros_like(y))
    if dtype == torch.int8:
        codes = y.round().to(torch.int8)
    else:  # four significant bits, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        codes = ((y / step).round() * step).float().to(dtype)
    return codes, torch.where(torch.isfinite(most), scale, torch.full_like(scale, math.nan))


class Cache:
    """CPU tensors of a paged cache, [pages, page, Hkv, d], filled with what must never be read; `on_gpu` gives them in a layout."""

    def __init__(self, gen, dtype, pages, page, hkv, d, batch, width):
        self.dtype, self.page, self.hkv, self.d = dtype, page, hkv, d
        shape = (pages, page, hkv, d)
        self.tensors = {}
        for n in ("k", "v"):
            if dtype == torch.float16:
                self.tensors[n + "_pages"] = torch.full(shape, math.nan, dtype=dtype)
            else:
                self.tensors[n + "_pages"] = torch.full(shape, 0x7f, dtype=torch.uint8).view(dtype)  # (e4m3: NaN)
                self.tensors[n + "_scales"] = torch.full((pages, hkv), math.nan)
                self.tensors[n + "_tail"] = torch.full((batch, page, hkv, d), math.nan, dtype=torch.float16)
        self.order = torch.randperm(pages, generator=gen).tolist()
        self.table = torch.full((batch, width), -1, dtype=torch.int32)
        self.rows = {n: [torch.empty(0, hkv, d, dtype=torch.float16) for _ in range(batch)] for n in ("k", "v")}

    def reserve(self, entry, positions):
        for i in range((positions + self.page - 1) // self.page):
            if self.table[entry, i] < 0:
                self.table[entry, i] = self.order.pop()

    def append(self, entry, k, v):
        """fp16 rows [L,Hkv,d] (rotated already); the pages that exist for them are written as the operator would."""
        page = self.page
        for n, x in (("k", k), ("v", v)):
            start = self.rows[n][entry].shape[0]
            rows = self.rows[n][entry] = torch.cat([self.rows[n][entry], x])
            end = rows.shape[0]
            for i in range(start // page, (end + page - 1) // page):
                at = int(self.table[entry, i])
                part = rows[i * page:(i + 1) * page]
                if self.dtype == torch.float16:
                    first = max(start - i * page, 0)
                    if at >= 0:
                        self.tensors[n + "_pages"][at, first:part.shape[0]] = part[first:]
                elif part.shape[0] == page:
                    if at >= 0:
                        codes, scales = quantise(part, self.dtype)
                        self.tensors[n + "_pages"].view(torch.uint8)[at] = codes.view(torch.uint8)
                        self.tensors[n + "_scales"][at] = scales
                else:
                    first = max(start - i * page, 0)
                    self.tensors[n + "_tail"][entry, first:part.shape[0]] = part[first:]

    def on_gpu(self, layout):
        def lay(n, t):
            if n.endswith("scales"):
                return t.cuda()
            bits = t.view(torch.uint8) if t.dtype.itemsize == 1 else t
            bits = bits if layout == "bshd" else bits.transpose(1, 2).contiguous()
            return bits.cuda().view(t.dtype)
        return {n: lay(n, t) for n, t in self.tensors.items()}

    def check(self, got, layout):
        for n, want in self.tensors.items():
            x = got[n]
            if n.endswith("scales"):
                assert torch.equal(x.cpu().view(torch.int32), want.view(torch.int32)), n
                continue
            kind = torch.uint8 if x.dtype.itemsize == 1 else torch.int16
            x = x.view(kind)
            x = x if layout == "bshd" else x.transpose(1, 2)
            assert torch.equal(x.cpu(), want.view(kind)), n

    def dense(self, entry, n):
        """The rows of an entry as its cache holds them, [n,Hkv,d] in 64 bits."""
        out = []
        for name in ("k", "v"):
            rows = self.rows[name][entry].double().clone()
            if self.dtype != torch.float16:
                for i in range(n // self.page):
                    at = int(self.table[entry, i])
                    scales = self.tensors[name + "_scales"][at].double()[None, :, None]
                    rows[i * self.page:(i + 1) * self.page] = self.tensors[name + "_pages"][at].float().double() * scales
            out.append(rows[:n])
        return out


def attention(q, k, v, scale):
    """q [L,Hq,d] of the last L positions; k, v [n,Hkv,d] in 64 bits -> (o, sum of the weighted magnitudes of v)."""
    L, hq, _ = q.shape
    n, hkv, _ = k.shape
    o = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(o)
    for h in range(hq):
        w = q[:, h].double() @ k[:, h // (hq // hkv)].T * scale
        hidden = torch.arange(n)[None, :] > torch.arange(L)[:, None] + n - L
        w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
        w = torch.where(hidden, torch.zeros_like(w), w)  # (rows without a key are NaN)
        o[:, h] = w @ v[:, h // (hq // hkv)]
        mag[:, h] = w @ v[:, h // (hq // hkv)].abs()
    return o, mag


def assert_close(got, want, mag, n, vmax):
    """fp16 output and fp16 weights: a rounding of each, 2^-11 of the output and of the weighted magnitudes; weights below 2^-14
    of a row's largest are off by up to 2^-25 each.  A fifth more for 32-bit sums, exponentials and the merge of the splits."""
    bound = 1.2 * (2.0 ** -11 * (want.abs() + mag) + n * 2.0 ** -25 * vmax) + 1e-7
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3f} of the bound"
