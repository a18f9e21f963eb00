"""Paged key/value caches: rows in pages that a table names, in fp16 or in 8 bits with a scale for each page and head.

Not in sirCamp/flash-attention-legacy, whose hook attends eagerly over the dense cache that the framework around it keeps
(flash_attn_legacy/integrations.py:77-98).

A cache is a set of tensors:

    k_pages, v_pages  [num_pages, page, Hkv, d] ("bshd") or [num_pages, Hkv, page, d] ("bhsd"); page: 16, 32, 64, 128, 256
                      rows; float16, int8 or float8_e4m3fn
    block_table       int32 [B, pages per entry]: position p of entry b is row p % page of page block_table[b, p // page]
    cache_seqlens     int32 [B]: positions that an entry holds; negative: an unused entry of a padded batch
    and for 8-bit pages
    k_scales, v_scales  float32 [num_pages, Hkv], not negative: a value is code * scale
    k_tail, v_tail    float16 [B, page, Hkv, d] (or [B, Hkv, page, d]): the rows of an entry's last, unfinished page

An 8-bit page is written when its last row arrives, from fp16 rows and with the largest magnitude of each head as its
scale (a / 127 or a / 448), so that a row is rounded to 8 bits once and the cache does not depend on how the rows came in.
The tail belongs to the batch entry: a program that moves an entry to another place in the batch moves its tail along.
"""
import math
from typing import Optional

import torch
from torch.autograd.forward_ad import unpack_dual

import flash_attn_legacy_cuda

from .flash_attn import SUPPORTED_HEAD_DIMS, _kernel_ready


def _inference_only(*tensors):
    tensors = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("paged caches are inference only: call under torch.no_grad() or detach the inputs")
    if any(unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("paged caches are inference only: they take no forward-mode tangents")


def _writable(*tensors):
    if not torch.is_inference_mode_enabled() and any(t is not None and t.is_inference() for t in tensors):
        raise RuntimeError("a paged cache made in inference mode is not to be written outside of it")


def _written(*tensors):
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def paged_cache_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    q: Optional[torch.Tensor] = None,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    rotary_interleaved: bool = False,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    k_tail: Optional[torch.Tensor] = None,
    v_tail: Optional[torch.Tensor] = None,
    cache_layout: str = "bshd",
):
    """Writes new rows into a paged cache, rotated by their positions on the way; returns (rotated q or None, new lengths).

    k, v [B,L,Hkv,d] fp16 go to positions cache_seqlens[b] ... + L - 1 of every entry; `cache_seqlens` itself is not
    modified.  With rotary_cos / rotary_sin ([positions, rotary_dim / 2], fp32 or fp16, positions for the whole block table)
    the first rotary_dim columns of k, and of q [B,L,Hq,d] if given, are rotated: columns i and i + rotary_dim / 2 together,
    or 2 i and 2 i + 1 with `rotary_interleaved`.  Rows without a place are dropped and the device status word becomes 2000:
    those behind the end of the block table, whose queries become 0 (as those of unused entries do), and those whose table
    entry names no page (with 8-bit pages the whole page, when it is full), whose queries are rotated like any other.  The new
    lengths end at the end of the table.  Pages that new rows go to must not be shared between entries.
    """
    # the ordinary call in one native function; None: any other
    out = flash_attn_legacy_cuda.paged_append_plain(k, v, k_pages, v_pages, block_table, cache_seqlens, rotary_cos, rotary_sin,
                                                    rotary_interleaved, k_scales, v_scales, k_tail, v_tail, cache_layout, q)
    if out is not None:
        return out
    assert k.dim() == 4 and v.dim() == 4, "k and v must be [B, L, H_kv, d]"
    assert k.dtype == torch.float16 and v.dtype == torch.float16, f"k and v must be float16, got {k.dtype}, {v.dtype}"
    assert q is None or q.dtype == torch.float16, f"Q must be float16, got {q.dtype}"
    d = k.shape[-1]
    assert d in SUPPORTED_HEAD_DIMS, f"head_dim must be 32, 64, 96, 128, or 256, got {d}"
    _inference_only(q, k, v, rotary_cos, rotary_sin, k_pages, v_pages, k_scales, v_scales, k_tail, v_tail)
    _writable(k_pages, v_pages, k_scales, v_scales, k_tail, v_tail)
    out = flash_attn_legacy_cuda.paged_append(
        _kernel_ready(k), _kernel_ready(v), k_pages, v_pages, block_table.to(torch.int32), cache_seqlens.to(torch.int32),
        _kernel_ready(q) if q is not None else None, rotary_cos, rotary_sin, rotary_interleaved,
        k_scales, v_scales, k_tail, v_tail, cache_layout)
    _written(k_pages, v_pages, k_scales, v_scales, k_tail, v_tail)
    return out


def flash_attn_with_paged_kvcache(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    rotary_interleaved: bool = False,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
    k_tail: Optional[torch.Tensor] = None,
    v_tail: Optional[torch.Tensor] = None,
    cache_layout: str = "bshd",
) -> torch.Tensor:
    """Attention of new query tokens against a paged cache: `flash_attn_with_kvcache` over pages.

    q [B,L,Hq,d]; returns [B,L,Hq,d].  If k, v ([B,L,Hkv,d]) are given they are first appended at cache_seqlens[b], they and
    q rotated if rotary tables are given (`paged_cache_append`).  Without them the cache holds the new tokens' rows already:
    they are the last L of cache_seqlens[b] positions.  Query i sees everything up to its own position; a query without
    any gives 0, and so does a token that runs over the end of its block table (the device status word is 2000 then; the
    lengths that `paged_cache_append` returns end there and would not tell where the tokens that fit are).  What the pages hold behind an entry's length does not matter; a position within it that has no page counts
    as a row of zeros and the device status word becomes 3000.  (Between new tokens the mask is a weight of 0: a NaN or an
    infinity in the value row of one of them reaches the earlier ones of the same call.)  Inference only.

    A call that is refused has not appended anything.  Should a launch fail behind the append, the error says so: the rows are
    in the cache then, and the same rows are not to be appended again.

    Up to 32 tokens run on a split-K pass that reads every page once for up to 32 (token, head) rows of a KV head; more run on
    the forward kernel, over the pages put in order in a workspace as large as the block table allows for (up to
    1 GiB at a time): pass a view of the table's first columns where entries are much shorter than it.
    """
    out = flash_attn_legacy_cuda.paged_attend_plain(q, k, v, k_pages, v_pages, block_table, cache_seqlens, rotary_cos, rotary_sin,
                                                    rotary_interleaved, k_scales, v_scales, k_tail, v_tail, cache_layout,
                                                    softmax_scale)
    if out is not None:
        return out
    assert q.dim() == 4, "q must be [B, L, H_q, d]"
    assert q.dtype == torch.float16, f"Q must be float16, got {q.dtype}"
    d = q.shape[-1]
    assert d in SUPPORTED_HEAD_DIMS, f"head_dim must be 32, 64, 96, 128, or 256, got {d}"
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(d)
    block_table, cache_seqlens = block_table.to(torch.int32), cache_seqlens.to(torch.int32)
    q, append = _kernel_ready(q), None
    if k is not None:
        assert v is not None and q.shape[:2] == k.shape[:2], "k, v must be [B, L, H_kv, d]"

        def append():
            turned, _ = paged_cache_append(
                k, v, k_pages, v_pages, block_table, cache_seqlens, q if rotary_cos is not None else None, rotary_cos, rotary_sin,
                rotary_interleaved, k_scales, v_scales, k_tail, v_tail, cache_layout)
            return turned if turned is not None else q
    else:
        assert v is None and rotary_cos is None and rotary_sin is None, "v and the rotary tables go with k"
    _inference_only(q, k_pages, v_pages, k_scales, v_scales, k_tail, v_tail)
    return flash_attn_legacy_cuda.paged_attention(q, k_pages, v_pages, block_table, cache_seqlens, softmax_scale, k_scales,
                                                  v_scales, k_tail, v_tail, cache_layout, append)
