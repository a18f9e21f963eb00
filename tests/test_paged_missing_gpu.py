"""GPU: every number that names no page is reported, the smallest integers among them."""
import math

import pytest
import torch

from paged_reference import assert_close, attention
from test_paged_gpu import DTYPES, _filled, _lens, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("number", [-2 ** 31, -2 ** 31 + 1, -1, 2 ** 31 - 1])
def test_numbers_that_name_no_page(dtype, rows, number):
    import flash_attn_legacy as fal
    import flash_attn_legacy_cuda as ext
    gen = torch.Generator().manual_seed(6)
    hq, hkv, d, page, n = 4, 2, 64, 16, 100
    cache = _filled(gen, DTYPES[dtype], [n], page, hkv, d)
    q = _rows(gen, 1, rows, hq, d)
    table = cache.table.clone()
    table[0, 2] = number
    ext.reset_device_status()
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=table.cuda(), cache_seqlens=_lens([n]), **cache.on_gpu("bshd")).cpu()
    status = ext.device_status()
    ext.reset_device_status()
    assert status == 3000
    k, v = cache.dense(0, n)
    k[2 * page:3 * page] = 0
    v[2 * page:3 * page] = 0
    want, mag = attention(q[0], k, v, 1 / math.sqrt(d))
    assert_close(o[0], want, mag, n, v.abs().max().item())
