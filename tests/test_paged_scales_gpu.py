"""GPU: attention over 8-bit pages whose scales are far apart, down to the 0 of a page of zeros."""
import math

import pytest
import torch

from paged_reference import Cache, assert_close, attention
from test_paged_gpu import DTYPES, _lens

pytestmark = pytest.mark.gpu


# One key of the largest value there is; all others are pages of zeros, each with a weight of 2^-20 of that key's, together 2^-5.
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 8, 40])
@pytest.mark.parametrize("front", [True, False])
def test_keys_of_pages_of_zeros_keep_their_weights(dtype, rows, front):
    import flash_attn_legacy as fal
    gen = torch.Generator().manual_seed(1)
    hq, hkv, d, page, n = 2, 1, 64, 256, 1 << 15
    cache = Cache(gen, DTYPES[dtype], n // page, page, hkv, d, 1, n // page)
    cache.reserve(0, n)
    at = 7 if front else n - rows - 9
    k, v = torch.zeros(n, hkv, d), torch.zeros(n, hkv, d)
    k[:, 0, 0] = -20 * math.log(2) / 8
    own = at // page * page
    k[own:own + page, 0, 0] = -8.0  # (times q's 8: the page's other keys count for nothing)
    k[at, 0, 0] = 0
    v[at] = 65504
    cache.append(0, k.half(), v.half())
    q = torch.zeros(1, rows, hq, d).half()
    q[..., 0] = 8
    o = fal.flash_attn_with_paged_kvcache(q.cuda(), block_table=cache.table.cuda(), cache_seqlens=_lens([n]), softmax_scale=1.0,
                                          **cache.on_gpu("bshd")).cpu()
    kd, vd = cache.dense(0, n)
    want, mag = attention(q[0], kd, vd, 1.0)
    assert want[0, 0, 0] < 0.98 * 65504
    assert_close(o[0], want, mag, n, 65504.0)
