"""GPU: how the split-K pass cuts entries into parts.  All keys count the same and the value rows of every 16 keys have a one in a
column of their own, so that each column of the output counts slices: one that a part left out or took twice shows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ONE = {torch.float16: 1.0, torch.int8: 127, torch.float8_e4m3fn: 448.0}


def _ramp(batch, low, high):
    return [low + (high - low) * i // (batch - 1) for i in range(batch)]


# Parts of a few lengths: the least one, one CTA for every place on the GPU, a few more CTAs than places (parts a quarter to a half
# longer, where those fit, and where they do not), several CTAs for every place; more entries than are counted in 16 bits.
CASES = {
    "least": ([900, 40, 1, 0, 3000], 1, 8, 8, 128, 16),
    "longer": ([6000] * 8, 5, 32, 8, 128, 64),
    "longer, short": ([2000] * 8, 5, 32, 8, 128, 16),
    "ragged, tokens": (_ramp(8, 500, 12000), 5, 32, 8, 128, 32),
    "one token": ([3000] * 16, 1, 8, 8, 128, 16),
    "wide heads": (_ramp(6, 100, 5000), 1, 16, 16, 256, 128),
    "narrow heads": ([32000] * 5 + [31, 17000], 1, 4, 4, 64, 64),
    "several places": (_ramp(40, 3000, 9000), 1, 8, 8, 128, 32),
    "several places, tokens": (_ramp(24, 100, 20000), 17, 8, 4, 64, 256),
    "many entries": ([3000] + [i % 90 for i in range(5000)] + [700], 1, 2, 1, 64, 16),
    "many entries, tokens": ([i % 300 for i in range(4500)] + [20000], 4, 1, 1, 64, 32),
    "as many as counted in 16 bits": ([i % 40 for i in range(4095)] + [60000], 1, 1, 1, 64, 16),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("case", list(CASES))
def test_every_slice_is_counted_once(dtype, case):
    import flash_attn_legacy as fal
    import flash_attn_legacy_cuda as ext
    lens, rows, hq, hkv, d, page = CASES[case]
    scaled = dtype != torch.float16
    used = [(n + page - 1) // page for n in lens]
    width = max(used) + 3
    pages = sum(used) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(len(lens)), dtype=torch.int32)
    at = 0
    for e, u in enumerate(used):
        table[e, :u] = order[at:at + u]
        at += u
    table = table.cuda()
    entry, index = torch.nonzero(table >= 0, as_tuple=True)
    # the value rows of the pages, by their positions
    pos = index[:, None] * page + torch.arange(page, device="cuda")
    ones = torch.nn.functional.one_hot(pos // 16 % d, d)
    v = torch.zeros((pages, page, hkv, d), dtype=torch.float32, device="cuda").to(dtype)
    v[table[entry, index].long()] = (ones * ONE[dtype]).to(torch.float32).to(dtype)[:, :, None].expand(-1, -1, hkv, -1)
    k = torch.zeros_like(v)
    n = torch.tensor(lens, device="cuda")
    extra = {}
    if scaled:
        extra["k_scales"] = torch.ones(pages, hkv, device="cuda")
        extra["v_scales"] = torch.full((pages, hkv), 1 / ONE[dtype], device="cuda")
        rest = (n // page * page)[:, None] + torch.arange(page, device="cuda")
        extra["v_tail"] = torch.nn.functional.one_hot(rest // 16 % d, d).half()[:, :, None].repeat(1, 1, hkv, 1)
        extra["k_tail"] = torch.zeros_like(extra["v_tail"])
    q = torch.randn(len(lens), rows, hq, d, generator=torch.Generator().manual_seed(1)).half().cuda()
    ext.reset_device_status()
    o = fal.flash_attn_with_paged_kvcache(q, k, v, table, n.int(), **extra)
    assert ext.device_status() == 0
    sees = (n[:, None] - rows + 1 + torch.arange(rows, device="cuda")).clamp(min=0)  # keys of every query
    slices = (sees + 15) // 16
    last = sees - (slices - 1) * 16  # keys of its last slice
    column = torch.arange(d, device="cuda")
    whole = (slices[..., None] - 1 - column).clamp(min=-1).div(d, rounding_mode="floor") + 1  # slices of the column
    count = whole * 16 - torch.where((slices[..., None] - 1) % d == column, 16 - last[..., None], 0) * (sees[..., None] > 0)
    want = (count.double() / sees.clamp(min=1)[..., None])[:, :, None]
    # Weights of 1, sums of whole numbers below 2^24.  The softmax sum adds weights / V's scale, in 32 bits: fewer than 200 sums in a
    # row, 2^-24 each, and V's scale by way of its logarithm, 2^-21: below 2^-16.  The output in fp16: 2^-11.
    assert bool(((o.double() - want).abs() <= want * (2.0 ** -11 + 2.0 ** -16) + 2.0 ** -25).all())
