"""GPU: paged caches made in inference mode are written inside of it only, as autograd has it."""
import pytest
import torch

from test_paged_gpu import _filled, _lens, _rows, _tables

pytestmark = pytest.mark.gpu


def _call(dtype):
    gen = torch.Generator().manual_seed(6)
    with torch.inference_mode():
        cache = _filled(gen, dtype, [20, 30], 16, 2, 64, extra=4)
        got = cache.on_gpu("bshd")
    q, k, v = (_rows(gen, 2, 2, h, 64).cuda() for h in (4, 2, 2))
    cos, sin = (t.cuda() for t in _tables(cache.table.shape[1] * 16, 64))
    return dict(q=q, k=k, v=v, rotary_cos=cos, rotary_sin=sin, block_table=cache.table.cuda(), cache_seqlens=_lens([20, 30]), **got)


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("native", [True, False])
def test_caches_made_in_inference_mode_are_not_written_outside_of_it(dtype, native, monkeypatch):
    import flash_attn_legacy as fal
    import flash_attn_legacy_cuda as ext
    if not native:
        monkeypatch.setattr(ext, "paged_attend_plain", ext._general)
        monkeypatch.setattr(ext, "paged_append_plain", ext._general)
    args = _call(dtype)
    caches = [n for n in args if n.endswith(("pages", "scales", "tail"))]
    before = {n: args[n].view(torch.uint8).clone() for n in caches}
    for call in (fal.flash_attn_with_paged_kvcache, fal.paged_cache_append):
        for context in (torch.no_grad, torch.enable_grad):
            with context(), pytest.raises(RuntimeError, match="inference"):
                call(**args)
    torch.cuda.synchronize()
    assert all(torch.equal(args[n].view(torch.uint8), t) for n, t in before.items())
    reads = {n: t for n, t in args.items() if n not in ("k", "v", "rotary_cos", "rotary_sin")}
    fal.flash_attn_with_paged_kvcache(**reads)  # reading them is all right
    with torch.inference_mode():
        fal.flash_attn_with_paged_kvcache(**args)
        fal.paged_cache_append(**args)
