"""GPU: the paged operators are inference only; what autograd has a say in is refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from test_paged_gpu import _filled, _lens, _rows, _tables

pytestmark = pytest.mark.gpu


def _call(dtype):
    """Arguments of a call that appends and attends, or appends alone."""
    gen = torch.Generator().manual_seed(6)
    cache = _filled(gen, dtype, [20, 30], 16, 2, 64, extra=4)
    got = cache.on_gpu("bshd")
    q, k, v = (_rows(gen, 2, 2, h, 64).cuda() for h in (4, 2, 2))
    cos, sin = (t.cuda() for t in _tables(cache.table.shape[1] * 16, 64))
    return dict(q=q, k=k, v=v, rotary_cos=cos, rotary_sin=sin, block_table=cache.table.cuda(), cache_seqlens=_lens([20, 30]), **got)


FLOATS = ["q", "k", "v", "rotary_cos", "rotary_sin", "k_scales", "v_scales", "k_tail", "v_tail"]


@pytest.mark.parametrize("name", FLOATS + ["k_pages", "v_pages"])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(name, grad):
    import flash_attn_legacy as fal
    args = _call(torch.float16 if name.endswith("pages") else torch.int8)
    before = {n: t.clone() for n, t in args.items()}
    with fwd_ad.dual_level(), torch.set_grad_enabled(grad):
        args[name] = fwd_ad.make_dual(args[name], torch.ones_like(args[name]))
        for call in (fal.flash_attn_with_paged_kvcache, fal.paged_cache_append):
            with pytest.raises(RuntimeError, match="inference only"):
                call(**args)
    torch.cuda.synchronize()
    for n, t in before.items():  # (bit by bit: what the cache does not hold is NaN)
        assert torch.equal(args[n].view(torch.uint8), t.view(torch.uint8)), n


@pytest.mark.parametrize("name", FLOATS)
def test_gradients_are_refused(name):
    import flash_attn_legacy as fal
    args = _call(torch.int8)
    args[name] = args[name].clone().requires_grad_()
    for call in (fal.flash_attn_with_paged_kvcache, fal.paged_cache_append):
        with pytest.raises(RuntimeError, match="inference only"):
            call(**args)
        with torch.no_grad():
            call(**args)
