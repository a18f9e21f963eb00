"""GPU: a call that appends and attends writes its rows once, also where the attention behind the append ends with an error."""
import ctypes

import pytest
import torch

from test_paged_gpu import _filled, _lens, _rows

pytestmark = pytest.mark.gpu

CUDA_ERROR = -5


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("dtype", ["float16", "int8", "float8_e4m3fn"])
def test_rows_are_appended_once(path, dtype, monkeypatch):
    """The library's attention stands in as a function that fails the first time; the new rows fill a page and begin another."""
    import flash_attn_legacy as fal
    import flash_attn_legacy_cuda as ext
    if path == "native" and ext._host is None:
        pytest.skip("no native host path was built")
    gen = torch.Generator().manual_seed(5)
    lens, rows, hq, hkv, d, page = [12, 30], 6, 4, 2, 64, 16
    cache = _filled(gen, getattr(torch, dtype), lens, page, hkv, d, extra=rows)
    got = cache.on_gpu("bshd")
    q, k, v = (_rows(gen, 2, rows, h, d).cuda() for h in (hq, hkv, hkv))
    attempts, appends = [], []

    def attend(block):
        attempts.append(block)
        return CUDA_ERROR if len(attempts) == 1 else real_lib.fal_paged_attn_run(ctypes.cast(block, ctypes.c_char_p))

    def append(block):
        appends.append(block)
        return real_append(block)

    call = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)
    real_append = call(ctypes.cast(ext._lib.fal_paged_append_run, ctypes.c_void_p).value)
    stand_ins = call(append), call(attend)

    class Lib:  # the library with both functions replaced
        fal_paged_append_run = staticmethod(lambda block: append(ctypes.cast(ctypes.c_char_p(block), ctypes.c_void_p).value))
        fal_paged_attn_run = staticmethod(lambda block: attend(block))

        def __getattr__(self, name):
            return getattr(real_lib, name)

    real_lib = ext._lib
    if path == "native":
        address = [ctypes.cast(f, ctypes.c_void_p).value for f in (
            ext._fwd_run, ext._decode_run, real_lib.fal_decode_workspace_bytes, *stand_ins, real_lib.fal_paged_attn_workspace_bytes)]
        host = type(ext._host)(*address[:3], ext._decode_ws, ext._DECODE_WS_MIN, *address[3:])
        host.set_status(q.get_device(), ext._status_ptr(q.get_device()))
        monkeypatch.setattr(ext, "paged_attend_plain", host.paged_attend)
    else:
        monkeypatch.setattr(ext, "paged_attend_plain", ext._general)
    monkeypatch.setattr(ext, "paged_append_plain", ext._general)
    monkeypatch.setattr(ext, "_lib", Lib())
    with pytest.raises(RuntimeError, match="has been made"):
        fal.flash_attn_with_paged_kvcache(q, block_table=cache.table.cuda(), cache_seqlens=_lens(lens), k=k, v=v, **got)
    assert len(attempts) == len(appends) == 1
    for e in range(2):
        cache.append(e, k[e].cpu(), v[e].cpu())
    cache.check(got, "bshd")
