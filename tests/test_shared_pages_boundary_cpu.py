"""CPU checks of serving in 8 bits on shared pages: the C ABI's argument errors (before any
launch; pointers are never dereferenced), workspace sizes, and the extension's refusals."""
import pytest
import torch

from ada_mla import capi
from test_operators_boundary_cpu import FAKE, _caller, _ext


@pytest.mark.parametrize("fn", ["mla_decode_paged_fp8_fp16", "mla_decode_paged_fp8_bf16"])
def test_paged_fp8_argument_errors(fn):
    names = "q kv scale bt cu out ws wsb batch heads total page pages stride splits stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(scale=0.5, wsb=1 << 40, batch=2, heads=16, total=100, page=64,
                                                   pages=10, stride=4, splits=0, stream=None)
    call = _caller(fn, names, ok)
    for bad in (dict(q=None), dict(kv=None), dict(bt=None), dict(cu=None), dict(out=None), dict(ws=None),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(batch=0),
                dict(heads=24), dict(heads=0), dict(heads=4112), dict(total=-1), dict(page=16), dict(page=96),
                dict(page=1 << 21), dict(pages=0), dict(stride=0)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(q=FAKE + 2), dict(kv=FAKE + 4), dict(out=FAKE + 8), dict(ws=FAKE + 4)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    assert call(wsb=16) == capi.STATUS_WORKSPACE_TOO_SMALL
    size = capi.load().mla_decode_paged_fp8_workspace_size
    assert size(2, 16, 100, 0) > 0 and size(0, 16, 100, 0) == size(2, 24, 100, 0) == size(2, 16, -1, 0) == 0
    # what the query gives is what the call asks for
    for heads, total, splits in ((16, 300000, 0), (32, 200000, 0), (64, 5000, 3), (128, 70000, 0)):
        ws = size(3, heads, total, splits)
        assert call(heads=heads, total=total, splits=splits, batch=3, wsb=ws - 1) == capi.STATUS_WORKSPACE_TOO_SMALL


def test_extension_refusals_paged_fp8():
    m = _ext()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    ok = dict(query=h(2, 16, 576), kv_cache=h(4, 64, 576).to(torch.float8_e4m3fn), block_table=i(2, 3), cu_seqlens=i(3),
              cache_scale=0.5)
    for bad, msg in ((dict(query=h(2, 16, 576).float()), "float8_e4m3fn"), (dict(cache_scale=0.0), "cache_scale"),
                     (dict(kv_cache=h(4, 64, 576)), "cache_scale is for"),
                     (dict(kv_cache=h(4, 64, 576).bfloat16()), "both be float16"),
                     (dict(kv_cache=h(4, 48, 576).to(torch.float8_e4m3fn)), "power of two"),
                     (dict(kv_cache=h(4, 64, 576).to(torch.float8_e5m2)), "both be float16"),
                     (dict(cu_seqlens=i(2)), "batch \\+ 1"), (dict(), "GPU tensors"),
                     (dict(query=h(2, 16, 576).bfloat16()), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_decode_paged(**{**ok, **bad})
