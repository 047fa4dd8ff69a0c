"""CPU checks of serving in 8 bits on shared pages: the C ABI's argument errors (before any
launch; pointers are never dereferenced), workspace sizes, and the extension's refusals."""
import pytest
import torch

from ada_mla import capi
from pages_reference import compact, fork
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


def test_fork_argument_errors():
    names = ("table lens parents kept pinned free start new new_lens copies next ws wsb rows batch pages num_free page "
             "stride stream")
    ok = {n: FAKE + 64 * i for i, n in enumerate(names.split())} | dict(
        wsb=1 << 30, rows=4, batch=4, pages=100, num_free=10, page=64, stride=4, stream=None)
    call = _caller("mla_fork_tables", names, ok)
    for bad in (dict(table=None), dict(lens=None), dict(parents=None), dict(free=None), dict(start=None), dict(new=None),
                dict(new_lens=None), dict(copies=None), dict(next=None), dict(ws=None), dict(rows=0), dict(rows=8193),
                dict(batch=0), dict(batch=2 ** 31 - 1), dict(pages=0), dict(pages=2 ** 18 + 1), dict(num_free=-1),
                dict(page=16), dict(page=48), dict(page=1 << 21), dict(stride=0), dict(stride=2 ** 20 + 1), dict(new=ok["table"]),
                dict(new_lens=ok["lens"]), dict(next=ok["start"])):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    assert call(ws=FAKE + 4) == capi.STATUS_MISALIGNED
    assert call(wsb=399) == capi.STATUS_WORKSPACE_TOO_SMALL


def test_compact_argument_errors():
    names = "table lens pinned free start new copies new_free ws wsb rows pages num_free page stride stream"
    ok = {n: FAKE + 64 * i for i, n in enumerate(names.split())} | dict(
        wsb=1 << 30, rows=4, pages=100, num_free=10, page=64, stride=4, stream=None)
    call = _caller("mla_compact_tables", names, ok)
    for bad in (dict(table=None), dict(lens=None), dict(free=None), dict(start=None), dict(new=None), dict(copies=None),
                dict(new_free=None), dict(ws=None), dict(rows=0), dict(rows=8193), dict(pages=0), dict(pages=2 ** 18 + 1),
                dict(num_free=-1), dict(page=16), dict(page=48), dict(stride=0), dict(new=ok["table"]),
                dict(new_free=ok["free"])):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    assert call(ws=FAKE + 4) == capi.STATUS_MISALIGNED
    assert call(wsb=399) == capi.STATUS_WORKSPACE_TOO_SMALL
    size = capi.load().mla_page_tables_workspace_size
    assert size(0) == size(2 ** 18 + 1) == 0 and size(1) >= 12 and size(2 ** 18) >= 4 * 2 ** 18 + 8


def test_copy_argument_errors():
    names = "cache copies count layers pages page size stream"
    ok = dict(cache=FAKE, copies=FAKE, count=3, layers=1, pages=10, page=64, size=2, stream=None)
    call = _caller("mla_copy_pages", names, ok)
    for bad in (dict(cache=None), dict(copies=None), dict(count=-1), dict(layers=0), dict(pages=0), dict(page=16),
                dict(page=96), dict(size=3), dict(size=8)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    assert call(cache=FAKE + 8) == capi.STATUS_MISALIGNED
    assert call(count=0, copies=None) == capi.STATUS_SUCCESS


def test_extension_refusals_pages():
    m = _ext()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pool = dict(block_table=i(2, 3), lens=i(2), free_pages=i(4), free_start=i(1), page_size=32, num_pages=9)
    for bad, msg in ((dict(block_table=i(2, 3).long()), "block_table must be"), (dict(block_table=i(2, 0)), "one column"),
                     (dict(lens=i(3)), "per request"), (dict(lens=i(2).long()), "lens must be"),
                     (dict(free_pages=i(4, 1)), "free_pages must be"), (dict(free_start=i(2)), "one entry"),
                     (dict(page_size=48), "power of two"), (dict(num_pages=0), "2\\^18"), (dict(num_pages=2 ** 18 + 1), "2\\^18"),
                     (dict(pinned=i(8)), "per page"), (dict(pinned=i(9).bool()), "pinned must be"),
                     (dict(block_table=i(8193, 3), lens=i(8193)), "8192"), (dict(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_compact_tables(**{**pool, **bad})
        with pytest.raises(RuntimeError, match=msg):
            m.mla_fork_tables(**{**pool, "parents": i(5), **bad})
    for bad, msg in ((dict(parents=i(0)), "at least one"), (dict(parents=i(5).long()), "parents must be"),
                     (dict(kept_lens=i(4)), "per parent"), (dict(free_pages=i(8)[::2]), "contiguous")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_fork_tables(**{**pool, "parents": i(5), **bad})
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    for cache, copies, msg in ((h(4, 64, 512), i(3, 3), "kv_cache must be"), (h(4, 576), i(3, 3), "kv_cache must be"),
                               (h(0, 64, 576), i(3, 3), "kv_cache must be"), (h(4, 48, 576), i(3, 3), "power of two"),
                               (h(4, 64, 1152)[..., :576], i(3, 3), "contiguous"),
                               (h(4, 64, 576).double(), i(3, 3), "1, 2 or 4"), (h(4, 64, 576), i(3, 2), "copies must be"),
                               (h(4, 64, 576), i(3, 3).long(), "copies must be"), (h(4, 64, 576), i(3, 3), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_copy_pages(cache, copies)


def test_pages_oracle_on_small_cases():
    # two rows share page 4; the first ends, the second is rolled back into its second page and forked
    t, lens, copies, nxt, free = fork([[4, 1], [4, 7]], [40, 64], [1, 1], [50, 50], [0] * 9, [-1, -1, -1, 8], 3, 32, 9)
    assert t == [[4, 7], [4, 1]] and lens == [50, 50] and copies == [[-1, -1, 0], [7, 1, 18]]
    assert nxt == 3 - 1 + 1 and free == [-1, -1, 1, 8]
    t, copies, free = compact([[8, 2], [5, -1]], [64, 3], [0] * 9, [-1, 0, 7, 3], 1, 32, 9)
    assert copies[:2] == [[8, 0, 32], [5, 3, 32]] and t == [[0, 2], [3, -1]] and free == [-1, 5, 7, 8]


@pytest.mark.parametrize("t", ["fp16", "bf16"])
def test_linear_argument_errors(t):
    call = _caller("mla_quantize_fp8_" + t, "x q s rows k stride stream",
                   dict(x=FAKE, q=FAKE, s=FAKE, rows=3, k=256, stride=256, stream=None))
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(rows=0), dict(rows=2 ** 26 + 1), dict(k=0), dict(k=24),
                dict(k=2 ** 22 + 16), dict(stride=-8), dict(stride=2 ** 22 + 8)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(x=FAKE + 2), dict(q=FAKE + 8), dict(stride=257)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    names = "x w ws out space bytes rows k n xstride wstride stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(bytes=1 << 40, rows=3, k=256, n=100, xstride=256, wstride=256, stream=None)
    common = (dict(x=None), dict(w=None), dict(ws=None), dict(out=None), dict(rows=0), dict(k=0), dict(k=24), dict(n=0),
              dict(n=2 ** 26 + 1), dict(rows=2 ** 26, n=2 ** 26), dict(xstride=-16), dict(wstride=-16),
              dict(wstride=2 ** 22 + 16))
    call = _caller("mla_linear_fp8_" + t, names, ok)
    for bad in (*common, dict(space=None)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(x=FAKE + 2), dict(w=FAKE + 8), dict(out=FAKE + 2), dict(space=FAKE + 4), dict(xstride=257), dict(wstride=264)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    assert call(bytes=16) == capi.STATUS_WORKSPACE_TOO_SMALL
    size = capi.load().mla_linear_fp8_workspace_size
    assert size(3, 256, 100) >= 3 * 256 + 3 * 2 * 4 and size(0, 256, 100) == size(3, 24, 100) == size(3, 256, 0) == 0
    names = "x xs w ws out space bytes rows k n xstride wstride srow sblock stream"
    call = _caller("mla_linear_fp8_quantized_" + t, names, {n: ok.get(n, FAKE) for n in names.split()} | dict(srow=2, sblock=1))
    for bad in (*common, dict(xs=None), dict(space=None), dict(srow=-1), dict(srow=2 ** 20 + 1), dict(sblock=-1)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(x=FAKE + 8), dict(w=FAKE + 8), dict(out=FAKE + 2), dict(space=FAKE + 4), dict(xstride=264), dict(wstride=264)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    assert call(bytes=16) == capi.STATUS_WORKSPACE_TOO_SMALL


def test_extension_refusals_linear():
    m = _ext()
    f8 = torch.float8_e4m3fn
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    ok = dict(x=h(3, 272), weight=h(200, 272).to(f8), weight_scale=torch.zeros(2, 3))
    for bad, msg in ((dict(x=h(3, 272).float()), "x must be float16"), (dict(x=h(3, 264)), "multiple of 16"),
                     (dict(x=h(3, 256)), "weight must be"), (dict(weight=h(200, 272)), "weight must be"),
                     (dict(weight=h(0, 272).to(f8)), "weight must be"), (dict(weight_scale=torch.zeros(2, 2)), "weight_scale must be"),
                     (dict(weight_scale=torch.zeros(3, 3)), "weight_scale must be"),
                     (dict(weight_scale=torch.zeros(2, 3).double()), "weight_scale must be"),
                     (dict(x_scale=torch.zeros(3, 3)), "x_scale comes with"), (dict(x=h(3, 272).to(f8)), "x_scale comes with"),
                     (dict(x=h(3, 272).to(f8), x_scale=torch.zeros(3, 2)), "x_scale must be"),
                     (dict(x=h(3, 272).to(f8), x_scale=torch.zeros(3, 3).half()), "x_scale must be"),
                     (dict(x=h(3, 272).to(f8), x_scale=torch.zeros(3, 3), dtype=torch.float32), "dtype must be"),
                     (dict(dtype=torch.bfloat16), "dtype is for"), (dict(x=torch.zeros((), dtype=torch.float16)), "inputs"),
                     (dict(), "GPU tensors"), (dict(x=h(3, 272).to(f8), x_scale=torch.zeros(3, 3)), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_linear_fp8(**{**ok, **bad})
    for x, msg in ((h(3, 272).float(), "float16 or bfloat16"), (h(3, 24), "multiple of 16"), (h(3, 0), "multiple of 16"),
                   (torch.zeros((), dtype=torch.float16), "inputs"), (h(3, 272), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_quantize_fp8(x)
