"""CPU checks of the operators around the decode: the C ABI's argument errors
(before any launch; pointers are never dereferenced), workspace sizes, and the
extension's refusals."""
import pytest
import torch

from ada_mla import capi
from operators_reference import tables

FAKE = 0x10000


def _ext():
    import ada_mla
    return ada_mla.extension()


def _caller(fn, names, ok):
    f = getattr(capi.load(), fn)

    def call(**kw):
        a = {**ok, **kw}
        return f(*[a[n] for n in names.split()])
    return call


def test_tables_argument_errors():
    names = "context new free start table cu cu_new slots positions next batch total num_free page stride stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(start=FAKE + 64, batch=4, total=100, num_free=10, page=64, stride=4,
                                                   stream=None)
    call = _caller("mla_paged_tables", names, ok)
    for bad in (dict(context=None), dict(new=None), dict(start=None), dict(table=None), dict(cu=None),
                dict(cu_new=None), dict(next=None), dict(free=None), dict(slots=None), dict(positions=None),
                dict(next=FAKE + 64), dict(batch=0), dict(total=-1), dict(num_free=-1), dict(page=16), dict(page=48),
                dict(page=1 << 21), dict(stride=0)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad


@pytest.mark.parametrize("fn", ["mla_append_kv_fp16", "mla_append_kv_bf16"])
def test_append_argument_errors(fn):
    names = "kv w cs pos slots q cache out eps scale tokens heads npos rows kvs qts qhs flags stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(eps=1e-6, scale=1.0, tokens=3, heads=16, npos=10, rows=64, kvs=576,
                                                   qts=1024, qhs=64, flags=0, stream=None)
    call = _caller(fn, names, ok)
    for bad in (dict(kv=None), dict(w=None), dict(cs=None), dict(pos=None), dict(slots=None), dict(cache=None),
                dict(q=None), dict(out=None), dict(tokens=0), dict(heads=-1), dict(heads=4097), dict(npos=0),
                dict(rows=0), dict(kvs=-8), dict(eps=-1.0), dict(eps=float("nan")), dict(scale=0.0),
                dict(scale=float("inf")), dict(flags=1), dict(qts=-8), dict(tokens=2 ** 31 - 1)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(kv=FAKE + 2), dict(w=FAKE + 2), dict(cs=FAKE + 4), dict(cache=FAKE + 8), dict(q=FAKE + 2),
                dict(out=FAKE + 2), dict(kvs=577), dict(qts=1025), dict(qhs=65)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad


@pytest.mark.parametrize("fn", ["mla_decode_tree_fp16", "mla_decode_tree_bf16"])
def test_tree_argument_errors(fn):
    names = "q kv bt cu mask lens out ws wsb batch drafts heads total page pages stride splits stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(wsb=1 << 40, batch=2, drafts=4, heads=16, total=100, page=64,
                                                   pages=10, stride=4, splits=0, stream=None)
    call = _caller(fn, names, ok)
    for bad in (dict(q=None), dict(kv=None), dict(bt=None), dict(cu=None), dict(mask=None), dict(out=None),
                dict(ws=None), dict(batch=0), dict(drafts=0), dict(drafts=65), dict(heads=24), dict(heads=0),
                dict(heads=4112), dict(total=-1), dict(total=2 ** 31 - 1), dict(page=16), dict(page=96), dict(pages=0),
                dict(stride=0), dict(batch=2 ** 30)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(q=FAKE + 2), dict(kv=FAKE + 4), dict(out=FAKE + 8), dict(ws=FAKE + 4)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    assert call(wsb=16) == capi.STATUS_WORKSPACE_TOO_SMALL


@pytest.mark.parametrize("fn", ["mla_prefill_fp16", "mla_prefill_bf16"])
def test_prefill_argument_errors(fn):
    names = "qn qr uk uv kv bt cq cu out ws wsb batch heads queries total page pages stride stream"
    ok = dict.fromkeys(names.split(), FAKE) | dict(wsb=1 << 40, batch=2, heads=16, queries=50, total=100, page=64,
                                                   pages=10, stride=4, stream=None)
    call = _caller(fn, names, ok)
    for bad in (dict(qn=None), dict(qr=None), dict(uk=None), dict(uv=None), dict(kv=None), dict(cq=None),
                dict(cu=None), dict(out=None), dict(ws=None), dict(batch=0), dict(heads=24), dict(heads=0),
                dict(queries=0), dict(total=-1), dict(total=2 ** 31 - 1), dict(page=48), dict(pages=0), dict(stride=0),
                dict(batch=2 ** 30)):
        assert call(**bad) == capi.STATUS_INVALID_VALUE, bad
    for bad in (dict(qn=FAKE + 2), dict(qr=FAKE + 2), dict(uk=FAKE + 2), dict(uv=FAKE + 2), dict(kv=FAKE + 2),
                dict(out=FAKE + 2), dict(ws=FAKE + 2)):
        assert call(**bad) == capi.STATUS_MISALIGNED, bad
    assert call(wsb=16) == capi.STATUS_WORKSPACE_TOO_SMALL


def test_workspace_sizes():
    lib = capi.load()
    assert lib.mla_decode_tree_workspace_size(1, 65, 16, 100, 0) == 0
    assert lib.mla_decode_tree_workspace_size(1, 4, 24, 100, 0) == 0
    assert lib.mla_decode_tree_workspace_size(1, 4, 16, 0, 0) > 0
    assert lib.mla_prefill_workspace_size(1, 24, 50, 100) == 0
    assert lib.mla_prefill_workspace_size(0, 16, 50, 100) == 0
    # K and V of whole tiles of 64 keys, at least 512 bytes a key and head
    assert lib.mla_prefill_workspace_size(3, 16, 1000, 1000) >= 1000 * 16 * 512
    # it never falls as the batch or the tokens grow
    for a, b in (((1, 16, 50, 100), (2, 16, 50, 100)), ((4, 32, 50, 100), (4, 32, 50, 101)), ((4, 32, 50, 127), (4, 32, 50, 128))):
        assert lib.mla_prefill_workspace_size(*a) <= lib.mla_prefill_workspace_size(*b)


def test_tree_splits_are_clamped_to_blocks():
    lib = capi.load()
    size = lib.mla_decode_tree_workspace_size
    # 100 tokens are 4 blocks of 32, whatever is asked for
    assert size(1, 4, 16, 100, 4) == size(1, 4, 16, 100, 5) == size(1, 4, 16, 100, 2 ** 31 - 1)
    assert size(3, 4, 16, 2 ** 31 - 5000, 2 ** 31 - 1) > 0
    assert size(1, 64, 4096, 0, 0) > 0


def test_extension_refusals_tables():
    m = _ext()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(context_lens=i(2), new_lens=i(2), block_table=i(2, 3), free_pages=i(4), free_start=i(1), page_size=32,
              total_new=5)
    for bad, msg in ((dict(context_lens=i(2).long()), "context_lens must be"), (dict(new_lens=i(3)), "per request"),
                     (dict(block_table=i(3, 3)), "per request"), (dict(block_table=i(2, 0)), "one column"),
                     (dict(block_table=i(3, 2).t()), "contiguous"), (dict(free_start=i(2)), "one entry"),
                     (dict(page_size=48), "power of two"), (dict(total_new=-1), "total_new"),
                     (dict(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_paged_tables(**{**ok, **bad})


def test_extension_refusals_append():
    m = _ext()
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    ok = dict(kv=h(3, 576), norm_weight=h(512), cos_sin=torch.zeros(9, 64), positions=torch.zeros(3, dtype=torch.int32),
              slots=torch.zeros(3, dtype=torch.int64), kv_cache=h(64, 576), q_rope=h(3, 16, 64))
    for bad, msg in ((dict(kv=h(3, 576).float()), "float16 or bfloat16"), (dict(kv=h(3, 512)), "kv must be"),
                     (dict(norm_weight=h(576)), "norm_weight"), (dict(norm_weight=h(512).bfloat16()), "norm_weight"),
                     (dict(cos_sin=h(9, 64)), "cos_sin"), (dict(cos_sin=torch.zeros(9, 32)), "cos_sin"),
                     (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
                     (dict(positions=torch.zeros(2, dtype=torch.int32)), "one entry per token"),
                     (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots"),
                     (dict(kv_cache=h(64, 512)), "kv_cache must be"), (dict(kv_cache=h(0, 576)), "kv_cache must be"),
                     (dict(kv_cache=h(64, 576).bfloat16()), "kv's dtype"),
                     (dict(kv_cache=h(64, 1152)[:, :576]), "contiguous"),
                     (dict(q_rope=h(3, 16, 32)), "q_rope must be"), (dict(q_rope=h(3, 0, 64)), "q_rope must be"),
                     (dict(q_rope=h(3, 16, 64).bfloat16()), "q_rope must have"),
                     (dict(eps=-1.0), "eps"), (dict(cache_scale=0.0), "cache_scale"),
                     (dict(cache_scale=0.5), "float8"), (dict(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_append_kv(**{**ok, **bad})


def test_extension_refusals_tree():
    m = _ext()
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(query=h(2, 4, 16, 576), kv_cache=h(4, 64, 576), block_table=i(2, 3), cu_seqlens=i(3),
              tree_mask=torch.zeros(2, 4, dtype=torch.int64))
    for bad, msg in ((dict(query=h(2, 16, 576)), "query must be"), (dict(query=h(2, 65, 16, 576)), "1 to 64"),
                     (dict(query=h(2, 4, 24, 576)), "multiple of 16"), (dict(query=h(2, 4, 16, 576).float()), "both be float16"),
                     (dict(kv_cache=h(4, 48, 576)), "power of two"), (dict(kv_cache=h(256, 576)), "kv_cache must be"),
                     (dict(kv_cache=h(4, 64, 576).bfloat16()), "both be float16"), (dict(block_table=i(1, 3)), "batch rows"),
                     (dict(cu_seqlens=i(2)), "batch \\+ 1"), (dict(tree_mask=i(2, 4)), "tree_mask"),
                     (dict(tree_mask=torch.zeros(2, 5, dtype=torch.int64)), "tree_mask"),
                     (dict(draft_lens=i(3)), "per request"), (dict(draft_lens=i(2).long()), "draft_lens"),
                     (dict(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_decode_tree(**{**ok, **bad})


def test_extension_refusals_prefill():
    m = _ext()
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ok = dict(q_nope=h(5, 16, 128), q_rope=h(5, 16, 64), w_uk=h(16, 128, 512), w_uv=h(16, 128, 512), kv_cache=h(9, 576),
              cu_q=i(3), cu_seqlens=i(3))
    paged = dict(kv_cache=h(4, 64, 576), block_table=i(2, 3))
    for bad, msg in ((dict(q_nope=h(5, 16, 64)), "q_nope must be"), (dict(q_nope=h(0, 16, 128)), "q_nope must be"),
                     (dict(q_nope=h(5, 24, 128)), "multiple of 16"), (dict(q_nope=h(5, 16, 128).float()), "float16 or"),
                     (dict(q_rope=h(4, 16, 64)), "q_rope must be"), (dict(w_uk=h(16, 512, 128)), "w_uk and w_uv"),
                     (dict(w_uv=h(8, 128, 512)), "w_uk and w_uv"), (dict(w_uv=h(16, 128, 512).bfloat16()), "dtype"),
                     (dict(cu_q=i(3).long()), "cu_q"), (dict(cu_seqlens=i(4)), "batch \\+ 1"), (dict(cu_q=i(1)), "batch \\+ 1"),
                     (dict(kv_cache=h(4, 64, 576)), "packed"), (dict(total_tokens=10), "exceeds"),
                     ({**paged, "kv_cache": h(9, 576)}, "paged"), ({**paged, "kv_cache": h(4, 48, 576)}, "power of two"),
                     ({**paged, "block_table": i(3, 3)}, "batch rows"), (paged, "GPU tensors"), (dict(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=msg):
            m.mla_prefill(**{**ok, **bad})


def test_table_oracle_on_a_small_case():
    # two requests on pages of 32: one page held and half full, one new request of 40 tokens
    t, cu, cu_new, slots, positions, nxt = tables([20, 0], [15, 40], [[5, -1], [-1, -1]], [9, 8, 7], 0, 32, 56)
    assert t == [[5, 9], [8, 7]] and cu == [0, 35, 75] and cu_new == [0, 15, 55] and nxt == 3
    assert slots[:15] == [5 * 32 + 20 + i for i in range(12)] + [9 * 32 + i for i in range(3)]
    assert slots[15:] == [8 * 32 + i for i in range(32)] + [7 * 32 + i for i in range(8)] + [-1]
    assert positions[:2] == [20, 21] and positions[15] == 0 and positions[-1] == 0
