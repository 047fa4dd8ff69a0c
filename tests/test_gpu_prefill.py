"""Causal attention of prompts in the expanded form (mla_prefill) against
float64. Tolerances: operators_reference."""
import random

import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import attention_check, gather_paged, half_step, paged_case

pytestmark = pytest.mark.gpu


def _inputs(gen, queries, heads, dtype):
    qn = torch.randn(max(1, queries), heads, 128, generator=gen).to(dtype).cuda()
    qr = torch.randn(max(1, queries), heads, 64, generator=gen).to(dtype).cuda()
    uk, uv = ((torch.randn(heads, 128, 512, generator=gen) * 512 ** -0.5).to(dtype).cuda() for _ in range(2))
    return qn, qr, uk, uv


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _check(got, qn, qr, uk, uv, rows, queries, lengths, dtype, what):
    se = sn = 0.0
    at = 0
    uk, uv, got = uk.double().cpu(), uv.double().cpu(), got.cpu()
    for b, (m, n) in enumerate(zip(queries, lengths)):
        c = rows(b)
        seen = torch.arange(n)[None] <= torch.arange(m)[:, None] + n - m
        for h in range(uk.shape[0]):
            k = torch.cat([c[:, :512] @ uk[h].T, c[:, 512:]], 1)
            q = torch.cat([qn[at:at + m, h], qr[at:at + m, h]], 1).double().cpu()
            e = attention_check(got[at:at + m, h], q, k, c[:, :512] @ uv[h].T, seen, dtype, rounded_kv=True,
                                what=f"{what} request {b} head {h}")
            se, sn = se + e[0], sn + e[1]
        at += m
    if sn:
        assert (se / sn) ** 0.5 <= 2 * half_step(dtype), f"{what}: 2-norm {(se / sn) ** 0.5:.2e}"


def _run(queries, context, heads, dtype, page, seed):
    rng = random.Random(seed)
    gen = torch.Generator()
    gen.manual_seed(seed)
    lengths = [q + c for q, c in zip(queries, context)]
    qn, qr, uk, uv = _inputs(gen, sum(queries), heads, dtype)
    cu_q, cu = _cu(queries), _cu(lengths)
    if page:
        cache, table, _ = paged_case(gen, rng, lengths, page, dtype)
        rows = lambda b: gather_paged(cache, table[b], lengths[b])  # noqa: E731
    else:
        cache, table = torch.randn(max(1, sum(lengths)), 576, generator=gen).to(dtype).cuda(), None
        rows = lambda b: cache[int(cu[b]):int(cu[b + 1])].double().cpu()  # noqa: E731
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu_q, cu, block_table=table, total_tokens=sum(lengths))
    torch.cuda.synchronize()
    _check(got, qn, qr, uk, uv, rows, queries, lengths, dtype, f"{queries} {context} heads {heads} page {page}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [0, 32, 256])
def test_lengths_at_edges(page, dtype):
    _run([1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200], [0] * 12, 16, dtype, page, seed=page)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [0, 64])
def test_chunks_behind_a_context(page, dtype):
    _run([1, 40, 128, 7, 150], [300, 64, 1, 0, 129], 16, dtype, page, seed=page + 1)


@pytest.mark.parametrize("heads", [16, 48, 128])
def test_heads(heads):
    _run([70, 3], [0, 66], heads, torch.float16, 32, seed=heads)


def test_long_prompt():
    _run([1500], [0], 16, torch.bfloat16, 64, seed=2)
    _run([300], [2200], 16, torch.float16, 0, seed=3)


def test_many_requests():
    rng = random.Random(4)
    queries = [rng.randint(0, 40) for _ in range(130)]
    _run(queries, [rng.randint(0, 30) for _ in queries], 16, torch.float16, 32, seed=4)


def test_requests_without_queries_or_keys():
    _run([0, 5, 0, 9], [20, 0, 0, 3], 16, torch.float16, 0, seed=5)


def test_more_queries_than_keys():
    # the first queries stand before the first key and see nothing
    gen = torch.Generator()
    gen.manual_seed(6)
    qn, qr, uk, uv = _inputs(gen, 150, 16, torch.float16)
    cache = torch.randn(10, 576, generator=gen).half().cuda()
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache, _cu([150]), _cu([10]))
    _check(got, qn, qr, uk, uv, lambda b: cache.double().cpu(), [150], [10], torch.float16, "early queries")
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache[:0], _cu([150]), _cu([0]))
    assert not got.any()


def test_rows_behind_the_last_request_are_zero():
    gen = torch.Generator()
    gen.manual_seed(7)
    for total in (130, 300):
        qn, qr, uk, uv = _inputs(gen, total, 16, torch.float16)
        cache = torch.randn(100, 576, generator=gen).half().cuda()
        cu = _cu([60, 40])
        out = torch.full((total, 16, 128), float("nan"), dtype=torch.float16, device="cuda")
        got = capi.prefill(qn, qr, uk, uv, cache, cu, cu, 100, out=out)
        assert torch.isfinite(got).all() and not got[100:].any()
        _check(got[:100], qn, qr, uk, uv, lambda b: cache[int(cu[b]):int(cu[b + 1])].double().cpu(), [60, 40], [60, 40],
               torch.float16, "padded")


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_key_that_is_not_finite_reaches_only_who_sees_it(value, dtype):
    gen = torch.Generator()
    gen.manual_seed(8)
    qn, qr, uk, uv = _inputs(gen, 200, 16, dtype)
    cache = torch.randn(200, 576, generator=gen).to(dtype).cuda()
    cu = _cu([200])
    want = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu)
    for t in (37, 64, 130):
        bad = cache.clone()
        bad[t, 9] = value
        got = ada_mla.mla_prefill(qn, qr, uk, uv, bad, cu, cu)
        assert torch.equal(got[:t], want[:t])
        assert torch.isnan(got[t:]).all()


def test_a_value_that_overflows_fp16():
    # finite keys whose values pass 65504: NaN for who sees them, nothing for the others
    gen = torch.Generator()
    gen.manual_seed(9)
    qn, qr, uk, uv = _inputs(gen, 100, 16, torch.float16)
    uk = torch.zeros_like(uk)
    cache = torch.randn(100, 576, generator=gen).half().cuda()
    cache[50, :512] = 60000.0 * (uv[3, 17].sign() + (uv[3, 17] == 0))
    cu = _cu([100])
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu)
    assert torch.isfinite(got[:50]).all() and torch.isnan(got[50:, 3]).all()


def test_workspace_of_nans():
    gen = torch.Generator()
    gen.manual_seed(10)
    lib = capi.load()
    ws = torch.full((lib.mla_prefill_workspace_size(4, 16, 231, 500),), 255, dtype=torch.uint8, device="cuda")
    for lengths in ([100, 3, 64, 65], [1, 1, 1, 1], [0, 200, 0, 31]):
        qn, qr, uk, uv = _inputs(gen, sum(lengths), 16, torch.float16)
        cache = torch.randn(sum(lengths), 576, generator=gen).half().cuda()
        cu = _cu(lengths)
        got = capi.prefill(qn, qr, uk, uv, cache, cu, cu, sum(lengths), workspace=ws)
        _check(got, qn, qr, uk, uv, lambda b: cache[int(cu[b]):int(cu[b + 1])].double().cpu(), lengths, lengths,
               torch.float16, f"{lengths}")


def test_captured_and_replayed():
    gen = torch.Generator()
    gen.manual_seed(11)
    qn, qr, uk, uv = _inputs(gen, 200, 16, torch.float16)
    cache = torch.randn(300, 576, generator=gen).half().cuda()
    cu_q, cu = _cu([150, 50]), _cu([150, 150])
    call = lambda: ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu_q, cu, total_tokens=300)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(4):
        qn.normal_()
        cache.normal_()
        cu_q[1:].sub_(10)
        want = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(out, want), r


def test_agrees_with_the_absorbed_form():
    # a prompt's last query, expanded, against the decode with the absorbed query and W_UV behind it
    gen = torch.Generator()
    gen.manual_seed(12)
    qn, qr, uk, uv = _inputs(gen, 90, 16, torch.float16)
    cache = torch.randn(90, 576, generator=gen).half().cuda()
    cu = _cu([90])
    expanded = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu)[-1].double().cpu()
    q = ada_mla.mla_absorb_query(qn[-1:].contiguous(), qr[-1:].contiguous(), uk)
    o = ada_mla.mla_decode_split(q[0], cache).double().cpu()
    absorbed = (uv.double().cpu() @ o[:, :, None])[:, :, 0]
    # norms: 2 u for the expanded form; the absorbed one rounds q*, p, its partials and o*: below 2 u again
    err = (expanded - absorbed).norm() / absorbed.norm()
    assert err <= 4 * half_step(torch.float16), err


def test_cache_rows_past_2_to_31_elements():
    gen = torch.Generator()
    gen.manual_seed(13)
    page, n = 64, 150
    pages = 2 ** 31 // (576 * page) + 6
    cache = torch.zeros(pages, page, 576, dtype=torch.bfloat16, device="cuda")
    ids = [pages - 1, 2, pages - 4]
    for i in ids:
        cache[i] = torch.randn(page, 576, generator=gen).bfloat16().cuda()
    qn, qr, uk, uv = _inputs(gen, n, 16, torch.bfloat16)
    cu = _cu([n])
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu, torch.tensor([ids], dtype=torch.int32, device="cuda"), n)
    rows = cache[ids].view(-1, 576)[:n].contiguous()
    assert torch.equal(got, ada_mla.mla_prefill(qn, qr, uk, uv, rows, cu, cu))
    _check(got, qn, qr, uk, uv, lambda b: rows.double().cpu(), [n], [n], torch.bfloat16, "far pages")


def test_page_ids_out_of_range_stay_inside_the_cache():
    gen = torch.Generator()
    gen.manual_seed(14)
    qn, qr, uk, uv = _inputs(gen, 100, 16, torch.float16)
    cache = torch.randn(4, 32, 576, generator=gen).half().cuda()
    cu = _cu([100])
    table = torch.tensor([[0, -9, 2 ** 31 - 1, 3]], dtype=torch.int32, device="cuda")
    got = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu, table, 100)
    same = ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu, cu, table.clamp(0, 3), 100)
    assert torch.equal(got, same)


def test_a_row_is_the_same_whatever_runs_beside_it():
    # a request's results do not depend on the others of the batch, nor on where its tiles begin
    gen = torch.Generator()
    gen.manual_seed(15)
    qn, qr, uk, uv = _inputs(gen, 300, 16, torch.float16)
    cache = torch.randn(300, 576, generator=gen).half().cuda()
    alone = ada_mla.mla_prefill(qn[90:], qr[90:], uk, uv, cache[90:], _cu([210]), _cu([210]))
    both = ada_mla.mla_prefill(qn, qr, uk, uv, cache, _cu([90, 210]), _cu([90, 210]))
    assert torch.equal(both[90:], alone)


def test_two_streams_at_once():
    gen = torch.Generator()
    gen.manual_seed(16)
    cases = []
    for n in (400, 700):
        qn, qr, uk, uv = _inputs(gen, n, 16, torch.bfloat16)
        cache, cu = torch.randn(n, 576, generator=gen).bfloat16().cuda(), _cu([n])
        cases.append((qn, qr, uk, uv, cache, cu, cu))
    want = [ada_mla.mla_prefill(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, stream in zip(cases * 2, streams * 2):
        with torch.cuda.stream(stream):
            got.append(ada_mla.mla_prefill(*c))
    torch.cuda.synchronize()
    for g, w in zip(got, want * 2):
        assert torch.equal(g, w)


def _partials(batch, heads, queries, total):
    """Whether a call splits its keys: its workspace then holds more than K, V, rotary parts and flags."""
    tiles = total // 64 + batch
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    plain = 2 * up(heads * tiles * 64 * 256) + up(tiles * 64 * 128) + up(heads * tiles * 32)
    return capi.load().mla_prefill_workspace_size(batch, heads, queries, total) > plain


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("queries,context,page,split", [
    ([1], [6000], 64, True), ([33], [4063], 0, True), ([200], [3900], 128, True), ([7, 3, 130], [11000, 12, 900], 32, True),
    ([7, 1, 0, 140, 3], [5000, 1, 900, 1337, 64], 32, False)])
def test_few_queries_behind_long_contexts(queries, context, page, split, dtype):
    # keys split over workgroups; a short request among long ones, tiles that end inside a split
    total = sum(queries) + sum(context)
    assert _partials(len(queries), 16, sum(queries), total) == split
    _run(queries, context, 16, dtype, page, seed=total)


def test_split_keys_padded_rows_and_values_that_are_not_finite():
    gen = torch.Generator()
    gen.manual_seed(17)
    n, m, rows = 5000, 40, 170
    assert _partials(1, 16, rows, n)
    qn, qr, uk, uv = _inputs(gen, rows, 16, torch.bfloat16)
    cache = torch.randn(n, 576, generator=gen).bfloat16().cuda()
    call = lambda: capi.prefill(qn, qr, uk, uv, cache, _cu([m]), _cu([n]), n,  # noqa: E731
                                out=torch.full((rows, 16, 128), float("nan"), dtype=torch.bfloat16, device="cuda"))
    want = call()
    assert torch.isfinite(want).all() and not want[m:].any()
    assert torch.equal(call(), want)
    cache[n - 20, 7] = float("inf")  # seen by the last 20 queries
    got = call()
    assert torch.equal(got[:20], want[:20]) and torch.isnan(got[20:m]).all() and not got[m:].any()
    cache[n - 20, 7] = 0
    cache[100, 3] = float("nan")  # seen by all
    got = call()
    assert torch.isnan(got[:m]).all() and not got[m:].any()


def test_split_keys_captured_and_replayed():
    gen = torch.Generator()
    gen.manual_seed(18)
    n = 9000
    qn, qr, uk, uv = _inputs(gen, 60, 16, torch.float16)
    cache = torch.randn(n, 576, generator=gen).half().cuda()
    cu_q, cu = _cu([10, 50]), _cu([500, n - 500])
    assert _partials(2, 16, 60, n)
    call = lambda: ada_mla.mla_prefill(qn, qr, uk, uv, cache, cu_q, cu, total_tokens=n)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(4):
        qn.normal_()
        cache.normal_()
        cu[1:2].add_(200)
        want = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(out, want), r


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("queries,context", [
    ([1], [0]), ([1], [64]), ([31], [33]), ([32], [31]), ([33], [224]), ([65], [192]), ([197], [0]), ([5, 0, 40], [700, 9, 3])])
def test_small_calls(queries, context, dtype):
    # 32 queries a workgroup whose waves take the key tiles in turn: from none of them to three each
    _run(queries, context, 16, dtype, 32, seed=sum(queries) + sum(context))


def test_many_requests_with_rows_behind_the_last():
    # enough query tiles to fill the chip by themselves
    gen = torch.Generator()
    gen.manual_seed(19)
    lengths = [70] * 40
    n, rows = sum(lengths), sum(lengths) + 150
    qn, qr, uk, uv = _inputs(gen, rows, 16, torch.float16)
    cache, cu = torch.randn(n, 576, generator=gen).half().cuda(), _cu(lengths)
    out = torch.full((rows, 16, 128), float("nan"), dtype=torch.float16, device="cuda")
    got = capi.prefill(qn, qr, uk, uv, cache, cu, cu, n, out=out)
    assert torch.isfinite(got).all() and not got[n:].any()
    _check(got[:n], qn, qr, uk, uv, lambda b: cache[int(cu[b]):int(cu[b + 1])].double().cpu(), lengths, lengths,
           torch.float16, "many, padded")
    cache[n - 30, 9] = float("nan")  # of the last request, seen by its last 30 queries
    bad = capi.prefill(qn, qr, uk, uv, cache, cu, cu, n)
    assert torch.equal(bad[:n - 30], got[:n - 30]) and torch.isnan(bad[n - 30:n]).all() and not bad[n:].any()
