"""mla_decode_paged over a paged cache of E4M3FN bytes, against softmax attention in float64.

Tolerance, element by element, with u half a step of the query's type (values are decoded exactly):
  out and the split partials rounded once each                 2 u max(|ref|, spread)
  p_t rounded where it is stored and where its half is scaled  2 u sum p |v| / l
  logits in fp32, as operators_reference.attention_check       2 g sum p |v| / l
  32- and 64-head tiles multiply Q* as two e4m3 parts: 2^-8 of a value and 2^-21 of the head's
  largest (the second part's smallest step is 2^-9 / 16 where that one stands at 128 .. 256): g +=
  2 scale sum (2^-8 |q| + 2^-21 max|q|) |k|
In the 2-norm the roundings are independent: four of u / sqrt(3) (out, partial, twice p) in quadrature are 1.16 u,
the parts of Q* change a logit by at most 2^-8 scale sqrt(sum q^2 k^2), 2^-8 sqrt(576 / 192) = 0.0068 for N(0, 1) values.
"""
import random

import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import SCALE, half_step

pytestmark = pytest.mark.gpu

NAN8 = 0x7F


def _case(seed, lengths, page, cache_scale):
    """E4M3FN pages of N(0, 1) / cache_scale, a shuffled table with wild ids behind each request's last page, NaN
    bytes wherever no request's token stands."""
    gen = torch.Generator()
    gen.manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = max(1, sum(need)) + 2
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    rows = torch.randn(pages, page, 576, generator=gen)
    cache = (rows / cache_scale).to(torch.float8_e4m3fn)
    width = max(need + [1]) + 2
    table, k, held = [], 0, []
    raw = cache.view(torch.uint8)
    for n, m in zip(lengths, need):
        ids = order[k:k + m]
        k += m
        if n % page:
            raw[ids[-1], n % page:] = NAN8
        table.append(ids + [pages + 1000003, -5] + [0] * (width - m - 2))
        held.append(cache[ids].double().reshape(-1, 576)[:n] * cache_scale)
    for p in order[k:]:
        raw[p] = NAN8
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return (cache.cuda(), torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda(),
            held, gen)


def _check(out, q, held, dtype, what=""):
    u, parts = half_step(dtype), q.shape[1] % 32 == 0  # 16-head tiles keep Q* whole: the bound below covers both
    err2 = ref2 = 0.0
    for b, c in enumerate(held):
        got = out[b].double().cpu()
        assert torch.isfinite(got).all(), f"{what}: request {b}"
        if c.shape[0] == 0:
            assert not got.any(), f"{what}: request {b} has no tokens"
            continue
        qb = q[b].double().cpu()
        s = qb @ c.T * SCALE
        p = torch.softmax(s, -1)
        v = c[:, :512]
        ref, spread = p @ v, p @ v.abs()
        reach = (qb.abs() @ c.abs().T).amax(1, keepdim=True) * SCALE
        g = 2 * (576 + 8) * 2.0 ** -24 * reach + 2.0 ** -18
        if parts:
            g = g + 2 * (2.0 ** -8 * reach + 2.0 ** -21 * qb.abs().amax(1, keepdim=True) * SCALE *
                         c.abs().sum(1).amax())
        bound = (4 * u + 2 * g) * (1 + g) * spread * 1.01
        if dtype == torch.float16:
            total = torch.exp(s - s.amax(1, keepdim=True)).sum(1, keepdim=True)
            bound = bound + 2 * c.shape[0] * 2.0 ** -25 * v.abs().amax() / total + 2.0 ** -24
        err = (got - ref).abs()
        worst = (err / bound).nan_to_num(0.0, posinf=float("inf")).max().item()  # 0 / 0: exactly 0, as it should be
        assert worst <= 1.0, f"{what}: request {b}: {worst:.2f} times its bound"
        err2 += (err ** 2).sum().item()
        ref2 += (ref ** 2).sum().item()
    if ref2:
        rel = (err2 / ref2) ** 0.5
        assert rel <= 1.5 * u + (0.0068 if parts else 0.0) + (2.0 ** -12 if dtype == torch.float16 else 0.0), (what, rel)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("page,lengths", [(32, [0, 1, 31, 32, 33, 0, 200]), (64, [129, 1, 64, 700]), (128, [1501]), (64, [1])])
def test_lengths_and_heads(dtype, heads, page, lengths):
    cache, table, cu, held, gen = _case(heads + page, lengths, page, 0.0625)
    q = torch.randn(len(lengths), heads, 576, generator=gen).to(dtype).cuda()
    out = ada_mla.mla_decode_paged(q, cache, table, cu, total_tokens=sum(lengths), cache_scale=0.0625)
    assert out.dtype == dtype and out.shape == (len(lengths), heads, 512)
    _check(out, q, held, dtype, f"{heads} heads")
    again = capi.decode_paged(q, cache, table, cu, sum(lengths), cache_scale=0.0625)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [16, 64])
def test_batches_without_a_token(dtype, heads):
    cache, table, cu, held, gen = _case(1, [0, 0, 0], 32, 1.0)
    q = torch.randn(3, heads, 576, generator=gen).to(dtype).cuda()
    for total in (0, 5):  # what the batch has, and an upper bound
        out = ada_mla.mla_decode_paged(q, cache, table, cu, total_tokens=total)
        assert (out == 0).all(), total


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("splits", [1, 3, 7, 64, 100000])
def test_forced_splits(dtype, splits):
    lengths = [300, 0, 1000, 5]
    cache, table, cu, held, gen = _case(splits, lengths, 32, 1.0)
    q = torch.randn(4, 64, 576, generator=gen).to(dtype).cuda()
    out = ada_mla.mla_decode_paged(q, cache, table, cu, total_tokens=sum(lengths), num_splits=splits)
    _check(out, q, held, dtype, f"{splits} splits")


@pytest.mark.parametrize("dtype,big", [(torch.bfloat16, 3.0e38), (torch.bfloat16, 1e-38), (torch.float16, 65504.0),
                                       (torch.float16, 2.0 ** -20)])
@pytest.mark.parametrize("heads", [16, 32, 64])
def test_queries_at_the_ends_of_their_range(dtype, big, heads):
    # two tokens, the first opposite to the query: whatever the query's size, the softmax picks the second, or,
    # where the query vanishes, takes both alike
    cache = torch.zeros(1, 32, 576)
    cache[0, 0], cache[0, 1] = -1.0, 1.0
    cache[0, 1, 7] = 0.5
    cache = cache.to(torch.float8_e4m3fn).cuda()
    q = torch.zeros(1, heads, 576, dtype=dtype)
    q[:, :, 3] = big
    out = ada_mla.mla_decode_paged(q.cuda(), cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                   torch.tensor([0, 2], dtype=torch.int32, device="cuda"), total_tokens=2)
    ref = cache[0, 1, :512].float().cpu() if big > 1 else cache[0, :2, :512].float().mean(0).cpu()
    assert (out.float().cpu() - ref).abs().max() <= 4 * half_step(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [16, 64])
def test_nan_and_infinite_queries_stay_in_their_heads(dtype, heads):
    lengths = [70, 40]
    cache, table, cu, held, gen = _case(5, lengths, 32, 0.5)
    q = torch.randn(2, heads, 576, generator=gen).to(dtype)
    clean = ada_mla.mla_decode_paged(q.cuda(), cache, table, cu, total_tokens=110, cache_scale=0.5)
    q[0, 3, 100] = float("nan")
    q[1, 5, 570] = float("inf")
    out = ada_mla.mla_decode_paged(q.cuda(), cache, table, cu, total_tokens=110, cache_scale=0.5)
    assert out[0, 3].isnan().all() and out[1, 5].isnan().all()
    out[0, 3], out[1, 5] = clean[0, 3], clean[1, 5]
    assert torch.equal(out, clean)


def test_reads_what_append_writes():
    gen = torch.Generator()
    gen.manual_seed(2)
    n, heads = 77, 32
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = torch.zeros(4, 32, 576, dtype=torch.float8_e4m3fn, device="cuda")
    table = torch.tensor([[2, 0, 3]], **i32)
    pos = torch.arange(n, **i32)
    slots = table[0, pos.long() // 32].long() * 32 + pos.long() % 32
    kv = torch.randn(n, 576, generator=gen).bfloat16().cuda()
    angle = torch.arange(128.0)[:, None] * 10000.0 ** (-torch.arange(32) / 32)
    ada_mla.mla_append_kv(kv, torch.ones(512, dtype=torch.bfloat16, device="cuda"),
                          torch.cat([angle.cos(), angle.sin()], 1).cuda(), pos, slots, cache, cache_scale=0.03125)
    q = torch.randn(1, heads, 576, generator=gen).bfloat16().cuda()
    out = ada_mla.mla_decode_paged(q, cache, table, torch.tensor([0, n], **i32), cache_scale=0.03125)
    held = [cache.view(-1, 576)[slots].double().cpu() * 0.03125]
    _check(out, q, held, torch.bfloat16)


def test_replays_of_a_captured_call():
    lengths = [500, 3, 90]
    cache, table, cu, held, gen = _case(9, lengths, 64, 0.0625)
    q = torch.randn(3, 64, 576, generator=gen).bfloat16().cuda()
    call = lambda: ada_mla.mla_decode_paged(q, cache, table, cu, total_tokens=593, cache_scale=0.0625)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        graph.replay()
        assert torch.equal(out, call()), k
        _check(out, q, held, torch.bfloat16)


def test_rows_past_2_31_bytes():
    pages, page = 60000, 64  # 2.2 GB: the last pages' bytes lie past 2^31
    cache = torch.zeros(pages, page, 576, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    gen = torch.Generator()
    gen.manual_seed(4)
    rows = torch.randn(2, page, 576, generator=gen).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[pages - 2:] = rows.view(torch.uint8).cuda()
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    for dtype in (torch.float16, torch.bfloat16):
        for heads in (16, 64):
            q = torch.randn(1, heads, 576, generator=gen).to(dtype).cuda()
            out = ada_mla.mla_decode_paged(q, cache, table, torch.tensor([0, 101], dtype=torch.int32, device="cuda"),
                                           total_tokens=101)
            _check(out, q, [torch.cat([rows[1], rows[0]]).double()[:101]], dtype)
