"""Latent rows into the cache and rotated queries (mla_append_kv) against
float64.

A row's values pass one rounding to their type: u |ref|. In fp32 before it:
the sum of 512 squares (each addition off by 2^-24: 2^-15 at most, halved by
the root), the root, a division and two products; a rotation is two products
and a difference, off by 2^-23 (|x| + |y|). So |error| <= u |ref| + 2^-14
|ref| for latents and u |ref| + 2^-22 (|x| + |y|) for rotated values; fp8 (u =
2^-4, below 2^-6 steps of 2^-9) in units of cache_scale.
"""
import pytest
import torch

import ada_mla
from operators_reference import half_step, latent_rows, rotate

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _inputs(tokens, heads, dtype, positions=5000, seed=0):
    gen = torch.Generator()
    gen.manual_seed(seed)
    kv = (1.5 * torch.randn(tokens, 576, generator=gen)).to(dtype)
    w = (1 + 0.3 * torch.randn(512, generator=gen)).to(dtype)
    q = torch.randn(tokens, max(heads, 1), 64, generator=gen).to(dtype)
    i = torch.arange(32, dtype=torch.float64)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-i / 32)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float()
    pos = torch.randint(0, positions, (tokens,), generator=gen, dtype=torch.int32)
    return kv, w, cs, pos, (q if heads else None)


def _rounded(dtype):
    """(relative half step, absolute half step where the type is subnormal)"""
    if dtype == torch.float8_e4m3fn:
        return 2.0 ** -4, 2.0 ** -10
    return half_step(dtype), 2.0 ** -25 if dtype == torch.float16 else 0.0


def _check_rows(got, ref, raw_rope, dtype, scale=1.0):
    u, tiny = _rounded(dtype)
    got, ref = got.double() * scale, ref
    lat = (got[:, :512] - ref[:, :512]).abs() - (ref[:, :512].abs() * (u + 2.0 ** -14) + tiny * scale)
    assert (lat <= 0).all(), f"latents: {lat.max()} past their bound"
    reach = raw_rope.double().abs().amax(1, keepdim=True) * 2
    rope = (got[:, 512:] - ref[:, 512:]).abs() - (ref[:, 512:].abs() * u + 2.0 ** -22 * (1 + u) * reach + tiny * scale)
    assert (rope <= 0).all(), f"rotary part: {rope.max()} past its bound"


def _run(kv, w, cs, pos, slots, cache, q, **kw):
    d = [t.cuda() if t is not None else None for t in (kv, w, cs, pos, slots)]
    out = ada_mla.mla_append_kv(*d, cache, q_rope=None if q is None else q.cuda(), eps=EPS, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads", [(1, 128), (3, 0), (65, 16), (257, 5), (30, 33)])
def test_rows_and_queries(dtype, fp8, interleaved, tokens, heads):
    kv, w, cs, pos, q = _inputs(tokens, heads, dtype, seed=tokens + heads)
    page, pages = 32, tokens // 32 + 3
    slots = torch.randperm(page * pages)[:tokens]
    scale = 0.03125 if fp8 else 1.0
    before = torch.randn(pages, page, 576).to(torch.float8_e4m3fn if fp8 else dtype)
    cache = before.cuda()
    out = _run(kv, w, cs, pos, slots, cache, q, cache_scale=scale, interleaved=interleaved)
    after = cache.cpu().float().view(-1, 576)
    angle = cs[pos.long()].double()
    ref = latent_rows(kv, w, angle[:, :32], angle[:, 32:], EPS, interleaved)
    _check_rows(after[slots], ref, kv[:, 512:], torch.float8_e4m3fn if fp8 else dtype, scale)
    others = torch.ones(page * pages, dtype=torch.bool)
    others[slots] = False
    assert torch.equal(after[others], before.float().view(-1, 576)[others])
    if heads == 0:
        assert out is None
        return
    want = rotate(q.double(), angle[:, None, :32], angle[:, None, 32:], interleaved)
    u, tiny = _rounded(dtype)
    bound = want.abs() * u + 2.0 ** -22 * (1 + u) * 2 * q.double().abs().amax(2, keepdim=True) + tiny
    assert out.shape == q.shape and ((out.cpu().double() - want).abs() <= bound).all()


def test_rows_without_a_slot_are_not_written():
    kv, w, cs, pos, q = _inputs(40, 16, torch.float16, seed=3)
    cache = torch.zeros(64, 576, dtype=torch.float16, device="cuda")
    slots = torch.arange(40)
    slots[::3] = -1
    slots[1] = 64          # just past the cache
    slots[4] = 2 ** 40     # far past it
    slots[7] = -2 ** 40
    out = _run(kv, w, cs, pos, slots, cache, q)
    written = cache.cpu().abs().sum(1) > 0
    keep = torch.zeros(64, dtype=torch.bool)
    keep[slots[(slots >= 0) & (slots < 64)]] = True
    assert torch.equal(written, keep)
    assert torch.isfinite(out).all()  # queries are rotated all the same


def test_positions_are_clamped_to_the_table():
    kv, w, cs, _, q = _inputs(4, 16, torch.float16, positions=10, seed=4)
    pos = torch.tensor([-5, 0, 9, 2 ** 31 - 1], dtype=torch.int32)
    a, b = (torch.zeros(4, 576, dtype=torch.float16, device="cuda") for _ in range(2))
    out = _run(kv, w, cs, pos, torch.arange(4), a, q)
    same = _run(kv, w, cs, pos.clamp(0, 9), torch.arange(4), b, q)
    assert torch.equal(out, same) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strided_rows_are_read_in_place_or_copied(dtype):
    kv, w, cs, pos, q = _inputs(21, 16, dtype, seed=5)
    dense = torch.zeros(32, 576, dtype=dtype, device="cuda")
    want = _run(kv, w, cs, pos, torch.arange(21), dense, q)
    # slices of wider projections: strides of 16 bytes, and odd ones (copied by the call)
    for extra, first in ((1536, 0), (1536, 8), (3, 1)):
        wide = torch.full((21, 576 + extra + first), 7.0, dtype=dtype, device="cuda")
        wide[:, first:first + 576] = kv.cuda()
        q_wide = torch.full((21, 16, 64 + 128 + first), 7.0, dtype=dtype, device="cuda")
        q_wide[:, :, first:first + 64] = q.cuda()
        cache = torch.zeros_like(dense)
        got = ada_mla.mla_append_kv(wide[:, first:first + 576], w.cuda(), cs.cuda(), pos.cuda(), torch.arange(21).cuda(),
                                    cache, q_rope=q_wide[:, :, first:first + 64], eps=EPS)
        assert torch.equal(got, want) and torch.equal(cache, dense), (extra, first)
    # heads in another order than the tokens
    turned = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    got = ada_mla.mla_append_kv(kv.cuda(), w.cuda(), cs.cuda(), pos.cuda(), torch.arange(21).cuda(), cache, q_rope=turned,
                                eps=EPS)
    assert torch.equal(got, want)


def test_one_token_as_a_row_of_a_wider_tensor():
    kv, w, cs, pos, q = _inputs(1, 1, torch.float16, seed=6)
    a, b = (torch.zeros(4, 576, dtype=torch.float16, device="cuda") for _ in range(2))
    want = _run(kv, w, cs, pos, torch.tensor([2]), a, q)
    got = ada_mla.mla_append_kv(kv.cuda().expand(1, 576).as_strided((1, 576), (3, 1)), w.cuda(), cs.cuda(), pos.cuda(),
                                torch.tensor([2]).cuda(), b, q_rope=q.cuda().as_strided((1, 1, 64), (5, 7, 1)), eps=EPS)
    assert torch.equal(got, want) and torch.equal(a, b)


def test_values_out_of_the_ordinary():
    # rows of zeros, of the type's largest values, with an infinity and with a NaN
    kv, w, cs, pos, _ = _inputs(5, 0, torch.float16, seed=7)
    kv[0] = 0
    kv[1, :512] = 65504.0
    kv[2, 3] = float("inf")
    kv[3, 4] = float("nan")
    for fp8 in (False, True):
        cache = torch.zeros(8, 576, dtype=torch.float8_e4m3fn if fp8 else torch.float16, device="cuda")
        _run(kv, w, cs, pos, torch.arange(5), cache, None, cache_scale=0.001 if fp8 else 1.0)
        got = cache.cpu().float()
        assert not got[0].any()
        if fp8:  # saturated, never an overflow to NaN
            assert (got[1, :512].abs() == 448).all() or (got[1, :512].abs() <= 448).all()
            assert torch.isfinite(got[1]).all()
        else:
            ref = latent_rows(kv, w, cs[pos.long()][:, :32].double(), cs[pos.long()][:, 32:].double(), EPS, True)
            _check_rows(got[1:2], ref[1:2], kv[1:2, 512:], torch.float16)
        assert torch.isnan(got[2, 3]) and torch.isnan(got[3]).sum() == 512
        assert torch.isfinite(got[4]).all()


def test_no_tokens():
    kv, w, cs, pos, q = _inputs(2, 16, torch.float16)
    cache = torch.ones(4, 576, dtype=torch.float16, device="cuda")
    out = _run(kv[:0], w, cs, pos[:0], torch.arange(0), cache, q[:0])
    assert out.shape == (0, 16, 64) and (cache == 1).all()


def test_slots_past_2_to_31_elements():
    kv, w, cs, pos, _ = _inputs(2, 0, torch.bfloat16, seed=8)
    rows = 2 ** 31 // 576 + 70
    cache = torch.zeros(rows, 576, dtype=torch.bfloat16, device="cuda")
    _run(kv, w, cs, pos, torch.tensor([rows - 1, 0]), cache, None)
    angle = cs[pos.long()].double()
    ref = latent_rows(kv, w, angle[:, :32], angle[:, 32:], EPS, True)
    _check_rows(torch.stack([cache[rows - 1], cache[0]]).cpu().float(), ref, kv[:, 512:], torch.bfloat16)
    assert cache[1:rows - 1].abs().max().item() == 0


def test_captured_on_another_stream():
    kv, w, cs, pos, q = [t.cuda() for t in _inputs(33, 16, torch.float16, seed=9)]
    slots = torch.arange(33, device="cuda")
    cache = torch.zeros(64, 576, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ada_mla.mla_append_kv(kv, w, cs, pos, slots, cache, q_rope=q)
    for r in range(3):
        kv.normal_()
        q.normal_()
        slots.copy_(torch.randperm(64, device="cuda")[:33])
        cache.zero_()
        eager = torch.zeros_like(cache)
        want = ada_mla.mla_append_kv(kv, w, cs, pos, slots, eager, q_rope=q)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache, eager), r
