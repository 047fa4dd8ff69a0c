"""The operators around the decode at the bounds of their types and buffers: rows whose
squares pass fp32's range, keys whose expansion passes fp16's, saturated fp8 rows,
inputs that begin off 16 bytes, workspaces of exactly the size that is asked for.
Tolerances: test_gpu_append_kv.py and operators_reference."""
import random

import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import attention_check, gather_paged, half_step, latent_rows, paged_case, random_tree, signed

pytestmark = pytest.mark.gpu


def _angles(positions=64):
    i = torch.arange(32, dtype=torch.float64)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-i / 32)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _rows(kv, w, eps, interleaved=True, fp8_scale=None):
    """kv's rows appended to an empty cache, and the same in float64."""
    n = kv.shape[0]
    cs, pos = _angles(), torch.arange(n, dtype=torch.int32)
    cache = torch.zeros(n, 576, dtype=kv.dtype if fp8_scale is None else torch.float8_e4m3fn, device="cuda")
    ada_mla.mla_append_kv(kv.cuda(), w.cuda(), cs.cuda(), pos.cuda(), torch.arange(n).cuda(), cache, eps=eps,
                          cache_scale=1.0 if fp8_scale is None else fp8_scale, interleaved=interleaved)
    angle = cs[:n].double()
    return cache.cpu().double(), latent_rows(kv, w, angle[:, :32], angle[:, 32:], eps, interleaved)


@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("largest", [2.0 ** 62, 2.0 ** 100, 2.0 ** 126])
def test_rows_whose_squares_pass_fp32(largest, eps):
    # bf16 reaches 2^128: the mean of the squares is past fp32's range, the normalised row is an ordinary one
    gen = torch.Generator()
    gen.manual_seed(1)
    kv = torch.randn(6, 576, generator=gen)
    kv[:, :512] *= largest / 4
    kv[1, 7:512] = 0        # one value alone
    kv[2, :256] *= 2.0 ** -40
    kv[3, :512] = largest * 1.5
    kv = kv.bfloat16()
    assert torch.isfinite(kv).all()
    w = (1 + 0.3 * torch.randn(512, generator=gen)).bfloat16()
    got, ref = _rows(kv, w, eps)
    bound = ref[:, :512].abs() * (half_step(torch.bfloat16) + 2.0 ** -14)
    assert ((got[:, :512] - ref[:, :512]).abs() <= bound).all()


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -75, 2.0 ** -120])
def test_rows_whose_squares_vanish_in_fp32(scale):
    # without an epsilon a row of tiny values is normalised like any other
    gen = torch.Generator()
    gen.manual_seed(2)
    kv = torch.randn(4, 576, generator=gen)
    kv[:, :512] *= scale
    kv = kv.bfloat16()
    w = (1 + 0.3 * torch.randn(512, generator=gen)).bfloat16()
    got, ref = _rows(kv, w, 0.0)
    bound = ref[:, :512].abs() * (half_step(torch.bfloat16) + 2.0 ** -14)
    assert ((got[:, :512] - ref[:, :512]).abs() <= bound).all()
    # with one they stay tiny: the epsilon is all there is under the root
    got, ref = _rows(kv, w, 1e-6)
    bound = ref[:, :512].abs() * (half_step(torch.bfloat16) + 2.0 ** -14) + 2.0 ** -134  # half a step of subnormals
    assert ((got[:, :512] - ref[:, :512]).abs() <= bound).all()


def test_rows_with_infinities_among_large_values():
    kv = torch.full((3, 576), 2.0 ** 100)
    kv[0, 5], kv[1, 6] = float("inf"), float("nan")
    got, _ = _rows(kv.bfloat16(), torch.ones(512).bfloat16(), 1e-6)
    assert torch.isnan(got[0, 5]) and not got[0, :5].any() and not got[0, 6:512].any()
    assert torch.isnan(got[1, :512]).all()
    assert (got[2, :512] == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_fp8_rows_saturate_at_448(dtype, interleaved):
    # every value past 448 scales is 448 of its sign, every other one within half a step of E4M3
    gen = torch.Generator()
    gen.manual_seed(3)
    kv = torch.randn(9, 576, generator=gen)
    kv[:, 512:] *= 3
    w = 1 + 0.3 * torch.randn(512, generator=gen)
    kv, w, scale = kv.to(dtype), w.to(dtype), 2.0 ** -8  # 448 scales are 1.75
    got, ref = _rows(kv, w, 1e-6, interleaved, scale)
    want = ref / scale
    # fp32 before the rounding: 2^-14 |ref| for latents, 2^-22 of the rotated pair's values
    slack = want.abs() * 2.0 ** -14
    slack[:, 512:] += 2.0 ** -21 * kv[:, 512:].double().abs().amax(1, keepdim=True) / scale
    past = want.abs() - slack > 448
    for part in (slice(0, 512), slice(512, 576)):
        for sign in (1.0, -1.0):
            assert (past[:, part] & (want[:, part].sign() == sign)).sum() >= 10
    assert torch.equal(got[past], 448 * want[past].sign())
    inside = want.clamp(-448, 448)
    bound = inside.abs() * 2.0 ** -4 + 2.0 ** -10 + slack * (1 + 2.0 ** -4)
    assert ((got - inside).abs() <= bound).all()


@pytest.mark.parametrize("queries", [100, 1500])
def test_a_key_that_overflows_fp16(queries):
    # A finite latent row whose key passes 65504 in one value. Its logit is large and positive; as an
    # infinity times a negative query value it would be -inf, and the key would silently count for nothing.
    gen = torch.Generator()
    gen.manual_seed(4)
    heads, t, h = 16, 50, 3
    qn = torch.randn(queries, heads, 128, generator=gen).half()
    qr = torch.randn(queries, heads, 64, generator=gen).half()
    uk, uv = ((torch.randn(heads, 128, 512, generator=gen) * 512 ** -0.5).half() for _ in range(2))
    cache = torch.randn(queries, 576, generator=gen).half()
    uk[h] = 0
    uk[h, 17], uk[h, 18] = 2.0, 0.5
    qn[:, h] = 0
    qn[:, h, 17], qn[:, h, 18] = -0.01, 1.0
    cu = torch.tensor([0, queries], dtype=torch.int32, device="cuda")
    args = [x.cuda() for x in (qn, qr, uk, uv)]
    want = ada_mla.mla_prefill(*args, cache.cuda(), cu, cu)
    cache[t, :512] = 128.0
    k = cache[t, :512].double() @ uk[h].double().T
    assert k[17] > 65504 and k[18] < 65504 and qn[0, h].double() @ k > 1000
    got = ada_mla.mla_prefill(*args, cache.cuda(), cu, cu)
    assert torch.equal(got[:t], want[:t])
    assert torch.isnan(got[t:, h]).all()
    others = [i for i in range(heads) if i != h]
    assert torch.isfinite(got[:, others]).all()


def _off(t, by=1):
    """The same values, contiguous, `by` entries into another buffer."""
    flat = torch.full((t.numel() + by,), 7.0, dtype=t.dtype, device="cuda")
    flat[by:] = t.flatten().cuda()
    view = flat[by:].view(t.shape)
    assert view.is_contiguous() and view.data_ptr() % 16 != 0
    return view


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_inputs_that_begin_off_16_bytes(dtype):
    gen = torch.Generator()
    gen.manual_seed(5)
    kv, q = torch.randn(21, 576, generator=gen).to(dtype), torch.randn(21, 16, 64, generator=gen).to(dtype)
    w, cs = (1 + 0.3 * torch.randn(512, generator=gen)).to(dtype), _angles()
    pos, slots = torch.arange(21, dtype=torch.int32).cuda(), torch.arange(21).cuda()

    def call(kv, w, cs, q):
        cache = torch.zeros(32, 576, dtype=dtype, device="cuda")
        return ada_mla.mla_append_kv(kv, w, cs, pos, slots, cache, q_rope=q), cache
    good = [kv.cuda(), w.cuda(), cs.cuda(), q.cuda()]
    want = call(*good)
    for i in range(4):
        got = call(*[_off(x) if i == k else x for k, x in enumerate(good)])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tree_inputs_that_begin_off_16_bytes(dtype):
    gen = torch.Generator()
    gen.manual_seed(6)
    cache, table, cu = paged_case(gen, random.Random(6), [100, 33], 32, dtype)
    q = torch.randn(2, 3, 16, 576, generator=gen).to(dtype).cuda()
    mask = torch.tensor([[1, 3, 5]] * 2, dtype=torch.int64, device="cuda")
    want = ada_mla.mla_decode_tree(q, cache, table, cu, mask)
    assert torch.equal(ada_mla.mla_decode_tree(_off(q), cache, table, cu, mask), want)
    assert torch.equal(ada_mla.mla_decode_tree(q, _off(cache), table, cu, mask), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("paged", [False, True])
def test_prefill_inputs_that_begin_off_16_bytes(dtype, paged):
    gen = torch.Generator()
    gen.manual_seed(7)
    qn, qr = torch.randn(70, 16, 128, generator=gen).to(dtype), torch.randn(70, 16, 64, generator=gen).to(dtype)
    uk, uv = ((torch.randn(16, 128, 512, generator=gen) * 512 ** -0.5).to(dtype) for _ in range(2))
    cache, table, cu = paged_case(gen, random.Random(7), [50, 20], 32, dtype)
    if not paged:
        cache, table = torch.randn(70, 576, generator=gen).to(dtype).cuda(), None
    good = [qn.cuda(), qr.cuda(), uk.cuda(), uv.cuda(), cache]
    want = ada_mla.mla_prefill(*good, cu, cu, table)
    for i in range(5):
        got = ada_mla.mla_prefill(*[_off(x) if i == k else x for k, x in enumerate(good)], cu, cu, table)
        assert torch.equal(got, want), i


@pytest.mark.parametrize("heads,m,lengths,splits", [
    # rows that fill the chip, most requests far below a split's tokens and a few past it
    (64, 16, [5, 30, 1025, 16, 700, 2049, 40, 1, 0, 1024] + [20 + i for i in range(30)], 0),
    # the same lengths in every request, and splits that one request asks for among short ones
    (16, 4, [300] * 7, 4), (16, 4, [4] * 20 + [900] + [4] * 20, 5),
    # no request can be split
    (128, 8, [7, 90, 13] * 20, 0)])
def test_tree_workspace_of_exactly_its_size(heads, m, lengths, splits):
    rng, gen = random.Random(8), torch.Generator()
    gen.manual_seed(8)
    dtype = torch.bfloat16
    cache, table, cu = paged_case(gen, rng, lengths, 32, dtype)
    q = torch.randn(len(lengths), m, heads, 576, generator=gen).to(dtype).cuda()
    masks = [random_tree(rng, m) for _ in lengths]
    mask = torch.tensor([signed(x) for x in masks], dtype=torch.int64, device="cuda")
    drafts = [min(m, n) for n in lengths]
    size = capi.load().mla_decode_tree_workspace_size(len(lengths), m, heads, sum(lengths), splits)
    room = torch.full((size + 4096,), 255, dtype=torch.uint8, device="cuda")
    got = capi.decode_tree(q, cache, table, cu, mask, sum(lengths), draft_lens=torch.tensor(drafts, dtype=torch.int32).cuda(),
                           num_splits=splits, workspace=room[:size]).cpu()
    assert (room[size:] == 255).all()
    for b, (n, k) in enumerate(zip(lengths, drafts)):
        c = gather_paged(cache, table[b], n)
        for i in range(m):
            seen = torch.zeros(1, n, dtype=torch.bool)
            if i < k:
                seen[0, :n - k] = True
                for j in range(k):
                    seen[0, n - k + j] = bool(masks[b][i] >> j & 1)
            attention_check(got[b, i], q[b, i].double().cpu(), c, c[:, :512], seen.expand(heads, n), dtype,
                            what=f"request {b} draft {i}")
