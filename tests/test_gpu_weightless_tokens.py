"""Decodes where the running maximum has nothing to start from: queries that hold a NaN (their heads are NaN, whichever
form of the call, and no other head), and tokens whose logit is -inf, which have no weight wherever
they stand: whole first blocks, whole splits. Softmax attention in float64 without those tokens is the reference.

Tolerance, u half a step of the type, as for the other decodes: out and the partials 2 u, P and its scaling 2 u, of
sum p |v| / l; logits in fp32, 2 g of it with g = 2 (576 + 8) 2^-24 scale sum |q| |k| + 2^-18 (operators_reference); in fp16
also P below its normal range, n 2^-25 max|v| / L, and out below it, 2^-24.
"""
import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import SCALE, half_step

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
F8 = torch.float8_e4m3fn
ROPE = 540  # a column that is in the logits and not in the values


def _gen(seed):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return gen


def _only(got, clean, at, what):
    assert got[at].isnan().all(), what
    rest = got.clone()
    rest[at] = clean[at]
    if got.dtype == torch.float32:  # a NaN sends the other heads of its workgroup through another sum: the last bits
        assert torch.allclose(rest, clean, rtol=1e-5, atol=1e-5), what
    else:
        assert torch.equal(rest, clean), what


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, F8])
@pytest.mark.parametrize("heads", [16, 32, 64])
@pytest.mark.parametrize("n", [1, 40, 700])
def test_nan_queries_one_sequence(dtype, heads, n):
    gen = _gen(heads + n)
    c = torch.randn(n, 576, generator=gen).to(dtype).cuda()
    q = torch.randn(heads, 576, generator=gen).to(torch.float16 if dtype == F8 else dtype)
    bad = q.clone()
    bad[3, 100], bad[heads - 1, ROPE] = float("nan"), float("nan")
    for splits in (0, 1, 3):
        clean, got = (ada_mla.mla_decode_split(x.cuda(), c, num_splits=splits) for x in (q, bad))
        _only(got, clean, [3, heads - 1], f"{splits} splits")
    if dtype == torch.float16:
        clean, got = (capi.decode_split_fp16(x.cuda(), c, 3, capi.FLAG_FP32_PARTIALS) for x in (q, bad))
        _only(got, clean, [3, heads - 1], "fp32 partials")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [16, 32, 64])
def test_nan_queries_of_batches(dtype, heads):
    gen = _gen(heads)
    cu = torch.tensor([0, 70, 70, 400], **I32)
    c = torch.randn(400, 576, generator=gen)
    q = torch.randn(3, heads, 576, generator=gen).to(dtype)
    bad = q.clone()
    bad[2, 5, 7], bad[0, 0, 575] = float("nan"), float("nan")
    pages = torch.randn(20, 32, 576, generator=gen)
    table = torch.arange(60, **I32).view(3, 20) % 20
    for splits in (0, 1, 5):
        calls = {
            "batched": lambda x: ada_mla.mla_decode_split_batched(x, c.to(dtype).cuda(), cu, num_splits=splits),
            "paged": lambda x: ada_mla.mla_decode_paged(x, pages.to(dtype).cuda(), table, cu, num_splits=splits),
            "paged fp8": lambda x: ada_mla.mla_decode_paged(x, pages.to(F8).cuda(), table, cu, num_splits=splits),
        }
        if dtype == torch.float16:
            calls["batched fp8"] = lambda x: ada_mla.mla_decode_split_batched(x, c.to(F8).cuda(), cu, num_splits=splits)
        for name, call in calls.items():
            clean, got = call(q.cuda()), call(bad.cuda())
            assert (got[1] == 0).all()  # no tokens
            assert got[2, 5].isnan().all() and got[0, 0].isnan().all(), name
            got[2, 5], got[0, 0] = clean[2, 5], clean[0, 0]
            assert torch.equal(got, clean), (name, splits)


def _check(got, q, c, gone, dtype, what):
    """got [heads, 512] against attention over the tokens of c that are not gone (float64)."""
    u, k = half_step(dtype), c[~gone].double()
    qd, v = q.double(), k[:, :512]
    s = qd @ k.T * SCALE
    p = torch.softmax(s, -1)
    reach = (qd.abs() @ k.abs().T).amax(1, keepdim=True) * SCALE
    g = 2 * (576 + 8) * 2.0 ** -24 * reach + 2.0 ** -18
    bound = (4 * u + 2 * g) * (1 + g) * (p @ v.abs()) * 1.01
    if dtype == torch.float16:
        total = torch.exp(s - s.amax(1, keepdim=True)).sum(1, keepdim=True)
        bound = bound + 2 * len(c) * 2.0 ** -25 * v.abs().amax() / total + 2.0 ** -24
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    worst = ((got - p @ v).abs() / bound).nan_to_num(0.0, posinf=float("inf")).max().item()  # 0 / 0: exactly 0, as it should be
    assert worst <= 1.0, (what, worst)


# which of 300 tokens have no weight: the first block of 32 and some of the next, all of the first split of
# three, all but the last token, the last split, every second block
GONE = {"first": lambda t: t < 50, "first split": lambda t: t < 150, "all but one": lambda t: t < 299, "last": lambda t: t >= 130,
        "blocks": lambda t: t // 32 % 2 == 0}


@pytest.mark.parametrize("gone", GONE)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [16, 32, 64])
def test_tokens_of_no_weight(dtype, heads, gone):
    gen, n = _gen(heads), 300
    out = GONE[gone](torch.arange(n))
    c = torch.randn(n, 576, generator=gen).to(dtype)
    q = torch.randn(heads, 576, generator=gen).to(dtype)
    q[:, ROPE] = -q[:, ROPE].abs() - 0.5
    c[out, ROPE] = float("inf")
    for splits in (0, 1, 3):
        _check(ada_mla.mla_decode_split(q.cuda(), c.cuda(), num_splits=splits), q, c, out, dtype, f"{splits} splits")
    if dtype == torch.float32:
        return
    if dtype == torch.float16:
        _check(capi.decode_split_fp16(q.cuda(), c.cuda(), 3, capi.FLAG_FP32_PARTIALS), q, c, out, dtype, "fp32 partials")
    # the same tokens behind another sequence's, packed and on pages
    cu = torch.tensor([0, 45, 45 + n], **I32)
    packed = torch.cat([torch.randn(45, 576, generator=gen).to(dtype), c])
    pages = torch.zeros(12, 32, 576, dtype=dtype)
    pages[:2].view(-1, 576)[:45] = packed[:45]
    pages[2:].view(-1, 576)[:n] = c
    table = torch.tensor([[0, 1] + [0] * 8, list(range(2, 12))], **I32)
    both = torch.stack([q, q])
    none = torch.zeros(45, dtype=torch.bool)
    for splits in (0, 1, 4):
        for name, y in (("batched", ada_mla.mla_decode_split_batched(both.cuda(), packed.cuda(), cu, num_splits=splits)),
                        ("paged", ada_mla.mla_decode_paged(both.cuda(), pages.cuda(), table, cu, num_splits=splits))):
            _check(y[0], q, packed[:45], none, dtype, (name, splits, "the other"))
            _check(y[1], q, c, out, dtype, (name, splits))


@pytest.mark.parametrize("heads", [16, 32, 64])
@pytest.mark.parametrize("gone", GONE)
def test_logits_past_the_range_over_an_fp8_cache(heads, gone):
    # a bf16 query so large that its logits are -inf where the cache does not hold 0: the others share the weight
    gen, n = _gen(heads), 300
    out = GONE[gone](torch.arange(n))
    c = torch.randn(n, 576, generator=gen).to(F8)
    raw = c.float()
    raw[:, ROPE] = torch.where(out, 448.0, 0.0)
    q = torch.zeros(heads, 576, dtype=torch.bfloat16)
    q[:, ROPE] = -3.0e38
    pages = torch.zeros(10, 32, 576)
    pages.view(-1, 576)[:n] = raw
    for splits in (0, 1, 3):
        y = ada_mla.mla_decode_paged(q[None].cuda(), pages.to(F8).cuda(), torch.arange(10, **I32)[None], torch.tensor([0, n], **I32),
                                     num_splits=splits)
        _check(y[0], torch.zeros_like(q), raw, out, torch.bfloat16, splits)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_no_token_of_any_weight(dtype):
    # 0 / 0, whichever way the sequence is split
    gen = _gen(1)
    c = torch.randn(100, 576, generator=gen).to(dtype)
    q = torch.randn(16, 576, generator=gen).to(dtype)
    q[:, ROPE], c[:, ROPE] = -1.0, float("inf")
    for splits in (0, 1, 3):
        assert ada_mla.mla_decode_split(q.cuda(), c.cuda(), num_splits=splits).isnan().all(), splits
