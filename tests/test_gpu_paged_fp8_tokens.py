"""mla_decode_paged over an fp8 cache: every token of every request reaches its heads, with each head tile; errors request
by request (paged_fp8_reference)."""
import pytest
import torch

import ada_mla
from paged_fp8_reference import needle_worst, needles, norm_bound, norm_error
from test_gpu_paged_fp8 import _case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
CASES = [(32, [0, 1, 31, 32, 33, 2, 200]), (64, [129, 1, 64, 700]), (32, [300, 0, 1000, 5]), (128, [1501]), (64, [4097, 63])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("page,lengths", CASES)
def test_every_token_is_found(dtype, heads, page, lengths):
    cache, table, cu, held, _ = _case(heads + page, lengths, page, 0.0625)
    held = [c.cuda() for c in held]
    for i in range(-(-max(lengths) // heads)):
        q = torch.zeros(len(lengths), heads, 576, dtype=dtype, device="cuda")
        at = [None] * len(lengths)
        for b, c in enumerate(held):
            if len(c):
                q[b], at[b] = needles(c, i * heads, heads, dtype)
        out = ada_mla.mla_decode_paged(q, cache, table, cu, total_tokens=sum(lengths), cache_scale=0.0625,
                                       num_splits=(0, 1, 3, 0, 7, 64)[i % 6])
        for b, c in enumerate(held):
            if len(c) == 0:
                assert (out[b] == 0).all()
            elif i * heads < len(c):
                worst = needle_worst(out[b], q[b], c, at[b])
                assert worst <= 1.0, (i, b, worst)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("page,lengths", CASES)
def test_each_request(dtype, heads, page, lengths):
    cache, table, cu, held, gen = _case(heads + page + 1, lengths, page, 0.0625)
    q = torch.randn(len(lengths), heads, 576, generator=gen).to(dtype)
    for splits in (0, 1, 5):
        out = ada_mla.mla_decode_paged(q.cuda(), cache, table, cu, total_tokens=sum(lengths), cache_scale=0.0625, num_splits=splits)
        for b, c in enumerate(held):
            if len(c):
                rel = norm_error(out[b].cpu(), q[b], c)
                assert rel <= norm_bound(dtype, heads % 32 == 0), (splits, b, rel)
