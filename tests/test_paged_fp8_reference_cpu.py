"""The checks of the paged fp8 decode notice a token that is missing, counted twice or read from elsewhere: exact
results, rounded once, of histories with such a mistake."""
import pytest
import torch

from paged_fp8_reference import attention, needle_worst, needles, norm_bound, norm_error

LENGTHS = [129, 64, 700, 300, 1000]


def _history(n, seed=0):
    gen = torch.Generator()
    gen.manual_seed(n + seed)
    return (torch.randn(n, 576, generator=gen) * 16).to(torch.float8_e4m3fn).double() / 16, gen


def _mistakes(c):
    return {"last": c[:-1], "first": c[1:], "page's first": torch.cat([c[:32], c[33:]]), "twice": torch.cat([c, c[-1:]]),
            "another": torch.cat([c[:-1], c[:1]])}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", LENGTHS)
def test_norms(n, dtype):
    c, gen = _history(n)
    q = torch.randn(64, 576, generator=gen).to(dtype)
    assert norm_error(attention(q, c).to(dtype), q, c) <= 0.5 * norm_bound(dtype, True)
    for what, wrong in _mistakes(c).items():
        assert norm_error(attention(q, wrong).to(dtype), q, c) > norm_bound(dtype, True), what


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, *LENGTHS])
def test_needles(n, dtype):
    c, _ = _history(n)
    for first in range(0, n, 64):
        q, at = needles(c, first, 64, dtype)
        assert needle_worst(attention(q, c).to(dtype), q, c, at) <= 1.0
        if n == 1:
            continue
        for gone in {0, n // 2, n - 1}:
            keep = torch.arange(n) != gone
            worst = needle_worst(attention(q, c[keep]).to(dtype), q, c, at)
            assert (worst > 1.0) == bool((at == gone).any()), gone
