"""How far the paged decode over an fp8 cache may be from softmax attention in float64, request by request, tight enough
that a single token missing or counted twice shows.

2-norm of a request's error, N(0, 1) queries and keys, u half a step of the type. Independent roundings of at most r of a
value, spread evenly, make r / sqrt(3) of the norm:
  out, the split partials, P where it is stored and where its half is scaled    4 of u, 1.16 u
  head tiles of 32 and 64 hold Q* in two parts, 8 significant bits: 2^-8 of a value at most, 2^-8 / sqrt(3)
  sqrt(sum q^2 k^2) / sqrt(192) = 2^-8 sqrt(576 / (3 192)) = 2^-8 of a logit; independent from token to
  token, so that of the weights' norm, and of the output's
  fp16: P below its normal range                                                2^-12
in quadrature, and a quarter more for what a request's heads and tokens are spread by.
A missing token of n takes 1 / sqrt(n) of the norm with it.

One token with all the weight (a query along its row): out is its values, with 4 u of them and what the others weigh at
most, n exp(-(gap - 2 d)), gap to the next logit, d a logit's error: 2^-8 of sum |q| |k| / sqrt(192) and a
hundredth for the second part's smallest step and the fp32 sums.
"""
import math

import torch

from operators_reference import SCALE, half_step


def norm_bound(dtype, parts):
    return 1.25 * math.hypot(1.16 * half_step(dtype), 2.0 ** -8 if parts else 0.0, 2.0 ** -12 if dtype == torch.float16 else 0.0)


def attention(q, c):
    """q [heads, 576] over all tokens of c [n, 576], in float64."""
    return torch.softmax(q.double() @ c.double().T * SCALE, -1) @ c.double()[:, :512]


def norm_error(got, q, c):
    ref = attention(q, c)
    return ((got.double() - ref).norm() / ref.norm()).item()


def needles(c, first, heads, dtype):
    """Queries along the rows first, first + 1, .. (cyclically) of c [n, 576], and those rows' numbers."""
    at = torch.arange(first, first + heads, device=c.device) % c.shape[0]
    return c[at].to(dtype), at


def needle_worst(got, q, c, at):
    """The largest error of got [heads, 512], in bounds, where head h has to find row at[h] of c [n, 576] (float64)."""
    u, n, heads = half_step(q.dtype), c.shape[0], torch.arange(len(at), device=c.device)
    s = q.double() @ c.T * SCALE
    own = s[heads, at]
    s[heads, at] = float("-inf")
    gap = own - s.amax(1) if n > 1 else torch.full_like(own, 100.0)
    d = (q.double().abs() @ c.abs().T * SCALE).amax(1) * (2.0 ** -8 + 2.0 ** -14) + 0.01
    others = n * torch.exp(-(gap - 2 * d))
    assert others.max() < 1e-4, "the others weigh too much"
    v = c[at, :512]
    bound = 4 * u * v.abs() + (2 * others * c[:, :512].abs().max())[:, None] + (2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -120)
    err = (got.double() - v).abs()
    return (err / bound).nan_to_num(float("inf"), posinf=float("inf")).max().item()
