"""Plain float64 forms of the operators around the decode (block tables, cache
rows, drafted trees, prompts), the inputs of their tests, and how far a result
may be from them.

Tolerances. A rounding to a 16-bit type is off by at most u = eps / 2 of the
value. attention_check() takes a result's error apart, element by element:
  out = sum_t p_t v_t / l, rounded once                      u |ref|
  p_t rounded to 16 bits (the sum l is of the fp32 values)   u sum p |v| / l
  p_t below the type's normal range (fp16: steps of 2^-24)   n 2^-25 max|v| / L
  logits in fp32: d values added up, each addition off by 2^-24 of a partial
  sum that is at most S = sum |q| |k|; the exponential adds 2^-22 of its
  argument: a factor (1 + g) on each p_t, g = 2 (d + 8) 2^-24 scale S + 2^-18,
  in the numerator and in l                                  2 g sum p |v| / l
  prefill: k and v rounded to 16 bits                        u sum p |v| / l, and
                                                             g += 2 u scale S
L = sum exp(s - max s) is at most the kernels' own l: their reference maximum
never exceeds the row's. Rounding errors are independent, so the 2-norm of the error
is far below the bound: each rounding of N values of random sign adds u /
sqrt(3) of the result's norm at most, the roundings adding in quadrature: two of them (p,
out) give 0.82 u, with k and v (the first through logits of standard deviation near
one) 1.2 u; 1.5 u and 2 u are asked for.
"""
import math

import torch

SCALE = 1.0 / math.sqrt(192.0)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention_check(got, q, k, v, seen, dtype, rounded_kv=False, what=""):
    """got [rows, dv] (16 bits) against softmax over the seen keys, q [rows, d], k [keys, d], v [keys, dv] in
    float64 (unrounded k, v). Returns (squared error, squared norm) for a 2-norm over several calls."""
    u = half_step(dtype)
    ref = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    some = seen.any(1)
    assert not got[~some].any(), f"{what}: a row that sees nothing is not zero"
    if not some.any():
        return 0.0, 0.0
    q, seen, out = q[some], seen[some], got[some].double()
    s = (q @ k.T * SCALE).masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(1, keepdim=True))
    total = p.sum(1, keepdim=True)
    ref = p @ v / total
    spread = p @ v.abs() / total
    reach = (q.abs() @ k.abs().T * SCALE).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    g = 2 * (q.shape[1] + 8) * 2.0 ** -24 * reach + 2.0 ** -18
    if rounded_kv:
        g = g + 2 * u * reach
    bound = u * ref.abs() * (1 + u) + (u * (2 if rounded_kv else 1) + 2 * g) * (1 + g) * spread
    if dtype == torch.float16:
        bound = bound + k.shape[0] * 2.0 ** -25 * v.abs().amax() / total
    # an output below the normal range has an absolute step
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    err = (out - ref).abs()
    worst = (err / bound).max().item()
    assert torch.isfinite(out).all() and worst <= 1.0, f"{what}: error {worst:.2f} times its bound"
    return (err ** 2).sum().item(), (ref ** 2).sum().item()


def chain_mask(drafts):
    return [(1 << (i + 1)) - 1 for i in range(drafts)]


def random_tree(rng, drafts):
    """Ancestor masks of a random tree: a list of drafted tokens' bits, each with its own."""
    masks = []
    for i in range(drafts):
        parent = rng.randint(-1, i - 1) if i else -1
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return masks


def signed(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def tables(context, new, block_table, free_pages, free_start, page, total_new):
    """The block table (a copy, updated), cu_seqlens, cu_new, slots, positions and free_next in plain Python."""
    table = [list(r) for r in block_table]
    most = 2 ** 31 - 1
    cu_seqlens, cu_new, slots, positions, at = [0], [0], [], [], free_start
    for b, (n, k) in enumerate(zip(context, new)):
        n, k = max(n, 0), max(k, 0)
        k = min(k, total_new - cu_new[-1])
        end = min(n + k, most)
        for col in range(-(-n // page), -(-end // page)):
            if col < len(table[b]):
                table[b][col] = free_pages[at] if 0 <= at < len(free_pages) else -1
            at += 1
        for p in range(n, n + k):
            col = p // page
            held = table[b][col] if col < len(table[b]) else -1
            slots.append(held * page + p % page if held >= 0 else -1)
            positions.append(p)
        cu_seqlens.append(min(cu_seqlens[-1] + end, most))
        cu_new.append(cu_new[-1] + k)
    pad = total_new - len(slots)
    return table, cu_seqlens, cu_new, slots + [-1] * pad, positions + [0] * pad, at


def rotate(x, cos, sin, interleaved):
    """Pairs of x [..., 64] turned by the angles of cos, sin [..., 32]."""
    even = torch.arange(0, 64, 2) if interleaved else torch.arange(32)
    odd = even + (1 if interleaved else 32)
    out = torch.empty_like(x)
    out[..., even] = x[..., even] * cos - x[..., odd] * sin
    out[..., odd] = x[..., odd] * cos + x[..., even] * sin
    return out


def latent_rows(kv, weight, cos, sin, eps, interleaved):
    """[tokens, 576] in float64: normalised latents and rotated keys."""
    kv = kv.double()
    x = kv[:, :512]
    x = x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * weight.double()
    return torch.cat([x, rotate(kv[:, 512:], cos, sin, interleaved)], 1)


def gather_paged(cache, row_of_table, n):
    """The first n latent rows of one request, float64 on the CPU."""
    page = cache.shape[1]
    ids = row_of_table[: -(-n // page)].long().cpu()
    return cache.cpu().double()[ids].reshape(-1, cache.shape[2])[:n]


def paged_case(gen, rng, lengths, page, dtype, spare_columns=2):
    """A paged cache of N(0, 1) rows and a shuffled block table for the lengths: rows behind a request's last are
    NaN, table columns behind its last hold ids far out of range. -> cache, block_table, cu_seqlens (on the GPU)."""
    need = [-(-n // page) for n in lengths]
    pages = max(1, sum(need)) + 2
    order = list(range(pages))
    rng.shuffle(order)
    cache = torch.randn(pages, page, 576, generator=gen).to(dtype)
    width = max(need + [1]) + spare_columns
    table, k = [], 0
    for n, m in zip(lengths, need):
        ids = order[k:k + m]
        k += m
        if n % page:
            cache[ids[-1], n % page:] = float("nan")
        table.append(ids + [pages + 1000003] * (width - m))
    for p in order[k:]:
        cache[p] = float("nan")
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return (cache.cuda(), torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda())
