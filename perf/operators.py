"""The operators around the latent-cache decode, as a serving loop calls them, for timing and checking.

Four operators, which a serving loop runs one after another on one paged cache of latent rows
(512 compressed values and 64 rotary ones a token):

  tables   block tables, slots and positions of the tokens of one step, from the requests' lengths
  append   a step's latent rows normalised, rotated and written to their slots, its queries rotated
  tree     attention of a tree of drafted tokens a request over the cache (absorbed form)
  prefill  causal attention of prompts or chunks of prompts (expanded form)

listed() holds fixed cases and draw() more of the same ranges; a case is one call. Where `own` is
false, run() computes the operator from elementary torch operations in 32 bits, else it calls ada_mla.
Latents, queries and rotary parts are N(0, 1), weights N(0, 1 / fan-in), as normalised activations are.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
LATENT, ROPE, ROW = 512, 64, 576
SCALE = 1.0 / math.sqrt(192.0)  # softmax scale: 128 + 64 values of a head's key before absorption
EPS = 1e-6
FP8_SCALE = 0.0625  # normalised latents stay below 448 * 0.0625 = 28
MOST_SCORES = 64 * 8192 * 8192  # most scores (head, query, key) of one case, padding counted


def listed():
    return [
        # one decode step of a serving batch: a token a request, latency is all there is
        dict(name="tables_step", op="tables", batch=64, context=8000, new=1, ragged=False, page=64, mix=1),
        # a burst of prompts admitted at once
        dict(name="tables_prompts", op="tables", batch=301, context=0, new=2000, ragged=True, page=128, mix=2),
        # the cache rows and queries of one decode step, all heads
        dict(name="append_step", op="append", tokens=64, heads=128, dtype="bf16", cache="bf16", page=64,
             interleaved=True, padded=0, mix=3),
        # the rows of long prompts into a quantised cache, on one rank of eight
        dict(name="append_prompts_fp8", op="append", tokens=32768, heads=16, dtype="fp16", cache="fp8", page=64,
             interleaved=False, padded=0, mix=4),
        # a small tree behind a short conversation, few heads: latency and one split over the chip
        dict(name="tree_short", op="tree", batch=1, drafts=7, ragged=False, heads=16, context=1003, mixed=False,
             page=64, dtype="fp16", mix=5),
        # a serving batch on one rank of eight: few rows a request, a memory stream
        dict(name="tree_few_heads", op="tree", batch=48, drafts=5, ragged=True, heads=16, context=12000, mixed=True,
             page=64, dtype="bf16", mix=6),
        # the same with all heads: many rows share each latent row
        dict(name="tree_batch", op="tree", batch=16, drafts=16, ragged=True, heads=128, context=4000, mixed=True,
             page=32, dtype="bf16", mix=7),
        # a wide tree behind a long document
        dict(name="tree_long", op="tree", batch=1, drafts=32, ragged=False, heads=128, context=50021, mixed=False,
             page=128, dtype="fp16", mix=8),
        # one short prompt on one rank of eight
        dict(name="prefill_short", op="prefill", batch=1, queries=197, context=0, mixed=False, heads=16, page=0,
             dtype="fp16", mix=9),
        # prompts of mixed lengths, packed, all heads
        dict(name="prefill_batch", op="prefill", batch=6, queries=1500, context=0, mixed=True, heads=128, page=0,
             dtype="bf16", mix=10),
        # chunks of prompts behind what the paged cache already holds
        dict(name="prefill_chunk", op="prefill", batch=2, queries=1024, context=9001, mixed=False, heads=32, page=64,
             dtype="fp16", mix=11),
        # one long prompt
        dict(name="prefill_long", op="prefill", batch=1, queries=8192, context=0, mixed=False, heads=64, page=64,
             dtype="bf16", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, odd ones among them."""
    op = rng.choice(["tables", "append", "tree", "tree", "prefill", "prefill"])
    page, mix = rng.choice([32, 64, 128]), rng.randrange(1 << 30)
    dtype = rng.choice(["fp16", "bf16"])
    if op == "tables":
        batch = _log(rng, 1, 2048)
        return dict(op=op, batch=batch, context=rng.choice([0, _log(rng, 1, 16384)]),
                    new=_log(rng, 1, min(8192, max(1, 600000 // batch))), ragged=rng.random() < 0.7, page=page, mix=mix)
    if op == "append":
        heads = rng.choice([0, 16, 48, 128])
        tokens = _log(rng, 1, 32768 if heads <= 16 else 4096)
        return dict(op=op, tokens=tokens, heads=heads, dtype=dtype, cache=rng.choice([dtype, dtype, "fp8"]), page=page,
                    interleaved=rng.random() < 0.5, padded=rng.choice([0, 0, tokens // 3]), mix=mix)
    if op == "tree":
        heads, batch, drafts = rng.choice([16, 32, 64, 128]), _log(rng, 1, 64), _log(rng, 1, 64)
        most = 128 * 32 * 50021 // (heads * batch * drafts)
        return dict(op=op, batch=batch, drafts=drafts, ragged=rng.random() < 0.5, heads=heads,
                    context=_log(rng, 1, max(2, min(65536, most, 576000 // batch) - drafts)), mixed=rng.random() < 0.6, page=page,
                    dtype=dtype, mix=mix)
    heads, batch = rng.choice([16, 32, 64, 128]), _log(rng, 1, 16)
    side = math.isqrt(MOST_SCORES // (2 * heads * batch))
    queries = _log(rng, 1, min(8192, side))
    # all keys are expanded, whatever the queries: they are bounded by themselves too
    most = min(MOST_SCORES // (4 * heads * batch * queries), 8192 * 64 // (heads * batch), 16384)
    return dict(op=op, batch=batch, queries=queries, context=rng.choice([0, _log(rng, 1, max(2, most - queries))]),
                mixed=rng.random() < 0.6, heads=heads, page=rng.choice([0, page]), dtype=dtype, mix=mix)


# ---- sizes of a case ------------------------------------------------------


def _prefix(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _tables_lengths(case):
    r = random.Random(case["mix"])
    context = [r.randint(0, case["context"]) for _ in range(case["batch"])]
    new = [r.randint(0, case["new"]) if case["ragged"] else case["new"] for _ in range(case["batch"])]
    if not any(new):
        new[0] = 1
    return context, new


def _tree_sizes(case):
    """(context length, drafted tokens, their ancestor masks) of each request."""
    r = random.Random(case["mix"])
    out = []
    for _ in range(case["batch"]):
        context = r.randint(0, case["context"]) if case["mixed"] else case["context"]
        drafts = r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"]
        masks = []
        for i in range(case["drafts"]):
            parent = r.randint(-1, i - 1) if i else -1
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        out.append((context, drafts, masks))
    return out


def _prefill_lengths(case):
    r = random.Random(case["mix"])
    queries = [r.randint(1, case["queries"]) if case["mixed"] else case["queries"] for _ in range(case["batch"])]
    context = [r.randint(0, case["context"]) if case["mixed"] else case["context"] for _ in range(case["batch"])]
    return queries, [q + c for q, c in zip(queries, context)]


# ---- inputs ---------------------------------------------------------------


class _State:
    pass


def _normal(gen, *shape, dtype, scale=1.0):
    t = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    return (t * scale if scale != 1.0 else t).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _cos_sin(positions):
    """[positions, 64] fp32: 32 cosines, then 32 sines; the angles in 64 bits."""
    i = torch.arange(32, device=DEV, dtype=torch.float64)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-i / 32)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _paged(gen, lengths, page):
    """A block table that deals out shuffled pages to the lengths (-1 behind a request's last), and its page count."""
    need = [-(-n // page) for n in lengths]
    pages, width = max(1, sum(need)), max(1, max(need))
    order = torch.randperm(pages, generator=gen, device=DEV, dtype=torch.int32)
    column = torch.arange(width, device=DEV)
    first, count = _ints(_prefix(need)[:-1], torch.int64), _ints(need, torch.int64)
    at = (first[:, None] + column).clamp(max=pages - 1)
    return torch.where(column < count[:, None], order[at], -1).to(torch.int32).contiguous(), pages


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = _State()
    s.case, s.op = case, case["op"]
    if s.op == "tables":
        context, new = _tables_lengths(case)
        page = case["page"]
        held = [-(-n // page) for n in context]
        want = [-(-(n + k) // page) for n, k in zip(context, new)]
        s.context_lens, s.new_lens = _ints(context), _ints(new)
        s.total_new, s.page = sum(new), page
        taken = sum(held)
        pool = torch.randperm(sum(want) + 5, generator=gen, device=DEV, dtype=torch.int32)
        width = max(1, max(want))
        column = torch.arange(width, device=DEV)
        first = _ints(_prefix(held)[:-1], torch.int64)
        at = (first[:, None] + column).clamp(max=pool.numel() - 1)
        s.block_table = torch.where(column < _ints(held, torch.int64)[:, None], pool[at], -1).to(torch.int32).contiguous()
        s.free_pages = torch.cat([pool[:3], pool[taken:]]).contiguous()  # three pages of it are taken already
        s.free_start = _ints([3])
        return s
    dt = DTYPES[case["dtype"]]
    if s.op == "append":
        r = random.Random(case["mix"])
        tokens, page = case["tokens"], case["page"]
        pages = -(-tokens // page) + 3
        s.kv = _normal(gen, tokens, ROW, dtype=dt, scale=1.7)
        s.weight = (1.0 + 0.2 * torch.randn(LATENT, generator=gen, device=DEV)).to(dt)
        s.q_rope = _normal(gen, tokens, case["heads"], ROPE, dtype=dt) if case["heads"] else None
        s.cos_sin = _cos_sin(32768 + 8192)
        base = r.randrange(8192)
        s.positions = (torch.arange(tokens, device=DEV, dtype=torch.int32) + base).contiguous()
        s.slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens].contiguous()
        if case["padded"]:  # a batch of fixed size whose last tokens are none
            s.slots[tokens - case["padded"]:] = -1
            s.positions[tokens - case["padded"]:] = 0
        s.cache = torch.zeros(pages, page, ROW, dtype=DTYPES[case["cache"]], device=DEV)
        return s
    h = case["heads"]
    if s.op == "tree":
        sizes = _tree_sizes(case)
        lengths = [c + d for c, d, _ in sizes]
        s.lens, s.draft_lens = _ints(lengths), _ints([d for _, d, _ in sizes])
        signed = [[m - (1 << 64) if m >> 63 else m for m in masks] for _, _, masks in sizes]
        s.tree_mask = _ints(signed, torch.int64)
        s.query = _normal(gen, case["batch"], case["drafts"], h, ROW, dtype=dt)
    else:
        queries, lengths = _prefill_lengths(case)
        total = sum(queries)
        s.q_lens, s.lens = _ints(queries), _ints(lengths)
        s.cu_q, s.most_q = _ints(_prefix(queries)), max(queries)
        s.q_nope = _normal(gen, total, h, 128, dtype=dt)
        s.q_rope = _normal(gen, total, h, ROPE, dtype=dt)
        s.w_uk = _normal(gen, h, 128, LATENT, dtype=dt, scale=LATENT ** -0.5)
        s.w_uv = _normal(gen, h, 128, LATENT, dtype=dt, scale=LATENT ** -0.5)
    s.cu_seqlens, s.total, s.most = _ints(_prefix(lengths)), sum(lengths), max(1, max(lengths))
    if case["page"]:
        s.block_table, pages = _paged(gen, lengths, case["page"])
        s.cache = _normal(gen, pages, case["page"], ROW, dtype=dt)
    else:
        s.block_table = None
        s.cache = _normal(gen, max(1, s.total), ROW, dtype=dt)
    return s


# ---- the plain forms ------------------------------------------------------


def _plain_tables(s):
    page, batch = s.page, s.context_lens.numel()
    context, new = s.context_lens.long(), s.new_lens.long()
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu_seqlens, cu_new = torch.cat([zero, (context + new).cumsum(0)]), torch.cat([zero, new.cumsum(0)])
    held, want = (context + page - 1) // page, (context + new + page - 1) // page
    first = s.free_start.long() + torch.cat([zero, (want - held).cumsum(0)])
    column = torch.arange(s.block_table.size(1), device=DEV)
    fresh = (column >= held[:, None]) & (column < want[:, None])
    at = (first[:batch, None] + column - held[:, None]).clamp(0, s.free_pages.numel() - 1)
    s.block_table.copy_(torch.where(fresh, s.free_pages[at], s.block_table))
    token = torch.arange(s.total_new, device=DEV)
    request = torch.searchsorted(cu_new, token, right=True) - 1
    positions = context[request] + token - cu_new[request]
    slots = s.block_table[request, positions // page].long() * page + positions % page
    return [s.block_table, cu_seqlens.int(), cu_new.int(), slots, positions.int(), first[batch:].int()]


def _rotate(x, cos, sin, interleaved):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)


def _plain_append(s):
    case = s.case
    angle = s.cos_sin[s.positions.long()]
    cos, sin = angle[:, :32], angle[:, 32:]
    x = s.kv.float()
    latent = x[:, :LATENT]
    latent = latent * torch.rsqrt((latent * latent).mean(-1, keepdim=True) + EPS) * s.weight.float()
    rows = torch.cat([latent, _rotate(x[:, LATENT:], cos, sin, case["interleaved"])], -1)
    slots, flat = s.slots, s.cache.view(-1, ROW)
    if case["padded"]:
        rows, slots = rows[slots >= 0], slots[slots >= 0]
    if case["cache"] == "fp8":
        quantised = (rows / FP8_SCALE).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        flat.view(torch.uint8)[slots] = quantised.view(torch.uint8)
    else:
        flat[slots] = rows.to(flat.dtype)
    if s.q_rope is None:
        return [s.cache]
    q = _rotate(s.q_rope.float(), cos[:, None], sin[:, None], case["interleaved"])
    return [s.cache, q.to(s.q_rope.dtype)]


def _rows(s):
    """The requests' latent rows in 32 bits, [batch, longest, 576], and which of them are tokens."""
    token = torch.arange(s.most, device=DEV)
    valid = token < s.lens[:, None]
    if s.block_table is None:
        at = s.cu_seqlens[:-1, None].long() + token
    else:
        page = s.cache.size(1)
        at = s.block_table[:, token // page].long() * page + token % page
    at = torch.where(valid, at, 0)
    return s.cache.view(-1, ROW)[at].float() * valid[..., None], valid


def _softmax(scores, seen):
    """exp(scores - max) over what is seen, and its sum (zeros where a row sees nothing)."""
    scores = scores.masked_fill(~seen, float("-inf"))
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == float("-inf"), 0.0, most))
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total == 0.0, 1.0, total)


def _plain_tree(s):
    batch, drafts, heads, _ = s.query.shape
    c, valid = _rows(s)
    token = torch.arange(s.most, device=DEV)
    behind = token - (s.lens - s.draft_lens)[:, None]  # which drafted token a key is; below 0: context
    bit = torch.bitwise_right_shift(s.tree_mask[:, :, None], behind.clamp(0, 63)[:, None, :]) & 1
    row = torch.arange(drafts, device=DEV)[:, None] < s.draft_lens[:, None, None]
    seen = valid[:, None, :] & ((behind < 0)[:, None, :] | (bit == 1)) & row
    q = s.query.float().view(batch, drafts * heads, ROW)
    scores = (torch.matmul(q, c.transpose(1, 2)) * SCALE).view(batch, drafts, heads, s.most)
    p, total = _softmax(scores, seen[:, :, None, :])
    out = torch.matmul(p.view(batch, drafts * heads, s.most), c[..., :LATENT])
    return (out.view(batch, drafts, heads, LATENT) / total).to(s.query.dtype)


def _plain_prefill(s):
    total, heads, _ = s.q_nope.shape
    c, valid = _rows(s)
    row = torch.arange(s.most_q, device=DEV)
    real = row < s.q_lens[:, None]
    at = torch.where(real, s.cu_q[:-1, None].long() + row, 0)
    latent, rope = c[:, None, :, :LATENT], c[:, None, :, LATENT:]
    k = torch.matmul(latent, s.w_uk.float().transpose(1, 2))
    v = torch.matmul(latent, s.w_uv.float().transpose(1, 2))
    q_nope, q_rope = s.q_nope.float()[at].transpose(1, 2), s.q_rope.float()[at].transpose(1, 2)
    scores = torch.matmul(q_nope, k.transpose(2, 3))
    scores += torch.matmul(q_rope, rope.transpose(2, 3))
    scores *= SCALE
    last = row + (s.lens - s.q_lens)[:, None]  # a query sees the keys up to its own position
    seen = valid[:, None, :] & (torch.arange(s.most, device=DEV) <= last[..., None])
    p, weight = _softmax(scores, seen[:, None])
    out = (torch.matmul(p, v) / weight).transpose(1, 2)
    return out[real].to(s.q_nope.dtype)


_PLAIN = {"tables": _plain_tables, "append": _plain_append, "tree": _plain_tree, "prefill": _plain_prefill}


# ---- the framework's operators --------------------------------------------

_package = None


def _ada_mla():
    global _package
    if _package is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ada-mla_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import ada_mla
        _package = ada_mla
    return _package


def _own_tables(s):
    cu_seqlens, cu_new, slots, positions, free_next = _ada_mla().mla_paged_tables(
        s.context_lens, s.new_lens, s.block_table, s.free_pages, s.free_start, s.page, s.total_new)
    return [s.block_table, cu_seqlens, cu_new, slots, positions, free_next]


def _own_append(s):
    q = _ada_mla().mla_append_kv(s.kv, s.weight, s.cos_sin, s.positions, s.slots, s.cache, q_rope=s.q_rope, eps=EPS,
                                 cache_scale=FP8_SCALE if s.case["cache"] == "fp8" else 1.0,
                                 interleaved=s.case["interleaved"])
    return [s.cache] if q is None else [s.cache, q]


def _own_tree(s):
    return _ada_mla().mla_decode_tree(s.query, s.cache, s.block_table, s.cu_seqlens, s.tree_mask,
                                      draft_lens=s.draft_lens, total_tokens=s.total)


def _own_prefill(s):
    return _ada_mla().mla_prefill(s.q_nope, s.q_rope, s.w_uk, s.w_uv, s.cache, s.cu_q, s.cu_seqlens,
                                  block_table=s.block_table, total_tokens=s.total)


_OWN = {"tables": _own_tables, "append": _own_append, "tree": _own_tree, "prefill": _own_prefill}


def run(state):
    return (_OWN if own else _PLAIN)[state.op](state)


# ---- what a pass cannot do without ----------------------------------------


def work(case):
    op = case["op"]
    if op == "tables":
        context, new = _tables_lengths(case)
        page = case["page"]
        pages = sum(-(-(n + k) // page) - -(-n // page) for n, k in zip(context, new))
        reads = sum(1 for n, k in zip(context, new) if k and n % page)  # a started page's entry
        return {"bytes": 16 * len(new) + 8 * pages + 4 * reads + 12 * sum(new), "flops": 0}
    if op == "append":
        n, h = case["tokens"], case["heads"]
        wide = 1 if case["cache"] == "fp8" else 2
        written = n - case["padded"]
        size = written * ROW * (2 + wide) + n * (12 + 256) + 2 * LATENT + n * h * ROPE * 4
        return {"bytes": size, "flops": written * LATENT * 4 + (written + n * h) * ROPE * 3}
    h, page = case["heads"], case["page"]
    if op == "tree":
        sizes = _tree_sizes(case)
        rows = case["batch"] * case["drafts"] * h
        pairs = sum(c * d + sum(bin(m & ((1 << d) - 1)).count("1") for m in masks[:d]) for c, d, masks in sizes)
        size = sum(c + d for c, d, _ in sizes) * ROW * 2 + rows * (ROW + LATENT) * 2
        size += sum(-(-(c + d) // page) for c, d, _ in sizes) * 4 + case["batch"] * (case["drafts"] * 8 + 8)
        return {"bytes": size, "flops": pairs * h * (ROW + LATENT) * 2}
    queries, lengths = _prefill_lengths(case)
    pairs = sum(q * n - q * (q - 1) // 2 for q, n in zip(queries, lengths))
    keys = sum(lengths)
    size = keys * ROW * 2 + sum(queries) * h * (192 + 128) * 2 + 2 * h * 128 * LATENT * 2 + 8 * len(queries)
    size += sum(-(-n // page) for n in lengths) * 4 if page else 0
    return {"bytes": size, "flops": pairs * h * (192 + 128) * 2 + keys * h * 256 * LATENT * 2}


# ---- the definitions in 64 bits -------------------------------------------


def _exact_append(s):
    case = s.case
    x = s.kv.double().cpu()
    pairs = list(range(32))
    even = [2 * i for i in pairs] if case["interleaved"] else pairs
    odd = [2 * i + 1 for i in pairs] if case["interleaved"] else [i + 32 for i in pairs]
    table = s.cos_sin.double().cpu()[s.positions.cpu().long()]

    def turn(y, turns):
        z = torch.complex(y[..., even], y[..., odd]) * turns
        out = torch.empty_like(y)
        out[..., even], out[..., odd] = z.real, z.imag
        return out

    turns = torch.complex(table[:, :32].contiguous(), table[:, 32:].contiguous())
    norm = x[:, :LATENT].square().sum(1).div(LATENT).add(EPS).sqrt()
    rows = torch.empty_like(x)
    rows[:, :LATENT] = x[:, :LATENT] / norm[:, None] * s.weight.double().cpu()
    rows[:, LATENT:] = turn(x[:, LATENT:], turns)
    if case["cache"] == "fp8":
        rows = rows / FP8_SCALE
    cache = torch.zeros(s.cache.numel() // ROW, ROW, dtype=torch.float64)
    slots = s.slots.cpu()
    kept = slots >= 0
    cache[slots[kept]] = rows[kept]
    out = [cache.view(s.cache.shape)]
    if s.q_rope is not None:
        out.append(turn(s.q_rope.double().cpu(), turns[:, None]))
    return out


def _request_rows(s, b):
    """Request b's latent rows in 64 bits."""
    n = int(s.lens[b])
    if s.block_table is None:
        at = int(s.cu_seqlens[b])
        return s.cache[at:at + n].double()
    page = s.cache.size(1)
    used = s.block_table[b, :-(-n // page)].long()
    return s.cache[used].double().reshape(-1, ROW)[:n]


def _exact_tree(s):
    batch, drafts, heads, _ = s.query.shape
    out = torch.zeros(batch, drafts, heads, LATENT, dtype=torch.float64, device=DEV)
    for b, (context, count, masks) in enumerate(_tree_sizes(s.case)):
        c = _request_rows(s, b)
        for i in range(count):
            at = list(range(context, context + count))
            keys = [t for t, j in zip(at, range(count)) if masks[i] >> j & 1]
            seen = torch.cat([c[:context], c[keys]])
            w = torch.softmax(s.query[b, i].double() @ seen.T * SCALE, -1)
            out[b, i] = w @ seen[:, :LATENT]
    return out


def _exact_prefill(s):
    total, heads, _ = s.q_nope.shape
    out = torch.zeros(total, heads, 128, dtype=torch.float64, device=DEV)
    queries, lengths = _prefill_lengths(s.case)
    at = 0
    for b, (m, n) in enumerate(zip(queries, lengths)):
        c = _request_rows(s, b)
        future = torch.ones(m, n, dtype=torch.bool, device=DEV).triu(n - m + 1)
        for h in range(heads):
            k = c[:, :LATENT] @ s.w_uk[h].double().T
            q = torch.cat([s.q_nope[at:at + m, h], s.q_rope[at:at + m, h]], 1).double()
            x = (q @ torch.cat([k, c[:, LATENT:]], 1).T * SCALE).masked_fill_(future, float("-inf"))
            out[at:at + m, h] = torch.softmax(x, -1) @ (c[:, :LATENT] @ s.w_uv[h].double().T)
        at += m
    return out


def exact(case, seed):
    if case["op"] == "tables":  # whole numbers
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "tree": _exact_tree, "prefill": _exact_prefill}[s.op](s)
