"""Decode of drafted trees (mla_decode_tree) against float64: head counts,
drafted tokens, lengths at the edges of blocks, pages and splits, masks, rows
that see nothing, and what masked places hold. Tolerances: operators_reference."""
import random

import pytest
import torch

import ada_mla
from ada_mla import capi
from operators_reference import (attention_check, chain_mask, gather_paged, half_step, paged_case, random_tree, signed)

pytestmark = pytest.mark.gpu


def _check(got, q, cache, table, lengths, drafts, masks, dtype, what):
    se = sn = 0.0
    batch, m, heads, _ = q.shape
    for b in range(batch):
        n, k = lengths[b], drafts[b]
        c = gather_paged(cache, table[b], n)
        context = n - k
        for i in range(m):
            seen = torch.zeros(1, n, dtype=torch.bool)
            if i < k:
                seen[0, :max(context, 0)] = True
                for j in range(k):
                    if masks[b][i] >> j & 1 and context + j >= 0:
                        seen[0, context + j] = True
            e = attention_check(got[b, i].cpu(), q[b, i].double().cpu(), c, c[:, :512], seen.expand(heads, n), dtype,
                                what=f"{what} request {b} draft {i}")
            se, sn = se + e[0], sn + e[1]
    if sn:
        assert (se / sn) ** 0.5 <= 1.5 * half_step(dtype), f"{what}: 2-norm {(se / sn) ** 0.5:.2e}"


def _run(heads, m, lengths, drafts, page, dtype, seed, splits=0, tree=True):
    rng = random.Random(seed)
    gen = torch.Generator()
    gen.manual_seed(seed)
    cache, table, cu = paged_case(gen, rng, lengths, page, dtype)
    q = torch.randn(len(lengths), m, heads, 576, generator=gen).to(dtype).cuda()
    masks = [random_tree(rng, m) if tree else chain_mask(m) for _ in lengths]
    mask = torch.tensor([signed(x) for x in masks], dtype=torch.int64, device="cuda")
    lens = torch.tensor(drafts, dtype=torch.int32, device="cuda") if drafts is not None else None
    got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, draft_lens=lens, total_tokens=sum(lengths),
                                  num_splits=splits)
    torch.cuda.synchronize()
    _check(got, q, cache, table, lengths, [m] * len(lengths) if drafts is None else drafts, masks, dtype,
           f"heads {heads} drafts {m} page {page} splits {splits}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,m", [(16, 1), (16, 3), (48, 5), (128, 1), (32, 64), (128, 7)])
def test_heads_and_drafts(heads, m, dtype):
    _run(heads, m, [max(n, m) for n in (m, 200, 97)], None, 32, dtype, seed=heads + m)


@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("splits", [0, 1, 3, 50])
def test_lengths_at_edges(page, splits):
    lengths = [4, 5, 31, 32, 33, 63, 64, 65, 127, 129, 300]
    _run(16, 4, lengths, None, page, torch.float16, seed=page + splits, splits=splits)


def test_ragged_drafts_and_empty_requests():
    lengths = [0, 9, 40, 0, 130, 1, 77]
    _run(32, 6, lengths, [0, 6, 0, 0, 5, 1, 3], 32, torch.bfloat16, seed=1)
    _run(32, 6, lengths, [0, 6, 0, 0, 5, 1, 3], 32, torch.float16, seed=2, splits=4)


def test_many_requests():
    rng = random.Random(3)
    lengths = [rng.randint(2, 120) for _ in range(150)]
    _run(16, 2, lengths, [rng.randint(0, 2) for _ in lengths], 32, torch.float16, seed=3)


def test_long_contexts():
    _run(16, 9, [5000, 17, 2100], None, 64, torch.bfloat16, seed=4)
    _run(128, 2, [9001], None, 128, torch.float16, seed=5)


def test_chain():
    _run(16, 8, [50, 8], None, 32, torch.float16, seed=6, tree=False)


def test_masks_without_bits_and_with_all():
    gen = torch.Generator()
    gen.manual_seed(7)
    # no context: a row without bits sees nothing and is zero; all 64 bits: everything
    for m, lengths in ((64, [64, 70]), (3, [3, 40])):
        cache, table, cu = paged_case(gen, random.Random(7), lengths, 32, torch.float16)
        q = torch.randn(2, m, 16, 576, generator=gen).half().cuda()
        masks = [[(0, (1 << 64) - 1, 1 << (m - 1))[i % 3] for i in range(m)] for _ in lengths]
        mask = torch.tensor([signed(x) for x in masks], dtype=torch.int64, device="cuda")
        got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=sum(lengths))
        _check(got, q, cache, table, lengths, [m, m], masks, torch.float16, f"m {m}")


def test_more_drafts_than_tokens():
    # inconsistent lengths (fewer tokens than drafts): the drafted tokens that are there count from the end
    gen = torch.Generator()
    gen.manual_seed(8)
    cache, table, cu = paged_case(gen, random.Random(8), [3], 32, torch.float16)
    q = torch.randn(1, 5, 16, 576, generator=gen).half().cuda()
    masks = [chain_mask(5)]
    mask = torch.tensor([signed(x) for x in masks], dtype=torch.int64, device="cuda")
    got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=3)
    _check(got, q, cache, table, [3], [5], masks, torch.float16, "short")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("splits", [1, 4])
def test_a_branch_that_is_not_finite_stays_its_own(dtype, value, splits):
    gen = torch.Generator()
    gen.manual_seed(9)
    m, n = 4, 132
    cache, table, cu = paged_case(gen, random.Random(9), [n], 32, dtype)
    q = torch.randn(1, m, 16, 576, generator=gen).to(dtype).cuda()
    masks = [[1, 2, 5, 8]]  # token 2 descends from 0
    mask = torch.tensor(masks, dtype=torch.int64, device="cuda")
    want = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=n, num_splits=splits)
    row = n - m + 2
    page = int(table[0, row // 32])
    cache[page, row % 32, 5] = value
    got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=n, num_splits=splits)
    assert torch.equal(got[0, [0, 1, 3]], want[0, [0, 1, 3]])
    # also where the logit is -inf: its weight 0 times the infinity is a NaN too
    assert torch.isnan(got[0, 2]).all()


def test_uniform_and_extreme_logits():
    gen = torch.Generator()
    gen.manual_seed(10)
    for scale in (0.0, 30.0):  # all weights equal; nearly one-hot, logits of hundreds
        cache, table, cu = paged_case(gen, random.Random(10), [333], 64, torch.float16)
        q = (scale * torch.randn(1, 2, 16, 576, generator=gen)).half().cuda()
        masks = [chain_mask(2)]
        mask = torch.tensor(masks, dtype=torch.int64, device="cuda")
        got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=333)
        c = gather_paged(cache, table[0], 333)
        for i in range(2):
            seen = torch.ones(16, 333, dtype=torch.bool)
            seen[:, 331 + i + 1:] = False
            attention_check(got[0, i].cpu(), q[0, i].double().cpu(), c, c[:, :512], seen, torch.float16,
                            what=f"scale {scale}")


def test_rising_logits_move_the_reference():
    # each block's largest logit exceeds the one before by more than the lazy rescale's margin
    gen = torch.Generator()
    gen.manual_seed(11)
    n = 320
    cache = torch.randn(10, 32, 576, generator=gen)
    direction = torch.randn(576, generator=gen)
    steps = torch.arange(n).view(10, 32, 1) / n
    cache = (cache * 0.1 + direction * steps * 2).half().cuda()
    table = torch.arange(10, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = (direction * 2).expand(1, 1, 16, 576).half().contiguous().cuda()
    mask = torch.ones(1, 1, dtype=torch.int64, device="cuda")
    for splits in (1, 3):
        got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=n, num_splits=splits)
        c = gather_paged(cache, table[0], n)
        attention_check(got[0, 0].cpu(), q[0, 0].double().cpu(), c, c[:, :512], torch.ones(16, n, dtype=torch.bool),
                        torch.float16, what=f"splits {splits}")


def test_matches_the_single_token_decode():
    gen = torch.Generator()
    gen.manual_seed(12)
    lengths = [700, 33, 1, 256]
    cache, table, cu = paged_case(gen, random.Random(12), lengths, 64, torch.float16)
    q = torch.randn(4, 1, 128, 576, generator=gen).half().cuda()
    mask = torch.ones(4, 1, dtype=torch.int64, device="cuda")
    tree = ada_mla.mla_decode_tree(q, cache, table, cu, mask)[:, 0].float()
    one = ada_mla.mla_decode_paged(q[:, 0].contiguous(), cache, table, cu).float()
    # both are within 2 u sum p |v| / l <= 2 u max |v| of the same value (and the paged decode rounds its partials once more)
    assert (tree - one).abs().max() <= 5 * half_step(torch.float16) * torch.nan_to_num(cache.float()).abs().max()


def test_page_ids_out_of_range_stay_inside_the_cache():
    gen = torch.Generator()
    gen.manual_seed(13)
    cache, table, cu = paged_case(gen, random.Random(13), [100, 64], 32, torch.float16)
    cache = torch.nan_to_num(cache)
    q = torch.randn(2, 2, 16, 576, generator=gen).half().cuda()
    mask = torch.tensor([[1, 3], [1, 3]], dtype=torch.int64, device="cuda")
    good = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=164)
    table[0, 1] = -5
    table[0, 2] = 2 ** 31 - 1
    got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=164)
    assert torch.isfinite(got).all() and torch.equal(got[1], good[1])


def test_shared_workspace_and_stale_partials():
    # a workspace of NaNs, reused by calls of other shapes
    gen = torch.Generator()
    gen.manual_seed(14)
    lib = capi.load()
    sizes = [(1, 3, 16, [400]), (3, 5, 32, [64, 0, 700]), (2, 1, 16, [31, 32])]
    need = max(lib.mla_decode_tree_workspace_size(b, m, h, sum(n), 7) for b, m, h, n in sizes)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    for b, m, h, n in sizes + sizes[:1]:
        cache, table, cu = paged_case(gen, random.Random(14), n, 32, torch.float16)
        q = torch.randn(b, m, h, 576, generator=gen).half().cuda()
        masks = [chain_mask(m)] * b
        mask = torch.tensor(masks, dtype=torch.int64, device="cuda")
        lens = [min(m, x) for x in n]
        got = capi.decode_tree(q, cache, table, cu, mask, sum(n), draft_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                               num_splits=7, workspace=ws)
        _check(got, q, cache, table, n, lens, masks, torch.float16, f"{b} {m} {h}")


def test_captured_and_replayed():
    gen = torch.Generator()
    gen.manual_seed(15)
    lengths = [300, 45, 128]
    cache, table, cu = paged_case(gen, random.Random(15), lengths, 32, torch.float16)
    cache = torch.nan_to_num(cache)
    q = torch.randn(3, 4, 16, 576, generator=gen).half().cuda()
    mask = torch.tensor([chain_mask(4)] * 3, dtype=torch.int64, device="cuda")
    call = lambda: ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=600)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(4):
        q.normal_()
        cache.normal_()
        cu[1:].sub_(r)  # shorter requests under the same plan
        want = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(out, want), r


def test_another_stream():
    gen = torch.Generator()
    gen.manual_seed(16)
    cache, table, cu = paged_case(gen, random.Random(16), [500], 32, torch.bfloat16)
    q = torch.randn(1, 4, 32, 576, generator=gen).bfloat16().cuda()
    mask = torch.tensor([chain_mask(4)], dtype=torch.int64, device="cuda")
    want = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=500)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=500)
    side.synchronize()
    assert torch.equal(got, want)


def test_cache_rows_past_2_to_31_elements():
    # a pool of more than 2^32 bytes whose last pages hold the request
    gen = torch.Generator()
    gen.manual_seed(17)
    page, n = 64, 200
    pages = 2 ** 31 // (576 * page) + 6
    cache = torch.zeros(pages, page, 576, dtype=torch.bfloat16, device="cuda")
    ids = [pages - 1, 3, pages - 2, pages - 3]
    for i in ids:
        cache[i] = torch.randn(page, 576, generator=gen).bfloat16().cuda()
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 3, 16, 576, generator=gen).bfloat16().cuda()
    masks = [chain_mask(3)]
    mask = torch.tensor(masks, dtype=torch.int64, device="cuda")
    got = ada_mla.mla_decode_tree(q, cache, table, cu, mask, total_tokens=n)
    small = cache[ids].contiguous()
    order = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(got, ada_mla.mla_decode_tree(q, small, order, cu, mask, total_tokens=n))
    _check(got, q, small, order, [n], [3], masks, torch.bfloat16, "far pages")


def test_one_long_request_among_empty_ones():
    lengths = [0] * 30 + [4000] + [0, 3] * 10
    _run(16, 3, lengths, [min(3, n) for n in lengths], 64, torch.float16, seed=18)


def test_most_drafts_and_heads():
    _run(256, 64, [100], [64], 32, torch.bfloat16, seed=19)


def test_splits_counted_through_many_requests():
    # more requests than lanes, several splits each, empty requests between
    rng = random.Random(23)
    lengths = [rng.choice([0, 1, 32, 200, 333, 700]) for _ in range(150)]
    drafts = [min(2, n) for n in lengths]
    _run(16, 2, lengths, drafts, 32, torch.float16, 23, splits=3)
    # equal lengths, whose splits leave every request's last slot empty
    _run(16, 3, [160] * 40, [3] * 40, 32, torch.bfloat16, 24, splits=1)
    _run(16, 3, [448] * 24, [3] * 24, 64, torch.float16, 25, splits=7)
