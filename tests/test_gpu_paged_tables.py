"""Block tables, slots and positions from request lengths (mla_paged_tables)
against a plain loop: whole numbers, equal to the last."""
import random

import pytest
import torch

import ada_mla
from operators_reference import tables

pytestmark = pytest.mark.gpu


def _call(context, new, table, free, start, page, total_new):
    dev = "cuda:0"
    i32 = dict(dtype=torch.int32, device=dev)
    t = torch.tensor(table, **i32)
    got = ada_mla.mla_paged_tables(torch.tensor(context, **i32), torch.tensor(new, **i32), t,
                                   torch.tensor(free, **i32), torch.tensor([start], **i32), page, total_new)
    return [t.tolist()] + [x.tolist() for x in got]


def _case(rng, batch, context, new, page, spare=0):
    """Lengths, a table whose held pages are distinct, and the free list behind them."""
    c = [rng.randint(0, context) for _ in range(batch)]
    n = [rng.randint(0, new) for _ in range(batch)]
    held = [-(-x // page) for x in c]
    width = max(1, max(-(-(x + y) // page) for x, y in zip(c, n))) + 1
    ids = list(range(sum(held) + sum(-(-(x + y) // page) for x, y in zip(c, n)) + spare + 4))
    rng.shuffle(ids)
    table, k = [], 0
    for h in held:
        table.append(ids[k:k + h] + [-7] * (width - h))
        k += h
    return c, n, table, ids[k:]


def _check(context, new, table, free, start, page, total_new):
    got = _call(context, new, table, free, start, page, total_new)
    t, cu, cu_new, slots, positions, nxt = tables(context, new, table, free, start, page, total_new)
    assert got[1] == cu and got[2] == cu_new and got[5] == [nxt]
    assert got[4] == positions
    assert got[3] == slots
    assert got[0] == t


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 255, 256, 257, 700])
@pytest.mark.parametrize("page", [32, 128])
def test_ragged_lengths(batch, page):
    rng = random.Random(batch * page)
    c, n, table, free = _case(rng, batch, 400, 70, page)
    _check(c, n, table, free, 2, page, sum(n))


@pytest.mark.parametrize("context,new", [(0, 1), (0, 3000), (31, 1), (32, 1), (33, 64), (1000, 0)])
def test_one_request(context, new):
    held = -(-context // 32)
    table = [list(range(held)) + [-1] * (-(-new // 32) + 2)]
    _check([context], [new], table, list(range(held, held + 200)), 0, 32, new)


def test_long_prompts_over_many_workgroups():
    rng = random.Random(5)
    c, n, table, free = _case(rng, 40, 100, 9000, 64)
    _check(c, n, table, free, 0, 64, sum(n))


def test_padded_and_clipped_token_counts():
    rng = random.Random(6)
    c, n, table, free = _case(rng, 300, 200, 20, 32)
    _check(c, n, table, free, 1, 32, sum(n) + 777)  # entries past the last token
    _check(c, n, table, free, 1, 32, sum(n) // 2)   # the last requests clipped
    _check(c, n, table, free, 1, 32, 0)


def test_the_free_list_ends():
    rng = random.Random(7)
    c, n, table, free = _case(rng, 50, 100, 90, 32)
    taken = tables(c, n, table, free, 0, 32, sum(n))[5]
    _check(c, n, table, free[:taken // 2], 0, 32, sum(n))
    _check(c, n, table, [], 0, 32, sum(n))
    _check(c, n, table, free, len(free) + 10, 32, sum(n))
    _check(c, n, table, free, -3, 32, sum(n))


def test_the_table_is_too_narrow_or_holds_no_page():
    rng = random.Random(8)
    c, n, table, free = _case(rng, 20, 300, 90, 32)
    narrow = [r[:3] for r in table]
    _check(c, n, narrow, free, 0, 32, sum(n))
    missing = [[-1] * len(r) for r in table]
    _check(c, n, missing, free, 0, 32, sum(n))


def test_negative_and_huge_lengths():
    big = 2 ** 31 - 1
    _check([-5, 40, 3], [10, -2, 5], [[-1] * 4, [0, 1, -1, -1], [2, -1, -1, -1]], [9, 8, 7], 0, 32, 15)
    # sums stop at INT_MAX; the huge request's positions run past its table
    _check([big - 40, 7], [20, 3], [[1] * 4, [2] * 4], [5, 6], 0, 32, 23)
    _check([big - 8, big], [0, 0], [[1], [1]], [5, 6], 0, 1 << 20, 0)


def test_slots_pass_32_bits():
    page = 1 << 20
    got = _call([page * 2 + 5], [3], [[1, 2, 2 ** 31 - 2]], [0], 0, page, 3)
    assert got[3] == [(2 ** 31 - 2) * page + 5 + i for i in range(3)]


def test_captured_and_replayed():
    i32 = dict(dtype=torch.int32, device="cuda:0")
    context, new = torch.zeros(9, **i32), torch.zeros(9, **i32)
    free, start = torch.arange(500, **i32), torch.zeros(1, **i32)
    table = torch.full((9, 20), -1, **i32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ada_mla.mla_paged_tables(context, new, table, free, start, 32, 128)
    rng = random.Random(9)
    have, rows, at = [0] * 9, [[-1] * 20 for _ in range(9)], 0
    for _ in range(6):  # a growing batch: each replay continues where the one before ended
        step = [rng.randint(0, 14) for _ in range(9)]
        context.copy_(torch.tensor(have, **i32))
        new.copy_(torch.tensor(step, **i32))
        graph.replay()
        torch.cuda.synchronize()
        rows, cu, cu_new, slots, positions, at = tables(have, step, rows, list(range(500)), at, 32, 128)
        assert table.tolist() == rows
        assert [x.tolist() for x in out] == [cu, cu_new, slots, positions, [at]]
        start.copy_(out[4])
        have = [a + b for a, b in zip(have, step)]
