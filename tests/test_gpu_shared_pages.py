"""Tables of shared pages (fork, compaction) against plain Python, and the copies that they ask for."""
import random

import pytest
import torch

import ada_mla
from ada_mla import capi
from pages_reference import compact, fork, random_pool

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def _t(values):
    return torch.tensor(values, **I32)


def _fork(table, lens, parents, kept, pinned, free, start, page, num_pages, what, module=ada_mla):
    free_t = _t(free)
    args = dict(kept_lens=None if kept is None else _t(kept), pinned=None if pinned is None else _t(pinned))
    f = ada_mla.mla_fork_tables if module is ada_mla else capi.fork_tables
    got = f(_t(table), _t(lens), _t(parents), free_t, _t([start]), page, num_pages, **args)
    want = fork(table, lens, parents, [2 ** 31 - 1] * len(parents) if kept is None else kept,
                [0] * num_pages if pinned is None else pinned, free, start, page, num_pages)
    for name, g, w in zip(("table", "lens", "copies", "free_next", "free_pages"), [*got, free_t],
                          [want[0], want[1], want[2], [want[3]], want[4]]):
        assert g.tolist() == w, (what, name)
    return got


def _compact(table, lens, pinned, free, start, page, num_pages, what, module=ada_mla):
    f = ada_mla.mla_compact_tables if module is ada_mla else capi.compact_tables
    got = f(_t(table), _t(lens), _t(free), _t([start]), page, num_pages, pinned=None if pinned is None else _t(pinned))
    want = compact(table, lens, [0] * num_pages if pinned is None else pinned, free, start, page, num_pages)
    for name, g, w in zip(("table", "copies", "free_pages"), got, want):
        assert g.tolist() == w, (what, name)
    return got


SIZES = [(1, 1, 1, 32, 1), (1, 1, 7, 64, 3), (3, 5, 4, 32, 20), (17, 30, 19, 64, 150), (64, 64, 9, 128, 700),
         (65, 1100, 5, 32, 300), (1030, 40, 3, 32, 3000), (2, 3, 300, 32, 900), (8192, 20, 2, 32, 9000)]


@pytest.mark.parametrize("rows,batch,width,page,num_pages", SIZES)
@pytest.mark.parametrize("seed", range(3))
def test_random_forks(rows, batch, width, page, num_pages, seed):
    rng = random.Random(1000 * seed + rows)
    table, lens, free, start, pinned = random_pool(rng, rows, width, page, num_pages, odd=0.2 if seed == 2 else 0.0)
    lens = [n if rng.random() < 0.95 else rng.choice([-7, n + 5 * page * width, 2 ** 31 - 1]) for n in lens]
    parents = [rng.choice([rng.randrange(rows), rng.randrange(rows), rng.randrange(rows), -1, rows, 2 ** 31 - 1, -2 ** 31])
               for _ in range(batch)]
    kept = [rng.choice([2 ** 31 - 1, rng.randint(0, width * page), 0, -3, page, page + 1]) for _ in range(batch)]
    _fork(table, lens, parents, kept, pinned, free, start, page, num_pages, "kept, pinned")
    _fork(table, lens, parents, None, None, free, start, page, num_pages, "all", module=capi)


@pytest.mark.parametrize("rows,batch,width,page,num_pages", SIZES)
@pytest.mark.parametrize("seed", range(3))
def test_random_compactions(rows, batch, width, page, num_pages, seed):
    rng = random.Random(1000 * seed + rows)
    num_pages *= rng.choice([1, 2, 3])
    table, lens, free, start, pinned = random_pool(rng, rows, width, page, num_pages, odd=0.2 if seed == 2 else 0.0)
    if seed == 1 and len(free) > start + 2:  # ids twice, none, out of range, held
        free[start + 1] = free[start]
        free[-1] = rng.choice([-1, num_pages, -2 ** 31, max(table[0][0], 0)])
    _compact(table, lens, pinned, free, start, page, num_pages, "pinned")
    _compact(table, lens, None, free, start, page, num_pages, "free", module=capi)


def test_beams_share_their_prompt():
    # one prompt of 70 tokens on pages of 32, three beams: the lowest keeps the last page, two copies
    table, lens, copies, nxt = _fork([[4, 7, 2]], [70], [0, 0, 0], None, None, [-1, -1, -1, 9, 8, 6], 3, 32, 10, "three")
    assert table.tolist() == [[4, 7, 2], [4, 7, 9], [4, 7, 8]] and copies.tolist() == [[-1, -1, 0], [2, 9, 6], [2, 8, 6]]
    # beams 1 and 2 go on from 1, 0 ends: its last page (2) is freed and taken at once
    got = _fork(table.tolist(), lens.tolist(), [1, 1], None, None, [-1, -1, -1, 9, 8, 6], int(nxt), 32, 10, "reordered")
    assert got[0].tolist() == [[4, 7, 9], [4, 7, 2]] and int(got[3]) == 5 - 2 + 1


def test_drafts_rolled_back():
    # 100 tokens, of which 61 stay: the third and fourth pages go back
    got = _fork([[5, 3, 1, 0]], [100], [0], [61], None, [-1, -1, -1, -1, 2, 4], 4, 32, 6, "rolled back")
    assert got[0].tolist() == [[5, 3, -1, -1]] and int(got[3]) == 2
    # a page that another row holds whole is not written on: the row rolled back into it gets a copy
    got = _fork([[5, 3, 1], [5, 3, 0]], [96, 96], [0, 1], [40, 96], None, [-1, -1, -1, -1, 2, 4], 4, 32, 6, "into a shared page")
    assert got[0].tolist() == [[5, 1, -1], [5, 3, 0]] and got[2].tolist() == [[3, 1, 8], [-1, -1, 0]]


@pytest.mark.parametrize("free,start", [([], 0), ([7], 0), ([7], 1), ([7, 8], 2), ([-1] * 5, 5), ([3, 3], -4), ([1], 2 ** 31 - 1)])
def test_free_lists_that_end(free, start):
    table, lens = [[0, 1], [2, 3]], [33, 64]
    _fork(table, lens, [0, 0, 0], None, None, free, start, 32, 9, "copies")
    _fork(table, lens, [-1], None, None, free, start, 32, 9, "freed")
    _compact(table, lens, None, free, start, 32, 9, "compact")


def test_the_largest_pool():
    rng = random.Random(8)
    num_pages, width = 1 << 18, 1000
    order = list(range(num_pages))
    rng.shuffle(order)
    rows = 150
    table = [order[width * r:width * (r + 1)] for r in range(rows)]
    lens = [rng.randint(1, width * 32) for _ in range(rows)]
    free = [-1] * (width * rows) + order[width * rows:]
    pinned = [0] * num_pages
    pinned[-1] = pinned[0] = pinned[order[5]] = 1
    parents = [rng.randrange(rows) for _ in range(300)]
    _fork(table, lens, parents, None, pinned, free, width * rows, 32, num_pages, "largest")
    _compact(table, lens, pinned, free, width * rows, 32, num_pages, "largest")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn, torch.float32])
@pytest.mark.parametrize("layers,page", [(0, 32), (1, 64), (3, 128), (2, 2048)])
def test_copies(dtype, layers, page):
    rng = random.Random(page)
    pages = 12
    shape = (pages, page, 576) if layers == 0 else (layers, pages, page, 576)
    raw = torch.randint(0, 255, (*shape[:-1], 576 * dtype.itemsize), dtype=torch.uint8, device="cuda")
    cache = raw.clone().view(dtype)
    assert cache.shape == shape
    copies = [[3, 5, 1], [2, 0, page], [-1, 4, page], [4, -1, page], [pages, 6, 3], [6, pages, 3], [9, 9, page], [1, 7, 0],
              [1, 8, -4], [4, 10, page + 100], [11, 1, page - 1], [3, 6, rng.randint(1, page)], [2 ** 31 - 1, 2, 5]]
    ada_mla.mla_copy_pages(cache, _t(copies))
    want = raw.view(-1, pages, page, raw.shape[-1])
    new = want.clone()
    for s, d, n in copies:
        if 0 <= s < pages and 0 <= d < pages and s != d:
            n = min(max(n, 0), page)
            new[:, d, :n] = want[:, s, :n]
    assert torch.equal(cache.view(torch.uint8).view(new.shape), new)
    ada_mla.mla_copy_pages(cache, _t(copies)[:0])  # none
    ada_mla.mla_copy_pages(cache, _t(copies).t().contiguous().t())  # strided, and again: nothing changes
    assert torch.equal(cache.view(torch.uint8).view(new.shape), new)


def test_copies_past_2_31_bytes():
    pages, page = 40000, 64
    cache = torch.zeros(2, pages, page, 576, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    raw = cache.view(torch.uint8)
    raw[:, pages - 1] = torch.randint(0, 255, (2, page, 576), dtype=torch.uint8, device="cuda")
    ada_mla.mla_copy_pages(cache, _t([[pages - 1, pages - 2, 40], [pages - 1, 3, page]]))
    assert torch.equal(raw[:, 3], raw[:, pages - 1])
    assert torch.equal(raw[:, pages - 2, :40], raw[:, pages - 1, :40]) and not raw[:, pages - 2, 40:].any()


def test_replays_of_captured_tables():
    rng = random.Random(3)
    page, num_pages = 32, 500
    table, lens, free, start, pinned = random_pool(rng, 40, 12, page, num_pages)
    tt, ll, ff, ss, pp = _t(table), _t(lens), _t(free), _t([start]), _t(pinned)
    parents, list_t = _t([0] * 30), ff.clone()
    cache = torch.randint(0, 255, (num_pages, page, 576), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)

    def call():
        a = ada_mla.mla_fork_tables(tt, ll, parents, list_t, ss, page, num_pages, pinned=pp)
        ada_mla.mla_copy_pages(cache, a[2])
        b = ada_mla.mla_compact_tables(a[0], a[1], list_t, a[3], page, num_pages, pinned=pp)
        return [*a, *b]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    list_t.copy_(ff)
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        new = [rng.randrange(-1, 41) for _ in range(30)]
        parents.copy_(_t(new))
        list_t.copy_(ff)
        before = cache.view(torch.uint8).clone()
        graph.replay()
        want = fork(table, lens, new, [2 ** 31 - 1] * 30, pinned, free, start, page, num_pages)
        assert [t.tolist() for t in out[:4]] == [want[0], want[1], want[2], [want[3]]], k
        assert list_t.tolist() == want[4]
        then = compact(want[0], want[1], pinned, want[4], want[3], page, num_pages)
        assert [t.tolist() for t in out[4:]] == list(then), k
        for s, d, n in want[2]:
            if d >= 0:
                before[d, :n] = before[s, :n]
        assert torch.equal(cache.view(torch.uint8), before), k


def test_other_streams_and_strided_inputs():
    rng = random.Random(6)
    table, lens, free, start, _ = random_pool(rng, 20, 10, 32, 200)
    wide = torch.full((20, 25), 77, **I32)
    wide[:, 3:13] = _t(table)
    lens2 = torch.stack([_t(lens), _t(lens)], 1)[:, 1]
    parents = [rng.randrange(20) for _ in range(9)]
    want = fork(table, lens, parents, [2 ** 31 - 1] * 9, [0] * 200, free, start, 32, 200)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        free_t = _t(free)
        got = ada_mla.mla_fork_tables(wide[:, 3:13], lens2, _t(parents), free_t, _t([start]), 32, 200)
        assert [t.tolist() for t in got] == [want[0], want[1], want[2], [want[3]]] and free_t.tolist() == want[4]
