"""Serving in 8 bits on shared pages, as it is used: projections in fp8, prompts into an fp8 cache, beams forked from
them, reordered, rolled back and ended between decode steps, the pool compacted; each step's attention
against float64 over the history that the beam ought to have."""
import random

import pytest
import torch

import ada_mla
from test_gpu_linear_fp8 import _check as check_linear, _quantised, _weight
from test_gpu_paged_fp8 import _check as check_decode

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")
HEADS, PAGE, HIDDEN, LAYERS, SCALE8 = 16, 32, 272, 2, 0.0625


class _Server:
    def __init__(self, dtype, pages, columns, seed):
        self.gen = torch.Generator()
        self.gen.manual_seed(seed)
        self.dtype, self.pages = dtype, pages
        self.cache = torch.full((LAYERS, pages, PAGE, 576), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        self.free = torch.randperm(pages, generator=self.gen).int().cuda()
        self.start = torch.zeros(1, **I32)
        self.columns = columns
        self.w_kv = [_weight(self.gen, 576, HIDDEN) for _ in range(LAYERS)]
        self.w_q = [_weight(self.gen, HEADS * 576, HIDDEN) for _ in range(LAYERS)]
        self.norm = torch.ones(512, dtype=dtype, device="cuda")
        angle = torch.arange(1024.0)[:, None] * 10000.0 ** (-torch.arange(32) / 32)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).cuda()

    def admit(self, lengths):
        self.table = torch.full((len(lengths), self.columns), -1, **I32)
        self.lens = torch.zeros(len(lengths), **I32)
        self.history = [[torch.zeros(0, 576, dtype=torch.float64) for _ in lengths] for _ in range(LAYERS)]
        return self.step(lengths, decode=False)

    def step(self, new, decode=True):
        """`new` tokens a row through every layer; checks projections, and the attention of the last tokens."""
        total = sum(new)
        cu, cu_new, slots, positions, self.start = ada_mla.mla_paged_tables(
            self.lens, torch.tensor(new, **I32), self.table, self.free, self.start, PAGE, total)
        outs = []
        for layer in range(LAYERS):
            hidden = (torch.randn(total, HIDDEN, generator=self.gen) * 1.6).to(self.dtype)
            xq, x_scale = ada_mla.mla_quantize_fp8(hidden.cuda())
            w, ws = self.w_kv[layer]
            kv = ada_mla.mla_linear_fp8(xq, w.cuda(), ws.cuda(), x_scale=x_scale, dtype=self.dtype)
            check_linear(kv, *_quantised(hidden), w, ws, self.dtype, f"kv of layer {layer}")
            ada_mla.mla_append_kv(kv, self.norm, self.cos_sin, positions, slots, self.cache[layer], cache_scale=SCALE8)
            rows = self.cache[layer].view(-1, 576)[slots].double().cpu() * SCALE8
            assert torch.isfinite(rows).all()
            at = 0
            for b, n in enumerate(new):
                self.history[layer][b] = torch.cat([self.history[layer][b], rows[at:at + n]])
                at += n
            if decode:
                w, ws = self.w_q[layer]
                q = ada_mla.mla_linear_fp8(hidden.cuda(), w.cuda(), ws.cuda()).view(total, HEADS, 576)
                outs.append(self.attend(layer, q, cu))
        self.lens = self.lens + torch.tensor(new, **I32)
        return outs

    def attend(self, layer, q, cu):
        out = ada_mla.mla_decode_paged(q, self.cache[layer], self.table, cu, cache_scale=SCALE8)
        check_decode(out, q, self.history[layer], self.dtype, f"layer {layer}")
        return out

    def fork(self, parents, kept=None, pinned=None):
        held = self.lens.tolist()
        self.table, self.lens, copies, self.start = ada_mla.mla_fork_tables(
            self.table, self.lens, torch.tensor(parents, **I32), self.free, self.start, PAGE, self.pages,
            kept_lens=None if kept is None else torch.tensor(kept, **I32), pinned=pinned)
        ada_mla.mla_copy_pages(self.cache, copies)
        kept = [held[p] if p >= 0 else 0 for p in parents] if kept is None else kept
        self.history = [[h[p][:n] if p >= 0 else h[0][:0] for p, n in zip(parents, kept)] for h in self.history]
        assert self.lens.tolist() == [h.shape[0] for h in self.history[0]]
        self.check_pool(pinned)

    def check_pool(self, pinned=None):
        """Every page is held by a row, free or pinned, and no page is both held and free."""
        held = {i for row, n in zip(self.table.tolist(), self.lens.tolist()) for i in row[: -(-n // PAGE)]}
        free = self.free.tolist()[int(self.start):]
        fixed = set() if pinned is None else set(pinned.nonzero()[:, 0].tolist())
        assert len(free) == len(set(free)) and not held & set(free)
        assert held | set(free) | fixed == set(range(self.pages)), "a page was lost"

    def compact(self):
        used = len({i for row, n in zip(self.table.tolist(), self.lens.tolist()) for i in row[: -(-n // PAGE)]})
        self.table, copies, self.free = ada_mla.mla_compact_tables(self.table, self.lens, self.free, self.start, PAGE, self.pages)
        ada_mla.mla_copy_pages(self.cache, copies)
        assert max(i for row in self.table.tolist() for i in row) == used - 1
        self.check_pool()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_beams(dtype):
    rng = random.Random(1)
    s = _Server(dtype, 60, 8, 1)
    s.admit([70, 33, 1])
    s.fork([r for r in range(3) for _ in range(4)])  # four beams of each prompt
    for i in range(6):
        s.step([1] * 12)
        s.fork([4 * (b // 4) + rng.randrange(4) for b in range(12)])
    # drafts: five more tokens each, of which some stay
    s.step([5] * 12, decode=False)
    lens = s.lens.tolist()
    s.fork(list(range(12)), [n - rng.randint(0, 5) for n in lens])
    s.step([1] * 12)
    # two of the requests end; the pool is tidied up, and what the others compute does not change
    s.fork([0, 1, 2, 3, -1, -1], [int(n) for n in s.lens[:4]] + [0, 0])
    cu = torch.cat([torch.zeros(1, **I32), s.lens.cumsum(0).int()])
    q = torch.randn(6, HEADS, 576, generator=s.gen).to(dtype).cuda()
    before = [s.attend(layer, q, cu) for layer in range(LAYERS)]
    s.compact()
    assert all(torch.equal(s.attend(layer, q, cu), x) for layer, x in enumerate(before))
    s.step([1, 1, 1, 1, 40, 1], decode=False)
    s.step([1] * 6)


def test_a_pinned_prompt_outlives_its_requests():
    s = _Server(torch.bfloat16, 40, 6, 2)
    s.admit([77])
    pinned = torch.zeros(s.pages, **I32)
    pinned[s.table[0, :3].long()] = 1
    prompt, row, n = s.table.clone(), [h[0] for h in s.history], s.lens.clone()
    s.fork([0, 0], pinned=pinned)  # the last page is pinned: both beams get a copy
    assert not {int(s.table[0, 2]), int(s.table[1, 2])} & {int(prompt[0, 2])}
    s.step([1, 1])
    s.fork([-1, -1], [0, 0], pinned=pinned)  # both end; the prompt stays
    s.table, s.lens, s.history = prompt, n, [[h] for h in row]
    s.fork([0, 0, 0], pinned=pinned)
    s.step([1, 30, 2], decode=False)
    s.step([1] * 3)
