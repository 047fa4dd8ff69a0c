"""The operators of a serving loop one after another, as they are used:
prompts admitted (tables, cache rows, prefill), a decode step, a step of
drafted tokens, each against float64 over the whole history of rows."""
import random

import pytest
import torch

import ada_mla
from operators_reference import attention_check, chain_mask, half_step, latent_rows, random_tree, rotate, signed

pytestmark = pytest.mark.gpu

HEADS, PAGE, EPS = 16, 32, 1e-6


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_prompts_then_steps(dtype, interleaved):
    rng = random.Random(1)
    gen = torch.Generator()
    gen.manual_seed(1)
    batch = 3
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((batch, 12), -1, **i32)
    free = torch.randperm(40, generator=gen).int().cuda()
    start = torch.zeros(1, **i32)
    cache = torch.full((40, PAGE, 576), float("nan"), dtype=dtype, device="cuda")
    w = (1 + 0.2 * torch.randn(512, generator=gen)).to(dtype)
    uk, uv = ((torch.randn(HEADS, 128, 512, generator=gen) * 512 ** -0.5).to(dtype) for _ in range(2))
    i = torch.arange(32, dtype=torch.float64)
    angle = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-i / 32)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float()
    history = [torch.zeros(0, 576, dtype=torch.float64) for _ in range(batch)]  # the rounded rows of each request
    u = half_step(dtype)

    def step(new):
        """Appends `new` tokens a request; -> rotated queries' parts, prefix sums, each token's request."""
        nonlocal start
        have = [h.shape[0] for h in history]
        total = sum(new)
        cu, cu_new, slots, positions, nxt = ada_mla.mla_paged_tables(
            torch.tensor(have, **i32), torch.tensor(new, **i32), table, free, start, PAGE, total)
        start = nxt
        kv = torch.randn(total, 576, generator=gen).to(dtype)
        q_nope = torch.randn(total, HEADS, 128, generator=gen).to(dtype)
        q_rope = torch.randn(total, HEADS, 64, generator=gen).to(dtype)
        turned = ada_mla.mla_append_kv(kv.cuda(), w.cuda(), cs.cuda(), positions, slots, cache, q_rope=q_rope.cuda(),
                                       eps=EPS, interleaved=interleaved)
        assert cu.tolist() == [0] + torch.tensor([a + b for a, b in zip(have, new)]).cumsum(0).tolist()
        # what was written, to the rounding; the attention below is checked on the written values
        pos = torch.cat([torch.arange(a, a + b) for a, b in zip(have, new)])
        c, s = cs[pos][:, :32].double(), cs[pos][:, 32:].double()
        rows = cache.view(-1, 576)[slots].double().cpu()
        ref = latent_rows(kv, w, c, s, EPS, interleaved)
        assert ((rows - ref).abs() <= 1.01 * u * ref.abs() + 2.0 ** -14 * ref.abs() + 1e-5).all()
        want = rotate(q_rope.double(), c[:, None], s[:, None], interleaved)
        assert ((turned.double().cpu() - want).abs() <= 1.01 * u * want.abs() + 1e-5).all()
        at = 0
        for b, k in enumerate(new):
            history[b] = torch.cat([history[b], rows[at:at + k]])
            at += k
        return q_nope.cuda(), turned, cu, cu_new

    # prompts, the second chunked in two
    for new in ([70, 33, 1], [0, 50, 64]):
        q_nope, q_rope, cu, cu_new = step(new)
        out = ada_mla.mla_prefill(q_nope, q_rope, uk.cuda(), uv.cuda(), cache, cu_new, cu, block_table=table)
        at = 0
        for b, m in enumerate(new):
            c, n = history[b], history[b].shape[0]
            seen = torch.arange(n)[None] <= torch.arange(m)[:, None] + n - m
            for h in range(HEADS):
                k = torch.cat([c[:, :512] @ uk[h].double().T, c[:, 512:]], 1)
                q = torch.cat([q_nope[at:at + m, h], q_rope[at:at + m, h]], 1).double().cpu()
                attention_check(out[at:at + m, h].cpu(), q, k, c[:, :512] @ uv[h].double().T, seen, dtype, True,
                                f"prompt {b} head {h}")
            at += m
    # one token a request, by the paged decode
    q_nope, q_rope, cu, _ = step([1, 1, 1])
    q = ada_mla.mla_absorb_query(q_nope, q_rope, uk.cuda())
    one = ada_mla.mla_decode_paged(q, cache, table, cu)
    tree = ada_mla.mla_decode_tree(q[:, None].contiguous(), cache, table, cu, torch.ones(3, 1, dtype=torch.int64).cuda())
    most = max(h.abs().max().item() for h in history)
    assert (one.float() - tree[:, 0].float()).abs().max() <= 6 * u * most
    # drafted trees
    m = 5
    masks = [random_tree(rng, m), chain_mask(m), random_tree(rng, m)]
    q_nope, q_rope, cu, _ = step([m] * 3)
    q = ada_mla.mla_absorb_query(q_nope, q_rope, uk.cuda()).view(3, m, HEADS, 576)
    out = ada_mla.mla_decode_tree(q, cache, table, cu, torch.tensor([signed(x) for x in masks]).cuda())
    for b in range(3):
        c, n = history[b], history[b].shape[0]
        for i in range(m):
            seen = torch.ones(1, n, dtype=torch.bool)
            for j in range(m):
                seen[0, n - m + j] = bool(masks[b][i] >> j & 1)
            attention_check(out[b, i].cpu(), q[b, i].double().cpu(), c, c[:, :512], seen.expand(HEADS, n), dtype,
                            what=f"tree {b} draft {i}")
    assert int(start) == sum(-(-h.shape[0] // PAGE) for h in history)
