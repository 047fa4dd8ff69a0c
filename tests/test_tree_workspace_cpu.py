"""Workspaces of the drafted trees: partials are reserved for the requests that can be
split and for no others, and the numbering of their slots holds for any lengths."""
import random

from ada_mla import capi

TILE = 128 * (512 + 2) * 4  # bytes of the partials of 128 rows: O, maxima, sums


def _size(*a):
    return capi.load().mla_decode_tree_workspace_size(*a)


def test_calls_that_cannot_be_split_need_next_to_nothing():
    # the rows fill the chip, and no request can be longer than the call's tokens
    for batch, drafts, heads, total in ((64, 64, 128, 1000), (64, 64, 128, 0), (300, 16, 128, 1024), (1, 64, 4096, 1000)):
        assert 0 < _size(batch, drafts, heads, total, 0) <= 4096, (batch, drafts, heads, total)


def test_short_requests_reserve_for_the_long_ones_only():
    # 256 requests of 100 tokens on average: those past 1024 tokens have two part slots for each
    # 1024 of all the tokens, whatever the batch
    batch, drafts, heads, total = 256, 32, 128, 25600
    slots, row_tiles = 2 * total // 1024, drafts * heads // 128
    assert _size(batch, drafts, heads, total, 0) <= slots * row_tiles * TILE + 4096
    assert _size(2 * batch, drafts, heads, total, 0) == _size(batch, drafts, heads, total, 0)


def test_long_requests_keep_a_slot_a_split():
    # one request in n splits: n + 1 part slots at most
    for n in (2, 5, 16):
        assert _size(1, 8, 16, 32 * 64, n) <= (n + 1) * TILE + 4096


def _slots(lengths, chunk, pairs):
    """The part slots of each request that has several splits, as the kernels number them."""
    lo, out = 0, []
    for b, n in enumerate(lengths):
        splits = -(-n // chunk)
        if splits > 1:
            first = 2 * lo // chunk if pairs else lo // chunk + b
            out.append(range(first, first + splits))
        lo += n
    return out


def test_part_slots_are_disjoint_and_in_bounds():
    rng = random.Random(1)
    for _ in range(4000):
        chunk = 32 * rng.randint(1, 8)
        lengths = [rng.choice([0, 1, chunk, chunk + 1, 2 * chunk, 2 * chunk + 1, rng.randint(0, 9 * chunk)])
                   for _ in range(rng.randint(1, 12))]
        total = sum(lengths) + rng.choice([0, 0, rng.randint(0, 3 * chunk)])
        for pairs, most in ((False, total // chunk + len(lengths)), (True, 2 * total // chunk)):
            taken = [s for r in _slots(lengths, chunk, pairs) for s in r]
            assert len(taken) == len(set(taken)) and all(0 <= s < most for s in taken), (lengths, chunk, pairs)
