"""The cache step (block table, slots, positions, tree masks) against a request-by-request statement: whole numbers,
equal."""
import random

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu


def ints(x, device, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=device)


def state(rng, requests, context, tokens, page, spare_held=False, cols_spare=0):
    ctx = [rng.randint(0, context) for _ in range(requests)]
    new = [rng.randint(0, tokens) for _ in range(requests)]
    held = [-(-c // page) + (rng.randint(0, 2) if spare_held else 0) for c in ctx]
    want = [max(h, -(-(c + t) // page)) for h, c, t in zip(held, ctx, new)]
    cols = max(want + [1]) + cols_spare
    order = list(range(sum(want) + 5))
    rng.shuffle(order)
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [0] * (cols - h))
        at += h
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    return ctx, cu, table, held, order[at:]


def check(cuda, ctx, cu, table, held, free, num_free, tokens, page, parents=None, words=0):
    want = orc.plan(ctx, cu, table, held, free, num_free, tokens, page, parents, words)
    t = ints(table, cuda)
    got = fa.plan_cache_step(ints(ctx, cuda), ints(cu, cuda), t, ints(held, cuda), ints(free, cuda),
                             ints([num_free], cuda), tokens, page,
                             parents=None if parents is None else ints(parents, cuda), mask_words=words)
    slots, positions, admitted, left, held_after, mask = got
    assert t.tolist() == want[0]
    assert slots.tolist() == want[1]
    assert positions.tolist() == want[2]
    assert admitted.tolist() == want[3]
    assert left.tolist() == [want[4]]
    assert held_after.tolist() == want[5]
    if parents is not None:
        assert [[w & 0xFFFFFFFF for w in r] for r in mask.tolist()] == want[6]
    else:
        assert mask is None
    assert fa.device_error() == 0


@pytest.mark.parametrize("requests,context,tokens,page", [(1, 0, 1, 16), (1, 16, 1, 16), (1, 15, 1, 16), (7, 100, 1, 8),
                                                           (33, 300, 40, 16), (300, 50, 9, 1), (700, 100, 3, 32),
                                                           (2, 5000, 3000, 128), (5, 10, 0, 16), (2049, 40, 2, 16)])
@pytest.mark.parametrize("spare_held", [False, True])
def test_chain(cuda, requests, context, tokens, page, spare_held):
    rng = random.Random(requests * 1000 + tokens)
    ctx, cu, table, held, free = state(rng, requests, context, tokens, page, spare_held)
    check(cuda, ctx, cu, table, held, free, len(free), cu[-1], page)
    check(cuda, ctx, cu, table, held, free, len(free), cu[-1] + 3, page)  # padding rows past the last request


@pytest.mark.parametrize("share", [0.0, 0.3, 0.7, 0.95])
def test_refused_requests(cuda, share):
    """Too few free blocks: requests in order, the refused ones unchanged."""
    rng = random.Random(5)
    ctx, cu, table, held, free = state(rng, 60, 200, 50, 16)
    check(cuda, ctx, cu, table, held, free, int(share * len(free)), cu[-1], 16)


def test_row_too_short(cuda):
    """A request whose blocks exceed its row is refused and takes none."""
    ctx, cu, held, free = [20, 3, 30], [0, 30, 32, 34], [2, 1, 2], [9, 8, 7, 6, 5]
    table = [[0, 1, 0], [2, 0, 0], [3, 4, 0]]
    check(cuda, ctx, cu, table, held, free, 5, 34, 16)


def random_tree(rng, n, kind):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] * n
    return [rng.randint(-1, i - 1) for i in range(n)]


@pytest.mark.parametrize("kind", ["chain", "star", "random"])
@pytest.mark.parametrize("nodes,words", [(1, 1), (31, 1), (32, 1), (33, 2), (64, 2), (61, 3), (200, 7)])
def test_trees(cuda, kind, nodes, words):
    rng = random.Random(nodes)
    ctx, cu, table, held, free = state(rng, 9, 70, nodes, 16)
    new = [b - a for a, b in zip(cu, cu[1:])]
    new[0], cu = nodes, [0]
    for t in new:
        cu.append(cu[-1] + t)
    cols = max(-(-(c + t) // 16) for c, t in zip(ctx, new))
    table = [(r + [0] * cols)[:max(cols, len(r))] for r in table]
    width = max(map(len, table))
    table = [r + [0] * (width - len(r)) for r in table]
    free = list(range(1000, 1000 + 9 * (nodes // 16 + 2)))
    parents = sum((random_tree(rng, t, kind) for t in new), [])
    check(cuda, ctx, cu, table, held, free, len(free), cu[-1], 16, parents, words)


def test_malformed_trees_and_lengths_are_recorded(cuda):
    """A parent that is no earlier token counts as a root; a node past the mask's words gets none; a negative length
    is refused. All are recorded, none is followed."""
    args = lambda ctx, cu: (ints(ctx, cuda), ints(cu, cuda), ints([[0, 1]] * len(ctx), cuda),  # noqa: E731
                            ints([1] * len(ctx), cuda), ints([2, 3], cuda), ints([2], cuda))
    got = fa.plan_cache_step(*args([3], [0, 3]), 3, 16, parents=ints([-1, 1, 7], cuda), mask_words=1)
    assert fa.device_error() == 2
    assert got[5].flatten().tolist() == [1, 2, 4] and got[1].tolist() == [3, 3, 3]
    got = fa.plan_cache_step(*args([3], [0, 34]), 34, 64, parents=ints(list(range(-1, 33)), cuda), mask_words=1)
    assert fa.device_error() == 2
    assert got[5].flatten().tolist()[32:] == [0, 0]
    got = fa.plan_cache_step(*args([-4, 5], [0, 2, 3]), 3, 16)
    assert fa.device_error() == 2
    assert got[0].tolist() == [-1, -1, 5] and got[2].tolist() == [False, True]
    got = fa.plan_cache_step(*args([4, 5], [0, 9, 3]), 3, 16)
    assert fa.device_error() == 2 and got[2].tolist() == [False, False]


def test_no_requests_and_no_tokens(cuda):
    none = ints([], cuda)
    got = fa.plan_cache_step(none, ints([0], cuda), torch.empty(0, 4, dtype=torch.int32, device=cuda), none,
                             ints([4], cuda), ints([1], cuda), 0, 16)
    assert got[3].tolist() == [1] and got[0].numel() == 0
    got = fa.plan_cache_step(none, ints([0], cuda), torch.empty(0, 4, dtype=torch.int32, device=cuda), none,
                             ints([4], cuda), ints([1], cuda), 5, 16)
    assert got[0].tolist() == [-1] * 5 and got[1].tolist() == [0] * 5


def test_table_of_wider_rows(cuda):
    """A block table that is a slice of a wider one keeps the columns beside it."""
    wide = torch.full((3, 9), 77, dtype=torch.int32, device=cuda)
    table = wide[:, 2:6]
    table[:] = 0
    fa.plan_cache_step(ints([0, 5, 0], cuda), ints([0, 20, 21, 21], cuda), table, ints([0, 1, 0], cuda),
                       ints([10, 11, 12, 13], cuda), ints([4], cuda), 21, 16)
    assert table.tolist() == [[13, 12, 0, 0], [0, 0, 0, 0], [0, 0, 0, 0]]
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 6:] == 77).all())
