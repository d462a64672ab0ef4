"""Requests that a step refuses: their rows see no key of anyone, nothing about them counts as an index out of range,
and the other requests' results are what they would be alone."""
import random

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.rotary import rotary_table
from flashlite_b200.serving import PagedCache

from test_tree_attention_gpu import Case

pytestmark = pytest.mark.gpu


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def step_of(cuda, heads, kv_heads, dim, new, num_blocks, max_blocks, positions, layout="bnhd", tree=False, seed=5):
    """Two requests with 20 and 3 cached tokens, then a step with `new` tokens of each: (step, out, device error, state)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    table = rotary_table(positions, dim, device=cuda)
    cache = PagedCache(2, num_blocks, 16, kv_heads, dim, max_blocks, layout=layout, device=cuda)
    draw = lambda n: torch.randn(n, heads + 2 * kv_heads, dim, generator=g, device=cuda).half()  # noqa: E731
    split = lambda x: x.split([heads, kv_heads, kv_heads], 1)  # noqa: E731
    first = cache.plan(ints([0, 20, 23], cuda), 23)
    cache.attend(0, *split(draw(23)), table, first)
    cache.commit(first, ints([20, 3], cuda))
    assert first.admitted.all() and fa.device_error() == 0
    rows = draw(60)  # the same tokens for a request whatever the other one has
    x = torch.cat([rows[:new[0]], rows[50:50 + new[1]]])
    more = dict(parents=ints([i - 1 for n in new for i in range(n)], cuda), mask_words=2) if tree else {}
    step = cache.plan(ints([0, new[0], sum(new)], cuda), sum(new), **more)
    out = cache.attend(0, *split(x), table, step)
    return step, out, fa.device_error(), cache


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("layout", ["bnhd", "bhnd"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (2, 2, 128), (8, 1, 64), (8, 2, 128)])
def test_row_too_short(cuda, heads, kv_heads, dim, layout, tree):
    """50 tokens where a row has room for 48: the step's positions reach past the rotary table too."""
    step, out, error, cache = step_of(cuda, heads, kv_heads, dim, (30, 2), 20, 3, 48, layout, tree)
    assert step.admitted.tolist() == [False, True] and error == 0
    assert bool((out[:30] == 0).all())
    _, alone, _, _ = step_of(cuda, heads, kv_heads, dim, (0, 2), 20, 3, 48, layout, tree)
    # the other kernel may have run: probabilities and results rounded to fp16 by each
    assert float((out[30:] - alone).abs().max()) <= 4 * 4 * 2.0 ** -11 and bool((out[30:] != 0).any())
    cache.commit(step, ints([30, 2], cuda))
    assert cache.context_lens.tolist() == [20, 5] and cache.held_blocks.tolist() == [2, 1]


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (8, 1, 128)])
def test_no_free_blocks(cuda, heads, kv_heads, dim):
    """The refused request's row names no blocks for its new tokens: zeros, which are another request's block."""
    step, out, error, _ = step_of(cuda, heads, kv_heads, dim, (30, 2), 4, 8, 64)
    assert step.admitted.tolist() == [False, True] and error == 0
    assert bool((out[:30] == 0).all()) and bool((out[30:] != 0).any())


@pytest.mark.parametrize("words", [0, 2])
@pytest.mark.parametrize("requests,heads,kv_heads,tokens", [(3, 2, 1, 4), (90, 4, 2, 3), (3, 8, 1, 20), (40, 16, 8, 20),
                                                             (700, 4, 2, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_requests_that_take_no_part(cuda, requests, heads, kv_heads, tokens, dim, words):
    """A length of -1: rows of 0 and -inf and no report, whatever the table's row holds; other rows keep their bits
    where nothing but that changes how they are divided, and their values within rounding otherwise."""
    rng = random.Random(requests)
    c = Case(cuda, [(rng.choice([0, 3, 200, 700]), rng.randint(1, tokens)) for _ in range(requests)], heads, kv_heads, dim,
             16, words=words, seed=requests)
    want, wlse = c.run()
    assert fa.device_error() == 0
    out_of = [b for b in range(requests) if b % 3 == 1]
    for b in out_of:
        c.context[b] = -1
        c.table[b] = [-7] * len(c.table[b])
    out, lse = c.run()
    assert fa.device_error() == 0
    gone = torch.zeros(c.cu[-1], dtype=torch.bool, device=cuda)
    for b in out_of:
        gone[c.cu[b]:c.cu[b + 1]] = True
    assert bool((out[gone] == 0).all()) and bool((lse[gone] == -float("inf")).all())
    live = ~gone
    # values of order 4 at most, rounded twice by either run; log-sum-exps held to 2^-20 (1 + R + |lse|) by either, R < 30
    assert float((out - want)[live].abs().max()) <= 4 * 4 * 2.0 ** -11
    seen = wlse[live] > -float("inf")
    assert torch.equal(lse[live] > -float("inf"), seen)
    assert float((lse - wlse)[live][seen].abs().max()) <= 2.0 ** -14


def test_other_negative_lengths_are_recorded(cuda):
    c = Case(cuda, [(30, 1), (10, 1)], 2, 1, 64, 16)
    c.context[0] = -2
    c.run()
    assert fa.device_error() == 2
