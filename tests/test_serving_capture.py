"""A serving step through PagedCache, captured once and replayed: the cache goes on from replay to replay."""
import pytest
import torch

import flashlite_b200.serving
from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.serving import PagedCache


@pytest.mark.parametrize("inference", [False, True])
def test_state_stays_where_it_is(monkeypatch, inference):
    """Whatever a step returns, the state that the next one reads lies at the same addresses, and it can be written
    whether or not the cache was made in inference mode."""

    def plan(context_lens, cu, table, held, free, num_free, total, page, parents=None, mask_words=0):
        n = context_lens.numel()
        return (torch.zeros(total, dtype=torch.long), torch.zeros(total, dtype=torch.int32),
                torch.ones(n, dtype=torch.bool), num_free - n, held + 1, None)

    def settle(context_lens, held, num_free, admitted, held_after, free_after):
        held.copy_(held_after)
        num_free.copy_(free_after)
        return torch.where(admitted, context_lens, -1)

    monkeypatch.setattr(flashlite_b200.serving, "plan_cache_step", plan)
    monkeypatch.setattr(flashlite_b200.serving, "settle_step", settle, raising=False)
    with torch.inference_mode(inference):
        cache = PagedCache(2, 8, 16, 1, 64, 4, device="cpu")
    state = lambda: (cache.context_lens, cache.held_blocks, cache.num_free, cache.free_blocks, cache.block_table)  # noqa: E731
    where = [x.data_ptr() for x in state()]
    for n in (1, 2):
        step = cache.plan(torch.tensor([0, 3, 4], dtype=torch.int32), 4)
        cache.commit(step, torch.tensor([3, 1]))
        assert cache.num_free.tolist() == [8 - 2 * n] and cache.held_blocks.tolist() == [n, n]
        assert cache.context_lens.tolist() == [3 * n, n]
        assert [x.data_ptr() for x in state()] == where
    cache.release(0)
    assert cache.num_free.tolist() == [6] and cache.context_lens.tolist() == [0, 2]
    assert [x.data_ptr() for x in state()] == where


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (128, 8, 1)])
def test_replayed_steps_agree_with_eager_ones(cuda, tree, dim, heads, kv_heads):
    from flashlite_b200.rotary import rotary_table

    requests, page, nodes, steps = 3, 16, 5 if tree else 1, 40
    g = torch.Generator(device=cuda).manual_seed(4)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table = rotary_table(512, dim, device=cuda)
    fill = torch.randn(66, heads + 2 * kv_heads, dim, generator=g, device=cuda).half()
    inputs = torch.randn(steps, requests * nodes, heads + 2 * kv_heads, dim, generator=g, device=cuda).half()
    more = dict(parents=ints([-1, 0, 0, 1, 3] * requests), mask_words=1) if tree else {}
    cu, kept = ints([nodes * b for b in range(requests + 1)]), ints([3, 1, 2] if tree else [1, 1, 1])
    path = ints([[0, 1, 3], [0, 0, 0], [0, 2, 0]]) if tree else None

    def start():
        cache = PagedCache(requests, 40, page, kv_heads, dim, 16, layers=2, device=cuda)
        step = cache.plan(ints([0, 20, 65, 66]), 66)
        for layer in range(2):
            cache.attend(layer, *fill.split([heads, kv_heads, kv_heads], 1), table, step)
        cache.commit(step, ints([20, 45, 1]))
        return cache

    def once(cache, x):
        step = cache.plan(cu, requests * nodes, **more)
        outs = [cache.attend(layer, *x.split([heads, kv_heads, kv_heads], 1), table, step) for layer in range(2)]
        cache.commit(step, kept, path)
        return outs

    eager, captured = start(), start()
    buffer = inputs[0].clone()
    once(start(), buffer)  # warm-up, on a cache of its own
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        outs = once(captured, buffer)
    torch.cuda.current_stream().wait_stream(side)
    for x in inputs:
        want = once(eager, x)
        buffer.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        for name in ("context_lens", "held_blocks", "num_free", "block_table"):
            assert torch.equal(getattr(captured, name), getattr(eager, name)), name
    assert int(eager.context_lens[0]) == 20 + steps * int(kept[0])
    assert fa.device_error() == 0
