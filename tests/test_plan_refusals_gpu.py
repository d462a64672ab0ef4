"""A request that the cache step refuses keeps its state, the blocks it holds among it, whatever the reason."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.serving import PagedCache

pytestmark = pytest.mark.gpu


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("ctx,cu,tokens,held,admitted,after", [
    ([-4, 5], [0, 2, 3], 3, [3, 1], [False, True], [3, 1]),        # a negative length
    ([4, 5], [0, 9, 3], 3, [2, 3], [False, False], [2, 3]),        # offsets that run back
    ([4, 5, 6], [0, 1, 4, 8], 6, [1, 2, 4], [True, True, False], [1, 2, 4]),  # more tokens than the call is given
    ([4, 5], [-2, 1, 2], 2, [2, 1], [False, True], [2, 1]),        # an offset before the first token
    ([2 ** 31 - 1, 5], [0, 1, 2], 2, [4, 1], [False, True], [4, 1]),  # a length past 32 bits with its token
])
def test_unsound_lengths_keep_their_blocks(cuda, ctx, cu, tokens, held, admitted, after):
    n = len(ctx)
    table = torch.arange(4 * n, dtype=torch.int32, device=cuda).view(n, 4)
    before = table.clone()
    got = fa.plan_cache_step(ints(ctx, cuda), ints(cu, cuda), table, ints(held, cuda), ints([90, 91], cuda),
                             ints([2], cuda), tokens, 16)
    assert fa.device_error() == 2
    assert got[2].tolist() == admitted and got[4].tolist() == after
    assert torch.equal(table, before) and got[3].tolist() == [2]


def test_no_block_is_lost(cuda):
    """PagedCache with too small a number of tokens for its offsets: what is released afterwards is what was held."""
    cache = PagedCache(2, 10, 16, 1, 64, 8, device=cuda)
    step = cache.plan(ints([0, 40, 60], cuda), 60)
    cache.commit(step, ints([10, 20], cuda))  # drafted blocks stay held: 3 blocks for 10 tokens
    cache.plan(ints([0, 4, 8], cuda), 3)
    assert fa.device_error() == 2
    assert cache.held_blocks.tolist() == [3, 2]
    cache.release(0)
    cache.release(1)
    assert cache.num_free.tolist() == [10] and sorted(cache.free_blocks.tolist()) == list(range(10))
