"""Offsets out of order: requests whose own are sound get their slots and positions all the same."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa

pytestmark = pytest.mark.gpu


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("cu,tokens,sound", [
    ([0, 9, 3, 5], 5, [False, False, True]),
    ([0, 2, 100, 4, 6], 6, [True, False, False, True]),
    ([7, 0, 2, -1, 2, 5], 6, [False, True, False, False, True]),
    ([0, 1, 2, 50], 4, [True, True, False]),
    ([0] + [3 * b for b in range(1, 301)], 900, [True] * 300),
    ([0] + [3 * b if b != 150 else 10 ** 6 for b in range(1, 301)], 900, [b not in (149, 150) for b in range(300)]),
])
def test_sound_requests_beside_unsound_ones(cuda, cu, tokens, sound, tree):
    n, page = len(cu) - 1, 16
    ctx = [5 + b % 40 for b in range(n)]
    held = [4] * n
    table = torch.arange(4 * n, dtype=torch.int32, device=cuda).view(n, 4)
    parents = ints([-1] * tokens, cuda) if tree else None
    slots, positions, admitted, left, _, mask = fa.plan_cache_step(
        ints(ctx, cuda), ints(cu, cuda), table, ints(held, cuda), ints([4 * n], cuda), ints([1], cuda), tokens, page,
        parents=parents, mask_words=1 if tree else 0)
    assert fa.device_error() == (0 if all(sound) else 2)
    assert admitted.tolist() == sound and left.tolist() == [1]
    want_slot, want_pos, want_mask = [-1] * tokens, [0] * tokens, [0] * tokens
    for b in range(n):
        if sound[b]:
            for i, t in enumerate(range(cu[b], cu[b + 1])):
                p = ctx[b] + i
                want_slot[t] = (4 * b + p // page) * page + p % page
                want_pos[t] = ctx[b] if tree else p
                want_mask[t] = 1 << i
    assert slots.tolist() == want_slot and positions.tolist() == want_pos
    if tree:
        assert mask.flatten().tolist() == want_mask
