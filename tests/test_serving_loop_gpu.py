"""The serving operators together: drafted trees against decoding token by token, through PagedCache."""
import sys
from pathlib import Path

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more", [dict(), dict(layout="bhnd", page=32), dict(dim=128, heads=6, kv_heads=6, nodes=40, steps=3),
                                  dict(requests=1, nodes=1, steps=9, heads=5, kv_heads=1)])
def test_trees_against_single_tokens(cuda, more):
    """Outputs are averages of values of order 1 rounded to fp16 (2^-11 each way, probabilities rounded to fp16 too):
    two ways of the same sum differ by a few 2^-11 of the largest value, about 4."""
    import tree_decode

    assert tree_decode.run(**more) < 4 * 4 * 2.0 ** -11
    assert fa.device_error() == 0


def test_refused_request_keeps_its_state(cuda):
    from flashlite_b200.serving import PagedCache

    cache = PagedCache(2, 3, 16, 1, 64, 4, device=cuda)
    cu = torch.tensor([0, 20, 60], dtype=torch.int32, device=cuda)
    step = cache.plan(cu, 60)
    assert step.admitted.tolist() == [True, False] and cache.num_free.tolist() == [1]
    x = torch.randn(60, 1, 64, device=cuda).half()
    from flashlite_b200.rotary import rotary_table

    cache.attend(0, x, x, x, rotary_table(64, 64, device=cuda), step)
    cache.commit(step, torch.tensor([20, 40], device=cuda))
    assert cache.context_lens.tolist() == [20, 0] and cache.held_blocks.tolist() == [2, 0]
    assert fa.device_error() == 0
    cache.release(0)
    assert cache.num_free.tolist() == [3]
