"""Tokens that a serving step refuses (slot -1) in rotary_append."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.rotary import rotary_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_position_of_a_token_without_a_slot(cuda, dtype):
    """Refused: its position need not be in the table. With a slot it has to be."""
    q, k = torch.randn(3, 2, 64, device=cuda).to(dtype), torch.randn(3, 1, 64, device=cuda).to(dtype)
    cache = torch.zeros(2, 16, 1, 64, device=cuda, dtype=dtype)
    table = rotary_table(8, 64, device=cuda)
    for slots, error in (([4, -1, 5], 0), ([4, 6, 5], 2)):
        fa.rotary_append(q, k, k, table, torch.tensor([0, 8, 7], dtype=torch.int32, device=cuda), torch.tensor(slots, device=cuda), cache, cache.clone())
        assert fa.device_error() == error
