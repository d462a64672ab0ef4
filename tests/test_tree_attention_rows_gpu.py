"""Rows of q that belong to no request: 0 and -inf, wherever they lie."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa

pytestmark = pytest.mark.gpu


def run(device, heads, kv_heads, tokens, cu, requests, seed=0):
    """Attention into buffers full of sevens; each request has 20 cached tokens in blocks of its own."""
    g = torch.Generator(device=device).manual_seed(seed)
    page, width = 16, 8
    blocks = requests * width
    k, v = (torch.randn(blocks, page, kv_heads, 64, generator=g, device=device).half() for _ in range(2))
    q = torch.randn(tokens, heads, 64, generator=g, device=device).half()
    table = torch.arange(blocks, dtype=torch.int32, device=device).view(requests, width)
    ctx = torch.full((requests,), 20, dtype=torch.int32, device=device)
    out = torch.full_like(q, 7.0)
    full = [torch.full((tokens, heads), 7.0, device=device) for _ in range(4)]  # what torch may give the log-sum-exps
    del full
    _, lse = fa.tree_attention(q, k, v, table, ctx, torch.tensor(cu, dtype=torch.int32, device=device), out=out, return_lse=True)
    torch.cuda.synchronize()
    return out, lse


CASES = [
    # cu_seqlens, rows that a request covers, whether something is out of range
    ([3, 5, 9], range(3, 9), 0),          # rows before the first request and after the last
    ([12, 12, 12], [], 0),                # no tokens at all
    ([0, 4, 100], range(0, 4), 2),        # a request that would end past q
    ([-3, 2, 6], range(2, 6), 2),         # one that would begin before it
    ([9, 2, 6], range(2, 6), 2),          # offsets that run back
    ([0, 3, 100, 5, 8], [0, 1, 2, 5, 6, 7], 2),  # two unsound requests in the middle
]


@pytest.mark.parametrize("cu,covered,error", CASES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (32, 1)])
def test_rows_without_a_request(cuda, heads, kv_heads, cu, covered, error):
    """heads: few rows to a unit, and many."""
    tokens, requests = 12, len(cu) - 1
    out, lse = run(cuda, heads, kv_heads, tokens, cu, requests)
    assert fa.device_error() == error
    mine = torch.zeros(tokens, dtype=torch.bool, device=cuda)
    mine[list(covered)] = True
    assert bool((out[~mine] == 0).all()) and bool((lse[~mine] == -float("inf")).all())
    assert bool((out[mine] != 7.0).all()) and bool(lse[mine].isfinite().all())


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (32, 1)])
def test_one_unsound_request_among_many(cuda, heads, kv_heads):
    cu = [2 * b for b in range(101)]
    cu[51] = 1000  # requests 50 and 51
    out, lse = run(cuda, heads, kv_heads, 203, cu, 100)
    assert fa.device_error() == 2
    gone = torch.zeros(203, dtype=torch.bool, device=cuda)
    gone[100:104] = True
    gone[200:] = True
    assert bool((out[gone] == 0).all()) and bool((lse[gone] == -float("inf")).all())
    assert bool((out[~gone] != 7.0).all()) and bool(lse[~gone].isfinite().all())
