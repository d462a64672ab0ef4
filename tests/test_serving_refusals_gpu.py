"""Arguments that the serving operators refuse: an error with its reason before anything is launched, and no output
written."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.rotary import rotary_table

pytestmark = pytest.mark.gpu


def zeros(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def refused(fn, good, changes):
    """fn takes `good`; with each of the changes it raises the error that stands beside it."""
    fn(**good)
    for match, change in changes:
        change = change() if callable(change) else change
        with pytest.raises(RuntimeError, match=match):
            fn(**{**good, **change})
    fn(**good)
    torch.cuda.synchronize()
    assert fa.device_error() == 0


def test_rotary(cuda):
    good = dict(q=zeros(2, 5, 4, 64), k=zeros(2, 5, 2, 64), table=rotary_table(8, 64, device=cuda), positions=ints(0, 1, 2, 3, 4))
    changes = [
        ("layout must be", dict(layout="nbhd")),
        ("supports fp16, bf16 and fp32", lambda: dict(q=zeros(2, 5, 4, 64).double(), k=None)),
        ("supports fp16, bf16 and fp32", lambda: dict(q=zeros(2, 5, 4, 64).int(), k=None)),
        (r"q must be \[tokens, heads, D\] or 4D", lambda: dict(q=zeros(5, 64), k=None)),
        ("q: the last dimension must be contiguous", lambda: dict(q=zeros(2, 5, 4, 128)[..., ::2])),
        ("k: the last dimension must be contiguous", lambda: dict(k=zeros(2, 5, 2, 128)[..., ::2])),
        ("k must have q's rank and type", lambda: dict(k=zeros(10, 2, 64))),
        ("k must have q's rank and type", lambda: dict(k=zeros(2, 5, 2, 64).bfloat16())),
        ("k must match q in all but its heads", lambda: dict(k=zeros(2, 4, 2, 64))),
        ("k must match q in all but its heads", lambda: dict(k=zeros(2, 5, 2, 32))),
        ("All tensors must be on CUDA", lambda: dict(k=torch.zeros(2, 5, 2, 64, dtype=torch.float16))),
        ("the table must be a contiguous float32 matrix", lambda: dict(table=zeros(8, 64))),
        ("the table must be a contiguous float32 matrix", lambda: dict(table=zeros(64, 8, dtype=torch.float32).t())),
        ("the table must be on q's CUDA device", dict(table=torch.zeros(8, 64))),
        ("an even number up to head_dim", lambda: dict(table=zeros(8, 63, dtype=torch.float32))),
        ("an even number up to head_dim", lambda: dict(table=zeros(8, 66, dtype=torch.float32))),
        ("positions must be int32 or int64", lambda: dict(positions=zeros(5, dtype=torch.int16))),
        (r"positions must be \[N\] or \[B, N\]", lambda: dict(positions=ints(0, 1, 2, 3))),
        (r"positions must be \[N\] or \[B, N\]", lambda: dict(positions=zeros(5, 2, dtype=torch.int32))),
        ("positions must be contiguous", lambda: dict(positions=zeros(10, dtype=torch.int32)[::2])),
        ("positions must be on q's CUDA device", dict(positions=torch.arange(5))),
        ("out_q must match its input", lambda: dict(out_q=zeros(2, 5, 2, 64))),
        ("out_k must match its input", lambda: dict(out_k=zeros(2, 5, 2, 64).float())),
        ("out_q must not be an expanded tensor", lambda: dict(out_q=zeros(1, 5, 4, 64).expand(2, 5, 4, 64))),
        ("out_q: the last dimension must be contiguous", lambda: dict(out_q=zeros(2, 5, 4, 128)[..., ::2])),
        ("out_k without k", lambda: dict(k=None, out_k=zeros(2, 5, 2, 64))),
    ]
    refused(fa.rotary, good, changes)
    back = dict(dq=good["q"], dk=good["k"], table=good["table"], positions=good["positions"])
    refused(fa.rotary_backward, back, [
        ("k must match q in all but its heads", lambda: dict(dk=zeros(2, 4, 2, 64))),
        ("an even number up to head_dim", lambda: dict(table=zeros(8, 66, dtype=torch.float32)))])


def test_rotary_append(cuda):
    good = dict(q=zeros(3, 4, 64), k=zeros(3, 2, 64), v=zeros(3, 2, 64), table=rotary_table(8, 64, device=cuda),
                positions=ints(0, 1, 2), slots=ints(5, -1, 17, dtype=torch.int64), k_cache=zeros(2, 16, 2, 64),
                v_cache=zeros(2, 16, 2, 64))
    changes = [
        ("layout must be", dict(layout="nbhd")),
        (r"q, k and v must be \[tokens, heads, D\]", lambda: dict(v=zeros(1, 3, 2, 64))),
        ("k and v must have q's type", lambda: dict(v=zeros(3, 2, 64).float())),
        ("k and v must match q", lambda: dict(v=zeros(3, 1, 64))),
        ("k and v must match q", lambda: dict(k=zeros(2, 2, 64), v=zeros(2, 2, 64))),
        ("slots must be Long", lambda: dict(slots=ints(5, -1, 17))),
        ("slots must hold one slot for each token", lambda: dict(slots=ints(5, -1, dtype=torch.int64))),
        ("slots must be contiguous", lambda: dict(slots=zeros(6, dtype=torch.int64)[::2])),
        ("k_cache must have q's type", lambda: dict(k_cache=zeros(2, 16, 2, 64).bfloat16())),
        (r"k_cache must be 4D \[blocks, page, heads, D\]", lambda: dict(k_cache=zeros(32, 2, 64))),
        ("the same shape", lambda: dict(v_cache=zeros(3, 16, 2, 64))),
        ("must have k's heads", lambda: dict(k_cache=zeros(2, 16, 1, 64), v_cache=zeros(2, 16, 1, 64))),
        ("must have k's heads", dict(layout="bhnd")),
        ("k_cache must not be an expanded tensor", lambda: dict(k_cache=zeros(1, 16, 2, 64).expand(2, 16, 2, 64))),
        ("v_cache must not be an expanded tensor", lambda: dict(v_cache=zeros(2, 16, 1, 64).expand(2, 16, 2, 64))),
        ("v_cache: the last dimension must be contiguous", lambda: dict(v_cache=zeros(2, 16, 2, 128)[..., ::2])),
        ("page_size must be positive", lambda: dict(k_cache=zeros(2, 0, 2, 64), v_cache=zeros(2, 0, 2, 64))),
        ("out_q must match its input", lambda: dict(out_q=zeros(3, 2, 64))),
    ]
    refused(fa.rotary_append, good, changes)


def test_plan(cuda):
    good = dict(context_lens=ints(3, 0), cu_seqlens=ints(0, 1, 3), block_table=zeros(2, 4, dtype=torch.int32),
                held_blocks=ints(1, 0), free_blocks=ints(1, 2, 3), num_free=ints(3), total_tokens=3, page_size=16,
                parents=ints(-1, -1, 0), mask_words=1)
    changes = [
        ("context_lens must be Int", lambda: dict(context_lens=ints(3, 0, dtype=torch.int64))),
        ("context_lens must have 1 dimension", lambda: dict(context_lens=ints(3, 0)[None])),
        ("cu_seqlens must hold one value more", lambda: dict(cu_seqlens=ints(0, 3))),
        ("block_table must be an Int matrix", lambda: dict(block_table=zeros(2, 4, dtype=torch.int64))),
        ("block_table must have a row for each request", lambda: dict(block_table=zeros(3, 4, dtype=torch.int32))),
        ("block_table: the last dimension", lambda: dict(block_table=zeros(4, 2, dtype=torch.int32).t())),
        ("block_table must not be an expanded", lambda: dict(block_table=zeros(1, 4, dtype=torch.int32).expand(2, 4))),
        ("held_blocks must hold one value", lambda: dict(held_blocks=ints(1))),
        ("free_blocks must be contiguous", lambda: dict(free_blocks=zeros(6, dtype=torch.int32)[::2])),
        ("num_free must hold one value", lambda: dict(num_free=ints(3, 3))),
        ("All tensors must be on the same CUDA device|All tensors must be on CUDA",
         dict(num_free=torch.tensor([3], dtype=torch.int32))),
        ("must not be negative", dict(total_tokens=-1)),
        ("must not be negative", dict(mask_words=-1)),
        ("page_size must be positive", dict(page_size=0)),
        ("parents must hold one value for each token", lambda: dict(parents=ints(-1, -1))),
        ("a tree needs mask_words > 0", dict(mask_words=0)),
    ]

    def fresh(block_table, **more):  # a step writes the table: each call starts from its own
        return fa.plan_cache_step(block_table=block_table.clone() if block_table.is_contiguous() else block_table, **more)

    refused(fresh, good, changes)
    many = zeros(16385, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="at most 16384 requests"):
        fa.plan_cache_step(many, zeros(16386, dtype=torch.int32), many[:, None], many, ints(), ints(0), 0, 16)


def test_tree_attention(cuda):
    good = dict(q=zeros(3, 4, 64), k_cache=zeros(2, 16, 2, 64), v_cache=zeros(2, 16, 2, 64), block_table=ints(0, 1)[:, None],
                context_lens=ints(4, 2), cu_seqlens=ints(0, 1, 3), tree_mask=ints(1, 1, 3)[:, None])
    changes = [
        ("layout must be", dict(layout="nbhd")),
        (r"q must be \[tokens, heads, D\]", lambda: dict(q=zeros(1, 3, 4, 64))),
        ("supports fp16 and bf16", lambda: dict(q=zeros(3, 4, 64).float())),
        ("k_cache must have q's type", lambda: dict(q=zeros(3, 4, 64).bfloat16())),
        ("head_dim 64 or 128", lambda: dict(q=zeros(3, 4, 96), k_cache=zeros(2, 16, 2, 96), v_cache=zeros(2, 16, 2, 96))),
        ("the caches must have q's head_dim", lambda: dict(q=zeros(3, 4, 128))),
        ("k_cache and v_cache must have the same shape", lambda: dict(v_cache=zeros(2, 16, 1, 64))),
        ("heads must be a multiple of kv_heads", lambda: dict(q=zeros(3, 5, 64))),
        ("heads must be a multiple of kv_heads", lambda: dict(q=zeros(3, 258, 64))),
        ("page_size must be a power of two", lambda: dict(k_cache=zeros(2, 24, 2, 64), v_cache=zeros(2, 24, 2, 64))),
        ("page_size must be a power of two", lambda: dict(k_cache=zeros(2, 4, 2, 64), v_cache=zeros(2, 4, 2, 64))),
        ("page_size must be a power of two", lambda: dict(k_cache=zeros(2, 512, 2, 64), v_cache=zeros(2, 512, 2, 64))),
        ("empty cache", lambda: dict(k_cache=zeros(0, 16, 2, 64), v_cache=zeros(0, 16, 2, 64))),
        ("the last dimension must be contiguous", lambda: dict(q=zeros(3, 4, 128)[..., ::2])),
        ("16-byte aligned", lambda: dict(q=zeros(3 * 4 * 64 + 1)[1:].view(3, 4, 64))),
        ("positive multiples of 8", lambda: dict(q=zeros(3, 4, 68)[..., :64])),
        ("positive multiples of 8", lambda: dict(k_cache=zeros(2, 16, 1, 64).expand(2, 16, 2, 64))),
        ("positive multiples of 8", lambda: dict(v_cache=zeros(2, 16, 2, 68)[..., :64])),
        ("context_lens must be Int", lambda: dict(context_lens=ints(4, 2, dtype=torch.int64))),
        ("cu_seqlens must hold one value more", lambda: dict(cu_seqlens=ints(0, 3))),
        ("block_table must have a row for each request", lambda: dict(block_table=ints(0)[:, None])),
        ("block_table: the last dimension", lambda: dict(block_table=zeros(4, 2, dtype=torch.int32).t())),
        ("tree_mask must be Int", lambda: dict(tree_mask=zeros(3, 1, dtype=torch.int64))),
        (r"tree_mask must be \[tokens, words\]", lambda: dict(tree_mask=zeros(2, 1, dtype=torch.int32))),
        (r"tree_mask must be \[tokens, words\]", lambda: dict(tree_mask=zeros(3, 0, dtype=torch.int32))),
        ("tree_mask must be contiguous", lambda: dict(tree_mask=zeros(3, 2, dtype=torch.int32)[:, :1])),
        ("out tensor must be contiguous", lambda: dict(out=zeros(3, 4, 128)[..., :64])),
        ("out tensor shape must match q", lambda: dict(out=zeros(3, 2, 64))),
        ("out tensor must have q's type", lambda: dict(out=zeros(3, 4, 64).float())),
    ]
    refused(fa.tree_attention, good, changes)
    n = zeros(4097, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="at most 4096 requests"):
        fa.tree_attention(good["q"], good["k_cache"], good["v_cache"], n[:, None], n, zeros(4098, dtype=torch.int32))


def test_refused_call_writes_nothing(cuda):
    cache, out = zeros(2, 24, 2, 64), torch.full((3, 4, 64), 7.0, dtype=torch.float16, device=cuda)
    with pytest.raises(RuntimeError, match="power of two"):
        fa.tree_attention(zeros(3, 4, 64), cache, cache, ints(0)[:, None], ints(4), ints(0, 3), out=out)
    assert bool((out == 7.0).all())
    q, k = zeros(3, 4, 64) + 1, zeros(3, 2, 64) + 1
    with pytest.raises(RuntimeError, match="must match its input"):
        fa.rotary(q, k, rotary_table(8, 64, device=cuda), out_q=out, out_k=q)
    assert bool((out == 7.0).all())
