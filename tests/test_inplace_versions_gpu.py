"""What the serving operators write in place counts as a change of the tensor: autograd sees it."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from flashlite_b200.rotary import rotary_table

pytestmark = pytest.mark.gpu


def test_saved_tensor_rotated_in_place(cuda):
    x = torch.randn(4, 2, 64, device=cuda, requires_grad=True)
    y = x * 2
    z = (y * y).sum()  # keeps y
    d = y.detach()
    fa.rotary(d, None, rotary_table(4, 64, device=cuda), out_q=d)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_every_output_that_is_given(cuda):
    table = rotary_table(8, 64, device=cuda)
    q, k = torch.randn(3, 4, 64, device=cuda).half(), torch.randn(3, 2, 64, device=cuda).half()
    kc, vc = torch.zeros(2, 16, 2, 64, device=cuda).half(), torch.zeros(2, 16, 2, 64, device=cuda).half()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    oq, ok, out, blocks = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), ints(0, 1)[:, None].contiguous()
    ctx, cu, held, free, left = ints(0, 0), ints(0, 1, 3), ints(0, 0), ints(1, 0), ints(2)
    slots = torch.tensor([0, 16, 17], device=cuda)
    written, read = [oq, ok, kc, vc, out, blocks], [q, k, table, ctx, cu, held, free, left, slots]
    versions = lambda ts: [t._version for t in ts]  # noqa: E731
    before, kept = versions(written), versions(read)
    fa.plan_cache_step(ctx, cu, blocks, held, free, left, 3, 16)
    fa.rotary(q, k, table, None, out_q=oq, out_k=ok)
    fa.rotary_append(q, k, k, table, None, slots, kc, vc, out_q=oq)
    fa.tree_attention(q, kc, vc, blocks, ctx, cu, out=out)
    assert all(a > b for a, b in zip(versions(written), before)), (versions(written), before)
    assert versions(read) == kept
    assert fa.device_error() == 0


def test_tensors_of_inference_mode(cuda):
    """They have no versions; they can be written outside of the mode as well as inside."""
    table = rotary_table(4, 64, device=cuda)
    with torch.inference_mode():
        q = torch.randn(4, 2, 64, device=cuda)
        want, _ = fa.rotary(q, None, table)
        out = torch.empty_like(q)
        fa.rotary(q, None, table, out_q=out)
    assert torch.equal(out, want)
    out2, _ = fa.rotary(q, None, table, out_q=q)
    assert torch.equal(out2, want)
