"""``flash_attention`` has first-order gradients: a second-order one is refused with an error, not left short of a term."""
import pytest
import torch

import flashlite_b200.attention


def test_second_order_is_refused(monkeypatch):
    def forward(q, k, v, sm_scale, is_causal, return_lse, layout):
        s = q @ k.transpose(-1, -2)
        return s.softmax(-1) @ v, s.logsumexp(-1)

    def backward(q, k, v, out, dout, lse, sm_scale, is_causal, layout):  # like the binding's, without history
        with torch.enable_grad():
            leaves = [x.detach().requires_grad_() for x in (q, k, v)]
            return tuple(g.detach() for g in torch.autograd.grad(forward(*leaves, 0, False, True, layout)[0], leaves, dout.detach()))

    monkeypatch.setattr(flashlite_b200.attention, "forward_flash2_ex", forward)
    monkeypatch.setattr(flashlite_b200.attention, "backward_flash2", backward)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 1, 3, 4, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(3))
    out = flashlite_b200.attention.flash_attention(q, k, v)
    first = torch.autograd.grad((out ** 2).sum(), (q, k, v), create_graph=True)
    plain = torch.autograd.grad((forward(q, k, v, 0, False, True, "bhnd")[0] ** 2).sum(), (q, k, v))
    assert all(torch.allclose(a, b, atol=1e-12) for a, b in zip(first, plain))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        ((first[0] ** 2).sum() + out.sum()).backward()  # a penalty on the gradient beside a loss
