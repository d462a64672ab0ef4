"""Second-order gradients of the autograd forms: right, or refused with an error, never silently short of a term."""
import pytest
import torch

import flashlite_b200.attention
import flashlite_b200.rotary
from oracle import serving_oracle as orc


def table_of(positions, rot, device="cpu"):
    angle = torch.rand(positions, rot // 2, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 6.3
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def statement(inverse):
    """The binding's call on the CPU, in 64 bits; like the binding's, its results have no history."""

    def call(q, k, table, positions=None, interleaved=False, layout="bnhd"):
        def one(x):
            if x is None:
                return None
            y = x.detach().transpose(1, 2) if layout == "bhnd" else x.detach()
            pos = torch.arange(y.shape[1]) if positions is None else positions
            z, _ = orc.rotate(y.reshape(-1, *y.shape[2:]), table, pos.repeat(y.shape[0]), interleaved, inverse)
            z = z.view(y.shape)
            return (z.transpose(1, 2) if layout == "bhnd" else z).contiguous()

        return one(q), one(k)

    return call


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(flashlite_b200.rotary, "rotary", statement(False))
    monkeypatch.setattr(flashlite_b200.rotary, "rotary_backward", statement(True))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_gradients_of_both_orders(on_cpu, interleaved, layout):
    g = torch.Generator().manual_seed(1)
    shape = (2, 3, 2, 6) if layout == "bnhd" else (2, 2, 3, 6)
    q, k = (torch.randn(shape, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    table = table_of(3, 4)
    fn = lambda a, b: flashlite_b200.rotary.rotary_embedding(a, b, table, None, interleaved, layout)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (q, k))
    assert torch.autograd.gradgradcheck(fn, (q, k))


def test_gradient_of_a_gradient(on_cpu):
    """L = sum R(x)^3: its gradient is R^T 3 R(x)^2, and that of the gradient's square 2 R^T 6 R(x) R(dL/dx)."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 1, 4, 6, generator=g, dtype=torch.float64, requires_grad=True)
    other = torch.randn(1, 1, 4, 6, generator=g, dtype=torch.float64)
    table = table_of(4, 6)
    forward, back = (lambda t, f=statement(i): f(t, None, table, layout="bhnd")[0] for i in (False, True))
    y, _ = flashlite_b200.rotary.rotary_embedding(x, other, table)
    first, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    assert torch.allclose(first, back(3 * forward(x) ** 2), atol=1e-12)
    second, = torch.autograd.grad((first ** 2).sum(), x)
    assert torch.allclose(second, 2 * back(6 * forward(x) * forward(first)), atol=1e-12)


def test_without_k(on_cpu):
    x = torch.randn(1, 1, 4, 6, dtype=torch.float64, requires_grad=True)
    y, none = flashlite_b200.rotary.rotary_embedding(x, None, table_of(4, 6))
    assert none is None
    grad, = torch.autograd.grad(y.sum(), x)
    assert torch.allclose(grad, statement(True)(torch.ones_like(x), None, table_of(4, 6), layout="bhnd")[0], atol=1e-12)


def test_table_that_wants_a_gradient(on_cpu):
    """There is no gradient of the table: refused instead of left out."""
    x = torch.randn(1, 1, 4, 6, dtype=torch.float64, requires_grad=True)
    with pytest.raises(ValueError, match="table"):
        flashlite_b200.rotary.rotary_embedding(x, x, table_of(4, 6).requires_grad_())


@pytest.mark.gpu
def test_second_order_on_the_kernel(cuda):
    """As above in fp32: three rotations (2^-22 of the magnitudes each) and the products around them, all of order 10^2
    at most."""
    from flashlite_b200.rotary import rotary_embedding

    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(1, 2, 5, 64, generator=g, device=cuda, requires_grad=True)
    table = table_of(5, 64, cuda)
    y, _ = rotary_embedding(x, x.detach(), table)
    first, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    second, = torch.autograd.grad((first ** 2).sum(), x)
    cpu = table.cpu()
    forward, back = (lambda t, f=statement(i): f(t, None, cpu, layout="bhnd")[0] for i in (False, True))
    exact = x.detach().cpu().double()
    want = 2 * back(6 * forward(exact) * forward(back(3 * forward(exact) ** 2)))
    assert float((second.cpu() - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max())
