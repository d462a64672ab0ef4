"""Rotary positions against the formula in 64 bits, and the gradient against the formula's and differences.

Tolerance: a rotated element is two products and one sum in fp32 (each rounds by at most 2^-24 of the magnitudes
involved: 3 roundings) and one rounding to the storage type; 2^-22 of the magnitude and the type's unit roundoff
bound them. Below the type's normal range a rounding is half of its smallest step (2^-25 for fp16)."""
import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def table_of(positions, rot, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(positions, rot // 2, generator=g, dtype=torch.float64) * 6.3
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def close(got, want, mag):
    u = orc.UNIT[got.dtype]
    got = got.double().cpu()
    bound = u * want.abs() + 2.0 ** -22 * mag * (1 + u) + 2.0 ** -25
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


def rows(x, layout):
    """[B, N, H, D] or [B, H, N, D] as [tokens, H, D]."""
    x = x.transpose(1, 2) if layout == "bhnd" else x
    return x.reshape(-1, x.shape[2], x.shape[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["bnhd", "bhnd"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 64), (2, 7, 8, 2, 64, 32), (1, 33, 3, 1, 128, 96),
                                   (2, 5, 2, 2, 80, 48), (1, 4, 2, 1, 20, 10), (1, 3, 1, 1, 7, 4), (1, 3, 40, 8, 128, 128),
                                   (1, 2, 1, 1, 256, 64)])
def test_rotary_matches_the_formula(cuda, dtype, layout, interleaved, shape):
    B, N, H, Hk, D, R = shape
    g = torch.Generator(device=cuda).manual_seed(1)
    make = lambda h: torch.randn((B, N, h, D) if layout == "bnhd" else (B, h, N, D), generator=g, device=cuda).to(dtype)  # noqa: E731
    q, k = make(H), make(Hk)
    table = table_of(N + 5, R, cuda)
    pos = torch.randint(0, N + 5, (N,), generator=g, device=cuda, dtype=torch.int32)
    for inverse, fn in ((False, fa.rotary), (True, fa.rotary_backward)):
        oq, ok = fn(q, k, table, pos, interleaved=interleaved, layout=layout)
        for x, y in ((q, oq), (k, ok)):
            want, mag = orc.rotate(rows(x, layout), table, pos.repeat(B), interleaved, inverse)
            close(rows(y, layout), want, mag)
            assert torch.equal(rows(y, layout)[..., R:], rows(x, layout)[..., R:])


def test_positions_forms(cuda):
    """[N], [B, N], int64 and none at all; three-dimensional q without k."""
    q = torch.randn(2, 6, 4, 64, device=cuda).half()
    table = table_of(9, 64, cuda)
    first = torch.arange(6, device=cuda, dtype=torch.int32)
    both = torch.stack([first, first + 3])
    a, none = fa.rotary(q, None, table)
    assert none is None
    assert torch.equal(a, fa.rotary(q, None, table, first)[0])
    assert torch.equal(a, fa.rotary(q, None, table, first.long())[0])
    b = fa.rotary(q, None, table, both)[0]
    assert torch.equal(b[0], a[0])
    assert torch.equal(b[1], fa.rotary(q[1], None, table, both[1])[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_in_place_and_offsets(cuda, dtype):
    """Slices of a fused projection, a tensor off a 16-byte boundary, an expanded gradient, in-place use."""
    T, H, D = 11, 4, 64
    table = table_of(T, D, cuda)
    fused = torch.randn(T, 3, H, D, device=cuda).to(dtype)
    q, k = fused[:, 0], fused[:, 1]
    want = fa.rotary(q.contiguous(), k.contiguous(), table)
    got = fa.rotary(q, k, table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(T * H * D + 1, device=cuda, dtype=dtype)[1:].view(T, H, D).copy_(q)
    assert torch.equal(fa.rotary(odd, None, table)[0], want[0])
    wide = torch.randn(1, H, D, device=cuda).to(dtype).expand(T, H, D)
    assert torch.equal(fa.rotary(wide, None, table)[0], fa.rotary(wide.contiguous(), None, table)[0])
    rest = fused[:, 2].clone()
    out = fa.rotary(q, k, table, out_q=q, out_k=k)
    assert out[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, 2], rest)


def test_position_outside_the_table(cuda):
    q = torch.randn(3, 2, 64, device=cuda).half()
    table = table_of(4, 32, cuda)
    assert fa.device_error() == 0
    out, _ = fa.rotary(q, None, table, torch.tensor([0, 4, -1], device=cuda, dtype=torch.int32))
    assert fa.device_error() == 2 and fa.device_error() == 0
    assert not out[0].isnan().any() and out[1:, :, :32].isnan().all()
    assert torch.equal(out[1:, :, 32:], q[1:, :, 32:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(cuda, interleaved):
    """The autograd form against differences: rotary is linear, so that a difference over a step of any size is
    exact up to rounding; in fp32 with a step of 1 it is within a few units in the last place."""
    from flashlite_b200.rotary import rotary_embedding

    g = torch.Generator(device=cuda).manual_seed(2)
    q = torch.randn(1, 2, 5, 8, generator=g, device=cuda, requires_grad=True)
    k = torch.randn(1, 1, 5, 8, generator=g, device=cuda, requires_grad=True)
    table = table_of(5, 6, cuda)
    wq, wk = torch.randn(q.shape, generator=g, device=cuda), torch.randn(k.shape, generator=g, device=cuda)

    def loss(a, b):
        x, y = rotary_embedding(a, b, table, interleaved=interleaved)
        return (x.double() * wq).sum() + (y.double() * wk).sum()

    loss(q, k).backward()
    base = loss(q, k).item()
    for x, other in ((q, False), (k, True)):
        for i in range(x.numel()):
            step = torch.zeros_like(x).view(-1)
            step[i] = 1.0
            moved = x.detach() + step.view_as(x)
            slope = (loss(q, moved) if other else loss(moved, k)).item() - base
            assert abs(slope - x.grad.view(-1)[i].item()) < 1e-5
    # an expanded gradient, as that of sum()
    q.grad = None
    x, _ = rotary_embedding(q, k, table, interleaved=interleaved)
    x.sum().backward()
    want, _ = fa.rotary_backward(torch.ones_like(q), None, table, interleaved=interleaved, layout="bhnd")
    assert torch.equal(q.grad, want)


def test_table_matches_the_formula():
    """The table against the scalings' formulas in plain Python, rounded once to fp32."""
    import math

    from flashlite_b200.rotary import rotary_table

    R, N, base, factor, original = 16, 40, 10000.0, 4.0, 256
    for scaling in ("none", "linear", "ntk", "by_parts"):
        got = rotary_table(N, R, base, scaling, factor, original, device="cpu")
        for p in (0, 1, 39):
            for j in range(R // 2):
                b = base * factor ** (R / (R - 2)) if scaling == "ntk" else base
                f = b ** (-2.0 * j / R)
                if scaling == "linear":
                    f /= factor
                scale = 1.0
                if scaling == "by_parts":
                    turns = original * f / (2 * math.pi)
                    keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
                    f = keep * f + (1 - keep) * f / factor
                    scale = 0.1 * math.log(factor) + 1.0
                assert abs(float(got[p, j]) - scale * math.cos(p * f)) < 2e-7
                assert abs(float(got[p, R // 2 + j]) - scale * math.sin(p * f)) < 2e-7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["bnhd", "bhnd"])
@pytest.mark.parametrize("shape", [(1, 8, 8, 64, 64, 16, False), (5, 4, 2, 128, 96, 8, True), (37, 7, 1, 64, 32, 32, False),
                                   (9, 2, 2, 40, 20, 5, True)])
def test_append(cuda, dtype, layout, shape):
    """Rotated keys and unchanged values at their slots, nothing elsewhere; slot -1 writes nothing."""
    T, H, Hk, D, R, page, interleaved = shape
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k, v = (torch.randn(T, h, D, generator=g, device=cuda).to(dtype) for h in (H, Hk, Hk))
    blocks = -(-T // page) + 2
    full = (blocks, page, Hk, D) if layout == "bnhd" else (blocks, Hk, page, D)
    kc, vc = torch.randn(full, generator=g, device=cuda).to(dtype), torch.randn(full, generator=g, device=cuda).to(dtype)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(blocks * page, generator=g, device=cuda)[:T].contiguous()
    if T > 2:
        slots[1] = -1
    table = table_of(50, R, cuda)
    pos = torch.randint(0, 50, (T,), generator=g, device=cuda)
    oq = fa.rotary_append(q, k, v, table, pos, slots, kc, vc, interleaved=interleaved, layout=layout)
    rq, rk = fa.rotary(q, k, table, pos, interleaved=interleaved)
    assert torch.equal(oq, rq)
    for cache, before, x in ((kc, k0, rk), (vc, v0, v)):
        want = (before if layout == "bnhd" else before.transpose(1, 2)).reshape(-1, Hk, D).clone()
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                want[s] = x[t]
        have = (cache if layout == "bnhd" else cache.transpose(1, 2)).reshape(-1, Hk, D)
        assert torch.equal(have, want)
    assert fa.device_error() == 0


@pytest.mark.parametrize("shape", [(2, 67, 2, 1, 64, 64), (1, 9, 32, 8, 64, 64), (3, 70, 16, 4, 64, 32), (1, 21, 8, 2, 128, 128),
                                   (2, 300, 3, 1, 64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_divisions(cuda, interleaved, shape):
    """Few heads and many, in odd numbers of tokens: tokens or heads side by side, one or more parts to a token."""
    test_rotary_matches_the_formula(cuda, torch.bfloat16, "bnhd", interleaved, shape)


@pytest.mark.parametrize("shape", [(11, 32, 8, 64, 64, 16, False), (6, 16, 4, 128, 128, 8, True), (131, 2, 1, 64, 64, 16, False),
                                   (50, 40, 40, 64, 32, 8, False)])
def test_append_divisions(cuda, shape):
    test_append(cuda, torch.float16, "bnhd", shape)


def test_append_slot_out_of_range(cuda):
    q = torch.randn(3, 2, 64, device=cuda).half()
    kc = torch.zeros(2, 8, 2, 64, device=cuda).half()
    vc = torch.zeros_like(kc)
    table = table_of(4, 64, cuda)
    fa.rotary_append(q, q, q, table, None, torch.tensor([16, -2, 3], device=cuda), kc, vc)
    assert fa.device_error() == 2
    assert torch.equal(vc.view(-1, 2, 64)[3], q[2]) and int((vc != 0).any(-1).any(-1).sum()) == 1


def test_other_stream(cuda):
    """On a side stream, in the order of that stream."""
    table = table_of(4096, 64, cuda)
    q = torch.randn(1, 4096, 8, 64, device=cuda).half()
    want, _ = fa.rotary(fa.rotary(q, None, table)[0], None, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = q.clone()
        for _ in range(2):
            x, _ = fa.rotary(x, None, table)
    side.synchronize()
    assert torch.equal(x, want)


def test_empty(cuda):
    table = table_of(4, 64, cuda)
    q = torch.empty(0, 8, 64, device=cuda).half()
    assert fa.rotary(q, q, table)[1].shape == q.shape
    kc = torch.zeros(1, 8, 8, 64, device=cuda).half()
    assert fa.rotary_append(q, q, q, table, None, torch.empty(0, dtype=torch.long, device=cuda), kc, kc.clone()).shape == q.shape
