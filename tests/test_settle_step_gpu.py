"""A step's results into the cache's state."""
import ctypes

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1, 7, 256, 257, 3000])
def test_state_and_lengths(cuda, n):
    g = torch.Generator(device=cuda).manual_seed(n)
    draw = lambda k: torch.randint(0, 1000, (k,), generator=g, device=cuda, dtype=torch.int32)  # noqa: E731
    ctx, held, free, after, left = draw(n), draw(n), draw(1), draw(n), draw(1)
    admitted = draw(n) % 3 > 0
    where, version = (held.data_ptr(), free.data_ptr()), held._version
    lens = fa.settle_step(ctx, held, free, admitted, after, left)
    assert torch.equal(held, after) and torch.equal(free, left) and (held.data_ptr(), free.data_ptr()) == where
    assert torch.equal(lens, torch.where(admitted, ctx, -1)) and held._version > version


@pytest.mark.gpu
def test_refusals(cuda):
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    good = dict(context_lens=ints(3, 4), held_blocks=ints(1, 1), num_free=ints(2), admitted=ints(1, 0).bool(),
                held_after=ints(2, 1), free_after=ints(1))
    for match, change in [("context_lens must be Int", dict(context_lens=ints(3, 4).long())),
                          ("admitted must be Bool", dict(admitted=ints(1, 0))),
                          ("one value for each request", dict(held_after=ints(2))),
                          ("must hold one value", dict(free_after=ints(1, 1))),
                          ("must be contiguous", dict(held_blocks=ints(1, 1, 1, 1)[::2])),
                          ("must be on CUDA", dict(num_free=torch.ones(1, dtype=torch.int32)))]:
        with pytest.raises(RuntimeError, match=match):
            fa.settle_step(**{**good, **change})
    assert good["held_blocks"].tolist() == [1, 1] and good["num_free"].tolist() == [2]


def test_c_checks_before_device(fl_lib):
    buf = ctypes.create_string_buffer(64)
    fn, p = fl_lib.fl_settle_step, ctypes.addressof(buf)
    fn.argtypes, fn.restype = [ctypes.c_void_p] * 7 + [ctypes.c_int64, ctypes.c_void_p], ctypes.c_int
    assert fn(p, p, p, p, p, p, p, -1, None) == 1
    assert fn(p, p, p, p, p, p, p, 16385, None) == 2
    for i in range(7):
        assert fn(*[None if j == i else p for j in range(7)], 1, None) == 1


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.settle_step(x, x, x, x.bool(), x, x)
