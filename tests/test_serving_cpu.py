"""Refusals of the serving operators and rotary positions, and their 64-bit statements against each other: no kernel is
launched here."""
import ctypes
import math

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from oracle import serving_oracle as orc

FL_OK, FL_ERR_INVALID_ARGUMENT, FL_ERR_UNSUPPORTED = 0, 1, 2


def zeros(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, table, ints = zeros(2, 4, 64), zeros(4, 64, dtype=torch.float32), zeros(2, dtype=torch.int32)
    cache = zeros(2, 16, 4, 64)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.rotary(q, q, table)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.rotary_backward(q, None, table)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.rotary_append(q, q, q, table, None, ints.long(), cache, cache)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.tree_attention(q, cache, cache, ints[None], ints[:1], ints)
    with pytest.raises(RuntimeError, match="All tensors must be on CUDA"):
        fa.plan_cache_step(ints, ints, ints[None], ints, ints, ints, 2, 16)
    with pytest.raises(RuntimeError, match="layout must be"):
        fa.rotary(q, q, table, layout="hnd")


def test_refusal_that_names_a_number():
    """An error text with a number in it (a C++ stream of the binding); tensors without storage stand for CUDA ones."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        ints = torch.empty((1, 2), dtype=torch.int32, device="cuda:0")
        with pytest.raises(RuntimeError, match=r"context_lens must have 1 dimension"):
            fa.plan_cache_step(ints, ints, ints, ints, ints, ints, 2, 16)


def test_table_arguments():
    from flashlite_b200.rotary import rotary_table

    assert rotary_table(3, 8, device="cpu").shape == (3, 8) and rotary_table(0, 8, device="cpu").shape == (0, 8)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.5),
                dict(rot_dim=8, scaling="other"), dict(rot_dim=2, scaling="ntk", factor=2.0),
                dict(rot_dim=8, scaling="by_parts", factor=2.0), dict(rot_dim=8, positions=-1)):
        with pytest.raises(ValueError):
            rotary_table(**{"positions": 3, "device": "cpu", **bad})


class RotaryArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_out", "v_out", "table", "positions", "slots")] + \
        [(n, ctypes.c_int64) for n in ("batch", "length", "heads", "kv_heads", "head_dim", "rot", "table_rows",
                                       "cache_blocks", "page_size")] + \
        [(n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride", "k_out_stride",
                                           "v_out_stride")] + \
        [(n, ctypes.c_int32) for n in ("dtype", "interleaved", "inverse", "positions_64", "positions_batch")]


class PlanArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("context_lens", "cu_seqlens", "block_table", "held_blocks", "free_blocks",
                                               "num_free", "parents", "slots", "positions", "admitted", "held_after",
                                               "num_free_after", "tree_mask")] + \
        [(n, ctypes.c_int64) for n in ("requests", "tokens", "table_cols", "table_stride", "free_capacity", "page_size",
                                       "mask_words")]


class TreeArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k_cache", "v_cache", "out", "lse", "block_table", "context_lens",
                                               "cu_seqlens", "tree_mask", "workspace")] + \
        [("workspace_bytes", ctypes.c_size_t)] + \
        [(n, ctypes.c_int64) for n in ("tokens", "requests", "heads", "kv_heads", "head_dim", "num_blocks", "page_size",
                                       "table_cols", "table_stride", "mask_words")] + \
        [("q_stride", ctypes.c_int64 * 2), ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
         ("dtype", ctypes.c_int32), ("sm_scale", ctypes.c_float)]


def call(lib, name, args):
    fn = getattr(lib, name)
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    return fn(ctypes.addressof(args) if args is not None else None, None)


def test_rotary_checks_before_device(fl_lib):
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)

    def status(**more):
        a = RotaryArgs(q=p, k=p, q_out=p, k_out=p, table=p, batch=1, length=2, heads=2, kv_heads=1, head_dim=64, rot=64,
                       table_rows=4)
        for n, v in more.items():
            setattr(a, n, v)
        return call(fl_lib, "fl_rotary", a)

    assert call(fl_lib, "fl_rotary", None) == FL_ERR_INVALID_ARGUMENT
    for more in (dict(batch=-1), dict(rot=63), dict(rot=66), dict(rot=-2), dict(head_dim=0), dict(q=None), dict(k_out=None),
                 dict(table=None), dict(v=p), dict(slots=p), dict(v=p, v_out=p, slots=p), dict(length=1 << 40)):
        assert status(**more) == FL_ERR_INVALID_ARGUMENT, more
    assert status(dtype=3) == FL_ERR_UNSUPPORTED
    assert status(length=0) == FL_OK and status(batch=0) == FL_OK


def test_plan_checks_before_device(fl_lib):
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)

    def status(**more):
        a = PlanArgs(**{n: p for n, t in PlanArgs._fields_ if t is ctypes.c_void_p}, requests=1, tokens=1, table_cols=1,
                     table_stride=1, free_capacity=1, page_size=16, mask_words=1)
        for n, v in more.items():
            setattr(a, n, v)
        return call(fl_lib, "fl_plan_cache_step", a)

    assert call(fl_lib, "fl_plan_cache_step", None) == FL_ERR_INVALID_ARGUMENT
    for more in (dict(tokens=-1), dict(page_size=0), dict(context_lens=None), dict(cu_seqlens=None), dict(num_free=None),
                 dict(held_after=None), dict(slots=None), dict(mask_words=0), dict(tree_mask=None), dict(tokens=1 << 40)):
        assert status(**more) == FL_ERR_INVALID_ARGUMENT, more
    assert status(requests=16385) == FL_ERR_UNSUPPORTED


def test_tree_attention_checks_before_device(fl_lib):
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)

    def status(**more):
        a = TreeArgs(**{n: p for n, t in TreeArgs._fields_ if t is ctypes.c_void_p}, tokens=1, requests=1, heads=4, kv_heads=2,
                     head_dim=64, num_blocks=2, page_size=16, table_cols=1, table_stride=1, mask_words=1)
        for n, v in more.items():
            setattr(a, n, v)
        return call(fl_lib, "fl_tree_attention", a)

    assert call(fl_lib, "fl_tree_attention", None) == FL_ERR_INVALID_ARGUMENT
    for more in (dict(tokens=-1), dict(heads=5), dict(kv_heads=0), dict(heads=258), dict(q=None), dict(cu_seqlens=None),
                 dict(context_lens=None), dict(block_table=None), dict(v_cache=None), dict(tokens=1 << 40)):
        assert status(**more) == FL_ERR_INVALID_ARGUMENT, more
    for more in (dict(head_dim=96), dict(dtype=2), dict(page_size=24), dict(page_size=4), dict(page_size=512),
                 dict(requests=4097)):
        assert status(**more) == FL_ERR_UNSUPPORTED, more
    assert status(tokens=0) == FL_OK


def test_oracle_rotation_is_a_complex_product():
    x = torch.randn(3, 2, 8, dtype=torch.float64)
    angle = torch.randn(5, 3, dtype=torch.float64)
    table = torch.cat([angle.cos(), angle.sin()], 1)
    pos = torch.tensor([4, 0, 2])
    turn = torch.polar(torch.ones_like(angle), angle)[pos][:, None]
    y, mag = orc.rotate(x, table, pos, interleaved=True)
    z = torch.view_as_complex(x[..., :6].reshape(3, 2, 3, 2).contiguous()) * turn
    assert torch.allclose(y[..., :6].reshape(3, 2, 3, 2), torch.view_as_real(z), atol=1e-14)
    assert torch.equal(y[..., 6:], x[..., 6:]) and bool((mag >= y.abs() - 1e-15).all())
    back, _ = orc.rotate(y, table, pos, interleaved=True, inverse=True)
    assert torch.allclose(back, x, atol=1e-14)
    y, _ = orc.rotate(x, table, pos)
    z = torch.complex(x[..., :3], x[..., 3:6]) * turn
    assert torch.allclose(y[..., :6], torch.cat([z.real, z.imag], -1), atol=1e-14)


def test_oracle_attention_is_softmax_attention():
    """One request whose pages lie in order: the dense causal attention of the same rows."""
    torch.manual_seed(0)
    k, v = torch.randn(2, 8, 2, 64, dtype=torch.float64), torch.randn(2, 8, 2, 64, dtype=torch.float64)
    q = torch.randn(5, 4, 64, dtype=torch.float64)
    out, lse, weight, reach = orc.tree_attention(q, k, v, [[0, 1]], [7], [0, 5])
    dense_k, dense_v = (x.reshape(16, 2, 64)[:12].repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
    s = (q.transpose(0, 1) @ dense_k.transpose(1, 2)) / math.sqrt(64)
    s = s.masked_fill(torch.arange(12) > torch.arange(5)[:, None] + 7, -math.inf)
    assert torch.allclose(out, (s.softmax(-1) @ dense_v).transpose(0, 1), atol=1e-12)
    assert torch.allclose(lse, s.logsumexp(-1).T, atol=1e-12)
    assert bool((weight >= out.abs() - 1e-12).all()) and bool((reach > 0).all())
