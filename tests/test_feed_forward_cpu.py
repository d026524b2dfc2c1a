"""Refusals of the feed-forward operators, without a GPU: every bad call ends in ValueError before a launch."""

import random

import pytest
import torch

from llm_compileforge_b200 import B200Backend, _lib, ops
from test_abi_cpu import _fake_desc

BF16 = torch.bfloat16


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: ops.fused_linear(t(4, 8), t(16, 8)),  # K differs
    lambda: ops.fused_linear(t(4, 8), t(8, 8, 2)),
    lambda: ops.fused_linear(t(4, 0), t(0, 8)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8, dtype=torch.float16)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), t(8, dtype=torch.float32)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), activation="swish"),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), residual=t(4, 16)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), residual=t(4, 8, dtype=torch.float32)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), out=t(4, 4)),
    lambda: ops.fused_linear(t(2, 4, 8), t(8, 8), out=t(4, 2, 8).transpose(0, 1)),
    lambda: ops.fused_linear(t(4, 8), t(8, 8), up_weight=t(8, 8).t()[:, :], activation="silu"),
    lambda: ops.fused_linear(t(4, 8), t(8, 32)[:, ::2]),
    lambda: ops.grouped_linear(t(4, 8), t(8, 8), i32(2)),
    lambda: ops.grouped_linear(t(4, 8), t(2, 8, 8), torch.zeros(3, dtype=torch.int64)),
    lambda: ops.grouped_linear(t(4, 8), t(2, 8, 8), i32(3), row_index=torch.zeros(4)),
    lambda: ops.grouped_linear(t(4, 8), t(2, 8, 8), i32(3), out=t(5, 8)),
    lambda: ops.moe_route(t(4, 8), 9),
    lambda: ops.moe_route(t(4, 8), 0),
    lambda: ops.moe_route(t(4, 64), 33),
    lambda: ops.moe_route(t(4, 8, 2), 1),
    lambda: ops.moe_combine(t(4, 8), i32(2, 2), t(2, 2)),
    lambda: ops.moe_combine(t(4, 8), i32(2, 2), torch.zeros(2, 3)),
    lambda: ops.moe_combine(t(4, 8), torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2)),
    lambda: ops.moe_combine(t(4, 8), i32(2, 2), torch.zeros(2, 2), residual=t(3, 8)),
    # good calls, but on the CPU
    lambda: ops.fused_linear(t(4, 8), t(8, 8)),
    lambda: ops.moe_combine(t(4, 8), i32(2, 2), torch.zeros(2, 2)),
])
def test_bad_calls_raise_value_errors(call):
    with pytest.raises(ValueError):
        call()


def test_names_of_the_executor():
    assert {"fused_linear", "grouped_linear", "moe_route", "moe_combine"} <= set(B200Backend().supported_ops())


def lin(x, w, b, u, ub, r, o, layout=0, dtype=1, odt=1, act=0):
    import ctypes

    p = lambda d: ctypes.cast(ctypes.pointer(d), ctypes.c_void_p) if d is not None else None  # noqa: E731
    return _lib.load().sfb_fused_linear(p(x), p(w), p(b), p(u), p(ub), p(r), p(o), layout, dtype, odt, act, None, None)


def test_library_refuses_bad_descriptors():
    d = _fake_desc
    x, w, o = d((4, 8), 2), d((8, 16), 2), d((4, 16), 2)
    bad = [
        (lin(x, d((16, 8), 2), None, None, None, None, o), "weight is"),
        (lin(x, w, None, None, None, None, d((5, 16), 2)), "x [M, K]"),
        (lin(x, w, d((8,), 2), None, None, None, o), "bias"),
        (lin(x, w, None, None, d((16,), 2), None, o), "up_bias without"),
        (lin(x, w, None, d((8, 8), 2), None, None, o), "up_weight must have"),
        (lin(x, w, None, None, None, d((4, 8), 2), o), "residual"),
        (lin(x, w, None, None, None, None, o, layout=2), "layout"),
        (lin(x, w, None, None, None, None, o, act=9), "activation"),
        (lin(x, w, None, None, None, None, o, dtype=3, odt=3), "fp32, bf16 or fp16"),
        (lin(x, w, None, None, None, None, o, odt=2), "fp32, bf16 or fp16"),
        (lin(x, w, None, None, None, None, d((4, 16), 2, strides=[8, 1])), "overlap"),
        (lin(d((4, 8), 2, strides=[1, 4]), w, None, None, None, None, o), "contiguous"),
        (lin(d((4, 0), 2), d((0, 16), 2), None, None, None, None, o), "K is zero"),
        (lin(d((4, 8), 2, device=_lib.SFB_DEVICE_CPU), w, None, None, None, None, o), "CUDA"),
        (lin(None, w, None, None, None, None, o), "NULL"),
    ]
    for rc, _ in bad:
        assert rc in (_lib.SFB_ERR_INVALID_ARG, _lib.SFB_ERR_UNSUPPORTED)
    for args, text in (((x, d((16, 8), 2), None, None, None, None, o), "weight is"), ((x, w, None, None, d((16,), 2), None, o), "up_bias without")):
        lin(*args)
        assert text in _lib.load().sfb_last_error().decode()
    assert lin(d((0, 8), 2), w, None, None, None, None, d((0, 16), 2)) == _lib.SFB_OK  # nothing to do


def rows_desc(ptr, rows, columns, stride):
    return _fake_desc((rows, columns), 2, ptr=ptr, strides=[stride, 1])


def test_shared_memory_is_refused_where_it_is_shared():
    """out over x or over part of the residual, against the sets of their elements."""
    g = random.Random(4)
    refused = allowed = 0
    for case in range(400):
        rows, k, n = g.choice([1, 2, 5]), 8, g.choice([8, 16])
        stride = g.choice([16, 24, 40])
        xs = g.choice([stride, stride, k, 0, 4])
        x0, o0 = 0x10000, 0x10000 + 2 * g.randrange(-100, 100)
        x = {x0 + 2 * (r * xs + c) for r in range(rows) for c in range(k)}
        o = {o0 + 2 * (r * stride + c) for r in range(rows) for c in range(n)}
        if stride < n or (xs != stride and xs > k and stride > n):
            continue
        rc = lin(rows_desc(x0, rows, k, xs), _fake_desc((k, n), 2, ptr=0x900000), None, None, None, None, rows_desc(o0, rows, n, stride))
        assert rc != _lib.SFB_OK  # no device here: what passes the checks fails at the launch
        assert (rc == _lib.SFB_ERR_INVALID_ARG) == bool(x & o), (rows, k, n, stride, xs, o0 - x0)
        refused, allowed = refused + bool(x & o), allowed + (not x & o)
    assert refused > 50 and allowed > 50
    x, w, o = rows_desc(0x10000, 4, 8, 8), _fake_desc((8, 16), 2, ptr=0x20000), rows_desc(0x30000, 4, 16, 16)
    assert lin(x, w, None, None, None, o, o) != _lib.SFB_ERR_INVALID_ARG  # the residual itself
    assert lin(x, w, None, None, None, rows_desc(0x30020, 4, 16, 16), o) == _lib.SFB_ERR_INVALID_ARG  # a row further on
    assert lin(x, w, None, None, None, rows_desc(0x30000, 4, 16, 0), o) == _lib.SFB_ERR_INVALID_ARG  # its first row for all
    assert "residual" in _lib.load().sfb_last_error().decode()


def test_sizes_beyond_32_bit_rows_are_refused():
    n = 2 ** 31 - 1
    assert lin(rows_desc(0x10000, n, 8, 0), _fake_desc((8, 8), 2, ptr=0x20000), None, None, None, None, rows_desc(1 << 40, n, 8, 8)) == _lib.SFB_ERR_UNSUPPORTED
    with pytest.raises(ValueError):
        ops.linear_plan(n, 8, 8)


def test_types_of_out_and_of_top_k():
    with pytest.raises(ValueError, match="out_dtype"):
        ops.fused_linear(t(4, 8), t(8, 8), out=t(4, 8), out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out_dtype"):
        ops.grouped_linear(t(4, 8), t(2, 8, 8), i32(3), out=t(4, 8), out_dtype=torch.float32)
    with pytest.raises(TypeError):
        ops.moe_route(t(4, 8), 2.5)


def test_route_workspace_query():
    assert ops.moe_route_workspace_bytes(1, 64) == 0
    assert ops.moe_route_workspace_bytes(128 * 3, 64) >= 3 * 64 * 4
    with pytest.raises(ValueError):
        ops.moe_route_workspace_bytes(-1, 4)


def test_plan_of_tile_shapes():
    plan = ops.linear_plan
    # one token against 32 column tiles: their K is shared so that the SMs are full, in one round
    p = plan(1, 4096, 4096)
    assert p["tokens"] == 32 and not p["pair"] and 96 <= p["split"] * p["feature_tiles"] <= 148
    # many tokens: clusters of two; nothing to order
    assert plan(8192, 8192, 8192) == dict(tokens=256, pair=1, split=1, order=0, blocks_an_sm=1, feature_tiles=32)
    assert plan(8192, 8192, 8192, gated=True)["feature_tiles"] == 64
    # a decode batch whose tiles outnumber the SMs: two blocks an SM
    p = plan(64, 4096, 14336, gated=True)
    assert p["blocks_an_sm"] == 2 and p["tokens"] == 64 and p["split"] == 1
    # rows by index: ordered first where groups have many, but only with room for it
    assert plan(16384, 4096, 1792, groups=32, gated=True, indexed=True)["order"] == 1
    p = plan(16384, 4096, 1792, groups=32, gated=True, indexed=True, has_workspace=False)
    assert p["order"] == 0 and p["pair"] == 0
    assert plan(128, 2048, 1408, groups=32, gated=True, indexed=True)["order"] == 0
    # no split finer than K has steps, every shape one that exists
    for rows in (1, 7, 33, 100, 129, 500, 3000):
        for k in (8, 64, 72, 1000, 8192):
            for n in (8, 128, 1000, 14336):
                for groups in (0, 1, 16, 300):
                    p = plan(rows, k, n, groups=groups, indexed=groups > 1)
                    assert p["tokens"] in (32, 64, 128, 256) and p["pair"] == (p["tokens"] == 256) and 1 <= p["split"] <= min(8, -(-k // 64))
                    assert p == plan(rows, k, n, groups=groups, indexed=groups > 1)  # the kept one is the priced one
    for bad in ((0, 8, 8), (8, 0, 8), (8, 8, 0)):
        with pytest.raises(ValueError):
            plan(*bad)
    with pytest.raises(ValueError):
        plan(8, 8, 8, groups=2000)


def test_ordering_workspace_query():
    assert ops.grouped_linear_workspace_bytes(100, 64, 32) == 0  # few rows a group: gathered
    assert ops.grouped_linear_workspace_bytes(4096, 65, 32) == 4096 * 72 * 2
    assert ops.grouped_linear_workspace_bytes(4096, 65, 32, indexed=False) == 0
    with pytest.raises(ValueError):
        ops.grouped_linear_workspace_bytes(4096, 65, 0)
