"""More refusals of the feed-forward operators, without a GPU: every call here ends before a launch."""

import ctypes

import pytest
import torch

from llm_compileforge_b200 import B200Backend, _lib, ops
from test_abi_cpu import _fake_desc

TOKENS, EXPERTS, TOP = 300, 16, 2


def route(workspace, n_bytes):
    lib = _lib.load()
    descs = [_fake_desc((TOKENS, EXPERTS), 4), _fake_desc((TOKENS, TOP), 4), _fake_desc((TOKENS, TOP), 4), _fake_desc((EXPERTS + 1,), 4),
             _fake_desc((TOKENS * TOP,), 4), _fake_desc((TOKENS, TOP), 4)]
    return lib.sfb_moe_route(*(ctypes.cast(ctypes.pointer(d), ctypes.c_void_p) for d in descs), _lib.SFB_F32, 1, workspace, n_bytes, None)


@pytest.mark.parametrize("odd", [1, 2, 3, 5])
def test_route_workspace_off_four_bytes_is_refused(odd):
    need = ops.moe_route_workspace_bytes(TOKENS, EXPERTS)
    assert need > 0
    assert route(0x10000 + odd, need) == _lib.SFB_ERR_INVALID_ARG
    assert "4 bytes" in _lib.load().sfb_last_error().decode()
    assert route(0x10000 + odd, need - 1) == _lib.SFB_ERR_WORKSPACE


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2],
                                       torch.zeros(1024, 512, dtype=torch.uint8).t()])
def test_workspaces_that_are_not_one_piece_are_refused(workspace):
    x, w, index = torch.zeros(64, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.moe_route(torch.zeros(TOKENS, EXPERTS), TOP, workspace=workspace)
    with pytest.raises(ValueError, match="contiguous"):
        ops.grouped_linear(x, w, torch.zeros(3, dtype=torch.int32), row_index=index, workspace=workspace)


def test_executor_refuses_operands_that_it_does_not_take():
    hal = B200Backend()
    x, w, b, r = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8), torch.zeros(4, 8)
    i = torch.zeros(4, 2, dtype=torch.int32)
    for name, inputs in (("fused_linear", [x, w, b, r]), ("fused_linear", [x]), ("grouped_linear", [x, w[None], i[0], b[None], w[None]]), ("grouped_linear", [x, w[None]]),
                         ("moe_route", [x, x]), ("moe_route", []), ("moe_combine", [x, i, torch.zeros(4, 2), r]), ("moe_combine", [x, i])):
        with pytest.raises(ValueError, match=f"{name}: .* inputs"):
            hal.execute(name, inputs, **({"top_k": 2} if name == "moe_route" else {}))


def test_executor_asks_for_top_k():
    with pytest.raises(ValueError, match="top_k"):
        B200Backend().execute("moe_route", [torch.zeros(4, 8)])
