"""The feed-forward operators where a neighbour could go wrong: accumulators handed back across a cluster, and the
activations by themselves, over their whole range."""

import pytest
import torch

from test_feed_forward_gpu import BF16, assert_rounded, gen, linear64, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gated", [False, True])
def test_pair_accumulators_go_back_and_forth(gated):
    """One K step a tile and a dozen tiles a cluster: the two blocks' epilogues hand the accumulators back as fast as they can,
    and the next products overwrite them."""
    from llm_compileforge_b200 import ops

    rows, k, n = 4096, 64, 8192 if gated else 16384
    assert ops.linear_plan(rows, k, n, gated=gated)["pair"] == 1
    g = gen(11)
    x, w = make(g, rows, k), make(g, k, n, std=k ** -0.5)
    v = make(g, k, n, std=k ** -0.5) if gated else None
    got = ops.fused_linear(x, w, up_weight=v)
    for _ in range(20):
        assert torch.equal(ops.fused_linear(x, w, up_weight=v), got)
    want, tol = linear64(x, w, v=v)
    assert_rounded(got, want, tol)
