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


def values(low, high, dtype):
    """Values of a 16-bit type between low and high, dense where the type is."""
    v = torch.cat([torch.linspace(low, high, 4001), torch.linspace(max(low, -1), 1, 2001)])
    return v.to(dtype).unique().cuda()


FORMS = {  # (rows of a call, K, N, row stride of x): each form of the epilogue on the tensor cores, and the CUDA cores
    "few rows": (40, 8, 136, 8), "pairs": (9000, 1024, 4096, 1024), "K shared": (24, 1024, 136, 1024), "cuda cores": (9000, 8, 136, 9),
}


def act_alone(h, form, act, out_dtype=None, wide=False):
    """act(h) from a product whose sums are h itself: one column of x, one row of ones in the weight."""
    from llm_compileforge_b200 import ops

    rows, k, n, stride = FORMS[form]
    plan = ops.linear_plan(min(rows, len(h)), k, n)
    assert form == "cuda cores" or (plan["pair"] == 1) == (form == "pairs") and (plan["split"] > 1) == (form == "K shared")
    x = torch.zeros((len(h), stride), dtype=h.dtype, device=h.device)[:, :k]
    x[:, 0] = h
    w = torch.zeros((k, n), dtype=h.dtype, device=h.device)
    w[0] = 1
    got = torch.cat([ops.fused_linear(piece, w, activation=act, out_dtype=out_dtype) for piece in x.split(rows)])
    assert (got == got[:, :1]).all()
    return got[:, 0]


@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
@pytest.mark.parametrize("form", FORMS)
def test_erf_gelu_over_its_range(form, dtype, out_dtype):
    """On the tensor cores within 3e-7 |h| and, for negative h, within 2^-11 of the value; on the CUDA cores within 2^-15
    (erfcf of -h / sqrt 2, whose two roundings of 2^-24 and 2^-25 it multiplies by up to 2 (h^2 / 2) = 167, and 4 steps of its own)."""
    h = values(-12.875, 8, dtype)
    want = 0.5 * h.double() * torch.special.erfc(-h.double() * 0.5 ** 0.5)  # (torch's ndtr adds 1 to erf: nothing is left of it below -8)
    tol = want.abs() * 2.0 ** -15 if form == "cuda cores" else torch.minimum(3e-7 * h.double().abs(), torch.where(h < 0, want.abs() * 2.0 ** -11, 1.0))
    assert_rounded(act_alone(h, form, "gelu", out_dtype), want, tol, form)
    far = torch.tensor([-13.5, -20.0, -3e4, 20.0, 3e4], dtype=dtype, device="cuda")
    got = act_alone(far.repeat(800), form, "gelu", out_dtype).double()[:5]
    assert (got[:3].abs() < 1e-38).all() and (got[3:] == far[3:].double()).all()


@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("form", FORMS)
def test_silu_and_tanh_gelu_as_far_as_they_are_normal_numbers(form, out_dtype):
    """h / (1 + 2^t) in fp32: what t is off by, times ln 2, is the result's relative error.  silu, t = -h log2 e up to 132: half a step
    of t (2^-18) and the constant's 1.3e-8 of it, 4e-6 with the rest below 2^-17; from t = 126 on the logistic is a subnormal number of at
    least 15 bits, 2^-16 more.  tanh gelu, t up to 133: two roundings and a constant more, 2.5 steps of 2^-24 of t, 1.7e-5, and the same
    2^-16: below 2^-14."""
    h = values(-91.5, 30, BF16)
    tol = torch.where(h > -87, 2.0 ** -17, 2.0 ** -15)
    want = h.double() * torch.special.expit(h.double())
    assert_rounded(act_alone(h, form, "silu", out_dtype), want, want.abs() * tol, form)
    h = values(-10.0625, 10, BF16)
    d = h.double()
    want = d * torch.special.expit(2 * (2 / torch.pi) ** 0.5 * (d + 0.044715 * d ** 3))
    assert_rounded(act_alone(h, form, "gelu_tanh", out_dtype), want, want.abs() * 2.0 ** -14, form)
    far = torch.tensor([-3e38, -1e4, 1e-37, -1e-37, 1e4, 3e38], dtype=BF16, device="cuda")
    for act in ("silu", "gelu_tanh"):
        got = act_alone(far.repeat(800), form, act, out_dtype).double()[:6]
        assert (got[:2] == 0).all() and (got[4:] == far[4:].double()).all()
        assert ((got[2:4] - far[2:4].double() / 2).abs() <= 2.0 ** -8 * 1e-37).all()
