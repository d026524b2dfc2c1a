"""The feed-forward operators against plain 64-bit implementations of their definitions.

Tolerance of a product: 16-bit products are exact in fp32 and the sums are fp32; an accumulator is rounded once per 16 terms
on the tensor cores (once per term, to nearest, on the CUDA cores, which averages out), by at most 2^-23 of the sum of
magnitudes S = sum |x w| + |b|, and 32 steps are allowed for the products inside a group of terms and for the activation:
(K / 16 + 32) 2^-23 S.  An activation passes an error on by at most 1.13, a gate multiplies it.  The result is rounded once:
half a step of its type, eps / 2 of its value.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def act64(h, name):
    if name == "silu":
        return h * torch.special.expit(h)
    if name == "gelu":
        return h * torch.special.ndtr(h)
    if name == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3)))
    return h.clamp(min=0) if name == "relu" else h


def linear64(x, w, b=None, act="none", v=None, c=None, r=None):
    """Value and tolerance (before the final rounding) of one product, from CPU or GPU tensors."""
    d = lambda t: t.double()  # noqa: E731
    x = d(x)
    steps = (x.shape[-1] / 16 + 32) * 2.0 ** -23

    def product(m, bias):
        h, s = x @ d(m), x.abs() @ d(m).abs()
        return (h, s) if bias is None else (h + d(bias), s + d(bias).abs())

    h, s = product(w, b)
    y, tol = act64(h, act), 1.13 * steps * s
    if v is not None:
        u, su = product(v, c)
        y, tol = y * u, tol * u.abs() + y.abs() * steps * su
    if r is not None:
        y = y + d(r)
        tol = tol + y.abs() * 2.0 ** -23
    return y, tol


def assert_rounded(got, want, tol, what=""):
    """got is want, off by at most tol before one rounding to got's type."""
    half = torch.finfo(got.dtype).eps / 2
    allowed = tol + half * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * half * 2
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (off <= allowed).all(), f"{what}: off by {off.max().item():.3e}, {(off / allowed).max().item():.2f} of what is allowed"


def make(g, *shape, dtype=BF16, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(g, *lead, k, n, dtype, layout, pad=0):
    """[.., k, n] with n (kn) or k (nk) contiguous; rows of `pad` more values than they need."""
    if layout == "nk":
        return make(g, *lead, n, k + pad, dtype=dtype, std=k ** -0.5)[..., :k].transpose(-1, -2)
    return make(g, *lead, k, n + pad, dtype=dtype, std=k ** -0.5)[..., :n]


def check_linear(rows, k, n, *, dtype=BF16, layout="kn", act="none", gated=False, bias=False, residual=False, out_dtype=None, pad=0):
    from llm_compileforge_b200 import ops

    g = gen(rows * 7 + k * 3 + n)
    x = make(g, rows, k + pad, dtype=dtype)[:, :k]
    w = matrix(g, k=k, n=n, dtype=dtype, layout=layout, pad=pad)
    v = matrix(g, k=k, n=n, dtype=dtype, layout=layout, pad=pad) if gated else None
    b = make(g, n, dtype=dtype) if bias else None
    c = make(g, n, dtype=dtype) if bias and gated else None
    odt = out_dtype or dtype
    r = make(g, rows, n, dtype=odt) if residual else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    wide = torch.full((rows, n + 24), 7.0, dtype=odt, device="cuda")  # the result as columns 8 .. n + 8 of a wider matrix
    got = ops.fused_linear(x, w, b, activation=act, up_weight=v, up_bias=c, residual=r, out=wide[:, 8:8 + n], status=status)
    want, tol = linear64(x, w, b, act, v, c, r)
    assert_rounded(got, want, tol, f"{rows}x{k}x{n}")
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + n:] == 7).all(), "wrote beside its rows"
    again = ops.fused_linear(x, w, b, activation=act, up_weight=v, up_bias=c, residual=r, out_dtype=odt)
    assert torch.equal(again, got) and again.dtype == odt
    assert status.item() == 0


ROWS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 100, 127, 128, 129, 192, 255, 256, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_linear_rows(rows, layout):
    check_linear(rows, 320, 200, layout=layout, bias=True, residual=True, act="silu")


@pytest.mark.parametrize("k", [8, 16, 56, 64, 72, 128, 136, 1000, 4096, 8200])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_linear_depth(k, layout):
    for rows in (3, 70, 200):
        check_linear(rows, k, 136, layout=layout, gated=True, act="silu")


@pytest.mark.parametrize("n", [8, 16, 40, 64, 72, 120, 128, 136, 256, 264, 1000, 4104])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_width(n, gated):
    for rows, layout in ((1, "nk"), (40, "kn"), (140, "nk"), (260, "kn")):
        check_linear(rows, 192, n, layout=layout, gated=gated, bias=True, act="gelu")


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_activations_and_types(act, dtype, gated):
    check_linear(37, 264, 88, dtype=dtype, act=act, gated=gated, bias=True, residual=True)
    check_linear(150, 64, 88, dtype=dtype, act=act, gated=gated, bias=True, residual=not gated, out_dtype=F32, layout="nk")


@pytest.mark.parametrize("rows,k,n", [(1, 7, 5), (5, 1, 1), (3, 33, 130), (129, 65, 67), (64, 1001, 63)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_linear_odd_sizes(rows, k, n, layout):
    check_linear(rows, k, n, layout=layout, gated=True, bias=True, residual=True, act="gelu_tanh")
    check_linear(rows, k, n, layout=layout, dtype=F32)


@pytest.mark.parametrize("k,n", [(63, 101), (65, 100), (200, 33), (9, 6)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_linear_odd_sizes_in_padded_rows(k, n, layout):
    """Odd K and N in matrices whose rows start on 16 bytes."""
    inner = k if layout == "nk" else n
    if (-k) % 8 != (-inner) % 8:  # one pad serves x and the weight
        k = k + (-k) % 8 + (-((-inner) % 8)) % 8
        inner = k if layout == "nk" else n
    for rows in (1, 20, 300):
        check_linear(rows, k, n, layout=layout, pad=(-inner) % 8, bias=True, residual=True)
        check_linear(rows, k, n, layout=layout, pad=(-inner) % 8, gated=True, act="silu")


@pytest.mark.parametrize("rows,k,n,gated", [(2050, 512, 1288, False), (4100, 256, 2568, False), (3000, 192, 1160, True), (777, 2048, 1024, False)])
def test_linear_many_tiles(rows, k, n, gated):
    for layout in ("kn", "nk"):
        check_linear(rows, k, n, layout=layout, gated=gated, act="silu" if gated else "none", residual=not gated)


def test_linear_residual_in_place_leading_dimensions_and_empty():
    from llm_compileforge_b200 import ops

    g = gen(5)
    x, w, h = make(g, 3, 50, 128), make(g, 128, 96, std=0.1), make(g, 3, 50, 96)
    want, tol = linear64(x, w, r=h)
    got = ops.fused_linear(x, w, residual=h, out=h)
    assert got.data_ptr() == h.data_ptr() and got.shape == (3, 50, 96)
    assert_rounded(h, want, tol)
    one = ops.fused_linear(x[0, 0], w)
    assert one.shape == (96,) and torch.equal(one, ops.fused_linear(x[0, :1], w)[0])
    assert ops.fused_linear(x[:0], w).shape == (0, 50, 96)
    assert ops.fused_linear(x, w[:, :0]).shape == (3, 50, 0)
    cols = make(g, 128, 50).t()  # x with its rows strewn: copied into rows first
    want, tol = linear64(cols, w)
    assert_rounded(ops.fused_linear(cols, w), want, tol)


def test_linear_keeps_infinities_and_nan_in_their_rows():
    from llm_compileforge_b200 import ops

    g = gen(6)
    for rows in (5, 150):
        x, w = make(g, rows, 64), make(g, 64, 72, std=0.1)
        x[2, 3] = float("nan")
        x[4, 5] = float("inf")
        got = ops.fused_linear(x, w)
        assert got[2].isnan().all() and not got[4].isfinite().any()
        keep = [i for i in range(rows) if i not in (2, 4)]
        assert torch.equal(got[keep], ops.fused_linear(x[keep], w)) if rows == 5 else torch.isfinite(got[keep]).all()


@pytest.mark.parametrize("rows", [5, 40, 100, 200, 600, 1100])
@pytest.mark.parametrize("k,n", [(4096, 256), (2048, 101)])
def test_linear_every_output_form(rows, k, n):
    """fp32 and 16-bit results in whole pieces and value by value, on the shapes that split K, walk tiles and pair blocks."""
    pad = (-n) % 8 if n % 8 else 0
    k += (-(k + pad)) % 8
    for gated in (False, True):
        check_linear(rows, k, n, gated=gated, act="silu", bias=True, residual=True, out_dtype=F32, pad=pad)
        check_linear(rows, k, n, gated=gated, act="relu", residual=True, dtype=F16, pad=pad)


def test_linear_broadcast_and_unaligned_operands():
    from llm_compileforge_b200 import ops

    g = gen(21)
    w, b = make(g, 136, 96, std=0.1), make(g, 96)
    for rows in (6, 300):
        x = make(g, rows, 144)
        one = x[:1, :136].expand(rows, 136)  # rows that all lie in one place
        want, tol = linear64(one, w, b)
        assert_rounded(ops.fused_linear(one, w, b), want, tol)
        r = make(g, 1, 96).expand(rows, 96)
        want, tol = linear64(x[:, :136], w, r=r)
        assert_rounded(ops.fused_linear(x[:, :136], w, residual=r), want, tol)
        for shift in (1, 3):  # bases off 16 bytes
            xs = x[:, shift:136 + shift]
            want, tol = linear64(xs, w, b)
            assert_rounded(ops.fused_linear(xs, w, b), want, tol)
        flat = torch.zeros(rows * 100 + 8, dtype=BF16, device="cuda")
        out = flat[1:1 + rows * 100].view(rows, 100)[:, 3:99]  # rows of out off every piece
        ops.fused_linear(x[:, :136], w, b, out=out)
        want, tol = linear64(x[:, :136], w, b)
        assert_rounded(out, want, tol)
        assert flat[0] == 0 and (flat[1 + rows * 100:] == 0).all()


# ── grouped ──────────────────────────────────────────────────────────────────
def offsets_of(counts, first=0):
    at = [first]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def check_grouped(counts, k, n, *, dtype=BF16, layout="kn", act="none", gated=False, bias=False, gather=False, x_rows=None, first=0, behind=0,
                  out_dtype=None, pad=0):
    from llm_compileforge_b200 import ops

    e, rows = len(counts), first + sum(counts) + behind
    g = gen(sum(counts) * 5 + k + n + e)
    x_rows = x_rows or max(1, rows // 2) if gather else rows
    x = make(g, x_rows, k + pad, dtype=dtype)[:, :k]
    w = matrix(g, e, k=k, n=n, dtype=dtype, layout=layout, pad=pad)
    v = matrix(g, e, k=k, n=n, dtype=dtype, layout=layout, pad=pad) if gated else None
    b = make(g, e, n, dtype=dtype) if bias else None
    c = make(g, e, n, dtype=dtype) if bias and gated else None
    index = torch.randint(0, x_rows, (rows,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    odt = out_dtype or dtype
    wide = torch.full((rows, n + 16), 3.0, dtype=odt, device="cuda")
    offsets = offsets_of(counts, first)
    got = ops.grouped_linear(x, w, offsets, b, activation=act, up_weight=v, up_bias=c, row_index=index, out=wide[:, 8:8 + n], status=status)
    at = first
    for i, m in enumerate(counts):
        xi = x[at:at + m] if index is None else x[index[at:at + m].long()]
        want, tol = linear64(xi, w[i], b[i] if bias else None, act, v[i] if gated else None, c[i] if c is not None else None)
        if m:
            assert_rounded(got[at:at + m], want, tol, f"group {i} of {counts}")
        at += m
    assert (wide[:first] == 3).all() and (wide[at:] == 3).all() and (wide[:, :8] == 3).all() and (wide[:, 8 + n:] == 3).all(), "wrote outside the groups"
    assert status.item() == 0
    again = ops.grouped_linear(x, w, offsets, b, activation=act, up_weight=v, up_bias=c, row_index=index, out_dtype=odt)
    assert torch.equal(again[first:at], got[first:at])


COUNTS = [[1], [0, 0, 5, 0], [1, 1, 1, 1, 1, 1, 1, 1], [3, 0, 17, 16, 1, 0, 33, 8], [0, 130, 0, 1], [257, 31, 64, 0], [16] * 20, [300, 2, 0, 700], [128, 128, 256]]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_counts(counts, layout, gather):
    check_grouped(counts, 264, 200, layout=layout, gather=gather, bias=True, act="silu")
    check_grouped(counts, 128, 72, layout=layout, gather=gather, gated=True, act="silu", first=3, behind=21)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_types(dtype, gated):
    check_grouped([5, 0, 40, 9], 96, 104, dtype=dtype, gated=gated, bias=True, act="gelu", gather=True)
    check_grouped([150, 1, 290], 72, 264, dtype=dtype, gated=gated, act="relu", out_dtype=F32, layout="nk")


@pytest.mark.parametrize("k,n", [(7, 5), (33, 66), (64, 9)])
def test_grouped_odd_sizes(k, n):
    for layout in ("kn", "nk"):
        check_grouped([5, 0, 70, 1], k, n, layout=layout, gated=True, bias=True, gather=True, behind=2)


@pytest.mark.parametrize("experts", [1, 2, 64, 257, 1024])
def test_grouped_many_groups(experts):
    counts = [(i * 7) % 5 for i in range(experts)]
    counts[-1] += 40
    check_grouped(counts, 64, 72, gather=True, act="silu")


def test_grouped_large():
    check_grouped([900, 0, 513, 1100, 256, 31], 512, 1032, gather=True, x_rows=700)
    check_grouped([900, 0, 513, 1100, 256, 31], 320, 520, gated=True, act="silu", layout="nk", gather=True, x_rows=700)


def test_grouped_same_row_for_every_entry_and_no_rows():
    from llm_compileforge_b200 import ops

    g = gen(9)
    x, w = make(g, 4, 64), make(g, 3, 64, 40, std=0.1)
    index = torch.full((50,), 2, dtype=torch.int32, device="cuda")
    got = ops.grouped_linear(x, w, offsets_of([20, 0, 30]), row_index=index)
    for e, part in ((0, got[:20]), (2, got[20:])):
        want, tol = linear64(x[2:3], w[e])
        assert_rounded(part, want.expand(part.shape), tol.expand(part.shape))
    assert ops.grouped_linear(x[:0], w, offsets_of([0, 0, 0])).shape == (0, 40)
    out = torch.full((4, 40), 5.0, dtype=BF16, device="cuda")
    assert (ops.grouped_linear(x, w, offsets_of([0, 0, 0]), out=out) == 5).all()


def test_grouped_bad_offsets_and_indices_are_flagged_and_stay_inside():
    from llm_compileforge_b200 import _lib, ops

    g = gen(10)
    for k in (64, 63):  # both routes
        x, w = make(g, 40, k), make(g, 4, k, 72, std=0.1)
        for bad in ([0, 10, 50, 50, 50], [-3, 10, 20, 30, 40], [0, 30, 10, 40, 40], [0, 2 ** 31 - 1, 40, -2 ** 31, 7]):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = torch.full((48, 72), 3.0, dtype=BF16, device="cuda")
            ops.grouped_linear(x, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), out=out[:40], status=status)
            assert status.item() == _lib.SFB_STATUS_BAD_ROW_INDEX and (out[40:] == 3).all()
        index = torch.arange(40, dtype=torch.int32, device="cuda")
        index[7], index[33] = 40, -1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = ops.grouped_linear(x, w, offsets_of([10, 10, 10, 10]), row_index=index, status=status)
        assert status.item() == _lib.SFB_STATUS_BAD_ROW_INDEX
        want, tol = linear64(x[:1], w[0])
        assert_rounded(got[7:8], want, tol)
        keep = [i for i in range(40) if i not in (7, 33)]
        fine = ops.grouped_linear(x, w, offsets_of([10, 10, 10, 10]), row_index=torch.arange(40, dtype=torch.int32, device="cuda"))
        assert torch.equal(got[keep], fine[keep])


def test_grouped_many_groups_of_many_rows():
    for counts in ([90 + i % 40 for i in range(1024)], [300] * 200 + [0] * 57):
        check_grouped(counts, 64, 72, gather=True, x_rows=5000)
        check_grouped(counts, 64, 40, gated=True, act="silu", layout="nk")


def test_grouped_without_room_to_order_rows():
    from llm_compileforge_b200 import ops

    g = gen(31)
    counts = [140, 0, 260, 33]
    x, w, v = make(g, 200, 328), make(g, 4, 328, 264, std=0.06), make(g, 4, 328, 264, std=0.06)
    index = torch.randint(0, 200, (sum(counts),), generator=g, device="cuda", dtype=torch.int32)
    for gate in (None, v):
        ordered = ops.grouped_linear(x, w, offsets_of(counts), row_index=index, up_weight=gate)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        small = torch.empty(16, dtype=torch.uint8, device="cuda")
        assert ops.grouped_linear_workspace_bytes(sum(counts), 328, 4) > 16
        gathered = ops.grouped_linear(x, w, offsets_of(counts), row_index=index, up_weight=gate, workspace=small, status=status)
        at = 0
        for i, m in enumerate(counts):
            want, tol = linear64(x[index[at:at + m].long()], w[i], None, "none", None if gate is None else gate[i])
            assert_rounded(gathered[at:at + m], want, tol)
            assert_rounded(ordered[at:at + m], want, tol)
            at += m
        assert status.item() == 0


def test_grouped_broadcast_over_the_experts_and_nan_rows():
    from llm_compileforge_b200 import ops

    g = gen(32)
    for counts in ([7, 0, 20, 3], [200, 90, 0, 130]):
        x = make(g, sum(counts), 64)
        w, b = make(g, 1, 64, 72, std=0.1).expand(4, 64, 72), make(g, 1, 72).expand(4, 72)
        want, tol = linear64(x, w[0], b[0])
        assert_rounded(ops.grouped_linear(x, w, offsets_of(counts), b), want, tol)
        w = make(g, 4, 64, 72, std=0.1)
        clean = ops.grouped_linear(x, w, offsets_of(counts), b)
        x[counts[0] - 1] = math.nan  # the last row of a group: its tile also covers the next group's first rows
        got = ops.grouped_linear(x, w, offsets_of(counts), b)
        keep = [i for i in range(sum(counts)) if i != counts[0] - 1]
        assert got[counts[0] - 1].isnan().all() and torch.equal(got[keep], clean[keep])


# ── routing ──────────────────────────────────────────────────────────────────
def route_plain(logits, top_k, renormalize):
    rows = logits.double().cpu().tolist()
    n, e = len(rows), logits.shape[1]
    ids = torch.full((n, top_k), -1, dtype=torch.int32)
    weights = torch.zeros((n, top_k), dtype=torch.float64)
    groups = [[] for _ in range(e)]
    for t, row in enumerate(rows):
        order = sorted((-v, i) for i, v in enumerate(row) if v > -math.inf)  # NaN compares false
        if not order:
            continue
        top = -order[0][0]
        ex = lambda v: (1.0 if v == math.inf else 0.0) if top == math.inf else math.exp(v - top)  # noqa: E731
        total = sum(ex(-v) for v, _ in (order[:top_k] if renormalize else order))
        for j, (v, i) in enumerate(order[:top_k]):
            ids[t, j], weights[t, j] = i, ex(-v) / total
            groups[i].append((t, j))
    offsets = torch.zeros(e + 1, dtype=torch.int32)
    token_rows = torch.full((n * top_k,), -1, dtype=torch.int32)
    positions = torch.full((n, top_k), -1, dtype=torch.int32)
    at = 0
    for i, members in enumerate(groups):
        for t, j in members:
            token_rows[at], positions[t, j] = t, at
            at += 1
        offsets[i + 1] = at
    return ids, weights, offsets, token_rows, positions


def check_route(logits, top_k, renormalize=True):
    from llm_compileforge_b200 import ops

    got = ops.moe_route(logits, top_k, renormalize=renormalize)
    want = route_plain(logits, top_k, renormalize)
    for name, a, b in zip(got._fields, got, want):
        if name == "weights":
            # expf is within 2 steps, the sum of at most 1024 terms of one sign within 10 (a tree of 5 levels over 32 terms each at
            # most), the quotient within half a step of 2^-23: 16 steps are allowed
            assert a.dtype == F32 and ((a.cpu().double() - b).abs() <= 16 * 2.0 ** -23 * b + 1e-37).all()
        else:
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name


@pytest.mark.parametrize("tokens", [1, 2, 31, 127, 128, 129, 1000])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (8, 2), (33, 5), (64, 8), (65, 32), (128, 8), (256, 8), (300, 6), (1024, 4)])
def test_route(tokens, experts, top_k):
    logits = make(gen(tokens + experts), tokens, experts, dtype=F32, std=2.0)
    check_route(logits, top_k)
    check_route(logits.to(BF16), top_k, renormalize=False)  # many equal logits among them


def test_route_masks_ties_infinities_and_nan():
    g = gen(3)
    for tokens in (6, 400):
        logits = make(g, tokens, 40, dtype=F32)
        logits[0] = -math.inf
        logits[1, :38] = -math.inf
        logits[2] = 0.0
        logits[2, ::2] = -0.0  # ties with +0
        logits[3, 7] = math.nan
        logits[4, 9] = logits[4, 30] = math.inf
        logits[5] = torch.finfo(F32).min  # a finite lowest value is a candidate
        logits[:, 11] = -math.inf
        for renormalize in (True, False):
            check_route(logits, 6, renormalize)
    check_route(torch.full((300, 16), -math.inf, device="cuda"), 2)
    check_route(torch.zeros((300, 16), device="cuda", dtype=BF16), 2)
    check_route(make(g, 200, 48, dtype=F16)[:, 8:40], 4)  # rows of a wider matrix


def test_route_many_tokens_and_none():
    from llm_compileforge_b200 import ops

    check_route(make(gen(4), 20000, 24, dtype=F16), 3)
    r = ops.moe_route(torch.zeros((0, 8), device="cuda"), 2)
    assert r.expert_ids.shape == (0, 2) and r.token_rows.numel() == 0 and r.group_offsets.tolist() == [0] * 9


# ── combining ────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,top_k,h", [(1, 1, 8), (5, 2, 24), (33, 8, 200), (64, 9, 1024), (7, 32, 72), (300, 4, 2056), (3, 3, 7), (2, 2, 4099)])
def test_combine(dtype, tokens, top_k, h):
    from llm_compileforge_b200 import ops

    g = gen(tokens + top_k + h)
    y = make(g, tokens * top_k + 3, h, dtype=dtype)
    positions = torch.randperm(tokens * top_k + 3, generator=g, device="cuda")[:tokens * top_k].to(torch.int32).view(tokens, top_k)
    weights = torch.rand((tokens, top_k), generator=g, device="cuda")
    gone = torch.rand((tokens, top_k), generator=g, device="cuda") < 0.2
    positions = torch.where(gone, -1, positions)
    weights = torch.where(gone & (torch.rand_like(weights) < 0.5), math.nan, weights)  # the weight of nothing is not read as a number
    picked = torch.where(gone[..., None], 0.0, y[positions.clamp(min=0).long()].double())
    terms = torch.where(gone, 0.0, weights.double())[..., None] * picked
    for r in (None, make(g, tokens, h, dtype=dtype)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = ops.moe_combine(y, positions, weights, residual=r, status=status)
        want = terms.sum(1) + (0 if r is None else r.double())
        size = terms.abs().sum(1) + (0 if r is None else r.double().abs())
        assert_rounded(got, want, (top_k + 1) * 2.0 ** -24 * size)  # an fma each, and the residual's addition
        assert status.item() == 0
    view = torch.full((tokens, h + 16), 2.0, dtype=dtype, device="cuda")
    view[:, 8:8 + h] = r
    assert torch.equal(ops.moe_combine(y, positions, weights, residual=view[:, 8:8 + h], out=view[:, 8:8 + h]), got)
    assert (view[:, :8] == 2).all() and (view[:, 8 + h:] == 2).all()


@pytest.mark.parametrize("tokens,top_k,h,with_residual", [(2000, 32, 1024, False), (3000, 32, 256, True), (1500, 20, 2048, True), (1200, 17, 512, False), (5000, 16, 128, True)])
def test_combine_many_tokens_of_many_rows(tokens, top_k, h, with_residual):
    """Every token's rows go round the ring more than once, in several batches, many tokens after one another in a block."""
    from llm_compileforge_b200 import ops

    g = gen(tokens + h)
    y, weights = make(g, tokens * top_k, h), torch.rand((tokens, top_k), generator=g, device="cuda")
    positions = torch.randperm(tokens * top_k, generator=g, device="cuda").to(torch.int32).view(tokens, top_k)
    r = make(g, tokens, h) if with_residual else None
    terms = weights.double()[..., None] * y[positions.long()].double()
    want, size = terms.sum(1), terms.abs().sum(1)
    if with_residual:
        want, size = want + r.double(), size + r.double().abs()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        assert_rounded(ops.moe_combine(y, positions, weights, residual=r, status=status), want, (top_k + 1) * 2.0 ** -24 * size)
    assert status.item() == 0


def test_combine_bad_positions_empty_rows_and_no_tokens():
    from llm_compileforge_b200 import _lib, ops

    y = make(gen(2), 6, 64)
    positions = torch.tensor([[0, 6], [-2, 1], [-1, -1]], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.moe_combine(y, positions, torch.ones((3, 2), device="cuda"), status=status)
    assert status.item() == _lib.SFB_STATUS_BAD_ROW_INDEX
    assert torch.equal(got[0], y[0]) and torch.equal(got[1], y[1]) and (got[2] == 0).all()
    assert ops.moe_combine(y, positions[:0], torch.ones((0, 2), device="cuda")).shape == (0, 64)
    assert (ops.moe_combine(y[:0], torch.full((2, 2), -1, dtype=torch.int32, device="cuda"), torch.ones((2, 2), device="cuda")) == 0).all()


# ── together ─────────────────────────────────────────────────────────────────
def moe_block(be, x, router, w1, w3, w2, top_k):
    """Router, gated experts and combine on the residual stream, through the operator names of the executor."""
    route = be.execute("moe_route", [be.execute("fused_linear", [x, router], out_dtype=F32)], top_k=top_k)
    h = be.execute("grouped_linear", [x, w1, route.group_offsets], up_weight=w3, activation="silu", row_index=route.token_rows)
    y = be.execute("grouped_linear", [h, w2, route.group_offsets])
    return route, h, y, be.execute("moe_combine", [y, route.positions, route.weights], residual=x)


@pytest.mark.parametrize("tokens", [1, 30, 500])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_routed_feed_forward(tokens, dtype):
    import llm_compileforge_b200 as pkg

    g, hidden, inner, experts, top_k = gen(tokens), 256, 136, 12, 3
    x = make(g, tokens, hidden, dtype=dtype)
    router = matrix(g, k=hidden, n=experts, dtype=dtype, layout="nk")
    w1, w3 = (matrix(g, experts, k=hidden, n=inner, dtype=dtype, layout="nk") for _ in range(2))
    w2 = matrix(g, experts, k=inner, n=hidden, dtype=dtype, layout="nk")
    route, h, y, out = moe_block(pkg.B200Backend(), x, router, w1, w3, w2, top_k)
    # the routing from the logits that the router's product gave; every later step from the step before it as it was stored
    at = route.group_offsets.tolist()
    for e in range(experts):
        rows = slice(at[e], at[e + 1])
        if at[e] == at[e + 1]:
            continue
        want, tol = linear64(x[route.token_rows[rows].long()], w1[e], None, "silu", w3[e])
        assert_rounded(h[rows], want, tol, "experts, first half")
        assert_rounded(y[rows], *linear64(h[rows], w2[e]), "experts, second half")
    want = (route.weights.double()[..., None] * y[route.positions.long()].double()).sum(1) + x.double()
    size = (route.weights.double()[..., None] * y[route.positions.long()].double().abs()).sum(1) + x.double().abs()
    assert_rounded(out, want, 4 * 2.0 ** -24 * size, "combined")
    # and against the whole block in 64 bits on the same routing: three roundings to the 16-bit type on the way, each at most half
    # a step of what it rounds, so eps * the sum of magnitudes that the second product and the combine see
    xd, whole, mag = x.double(), x.double().clone(), x.double().abs()
    for t in range(tokens):
        for j in range(top_k):
            e = int(route.expert_ids[t, j])
            a = act64(xd[t] @ w1[e].double(), "silu") * (xd[t] @ w3[e].double())
            wgt = route.weights[t, j].double()
            whole[t] += wgt * (a @ w2[e].double())
            mag[t] += wgt * (a.abs() @ w2[e].double().abs())
    assert ((out.double() - whole).abs() <= torch.finfo(dtype).eps * mag + 1e-6).all()


def test_dense_layer_behind_the_norm():
    """fused_rms_norm_matmul's sibling: norm, gated half, second half back onto the residual stream."""
    from llm_compileforge_b200 import ops

    g = gen(12)
    for rows in (3, 280):
        x = make(g, rows, 256)
        norm_w = make(g, 256)
        w1, w3, w2 = make(g, 256, 520, std=0.06), make(g, 256, 520, std=0.06), make(g, 520, 256, std=0.04)
        h = ops.rms_norm(x, norm_w)
        a = ops.fused_linear(h, w1, up_weight=w3, activation="silu")
        assert_rounded(a, *linear64(h, w1, None, "silu", w3))
        want, tol = linear64(a, w2, r=x)
        ops.fused_linear(a, w2, residual=x, out=x)
        assert_rounded(x, want, tol)


def test_captured_graphs_streams_and_changed_inputs():
    """Two graphs over one set of weights, replayed in turn with new inputs, give what the eager calls give; so does another stream."""
    import llm_compileforge_b200 as pkg

    be, g, top_k = pkg.B200Backend(), gen(8), 2
    for tokens in (4, 300):
        x = make(g, tokens, 128)
        router, w1, w3, w2 = make(g, 128, 8, std=0.2), make(g, 8, 128, 200, std=0.1), make(g, 8, 128, 200, std=0.1), make(g, 8, 200, 128, std=0.1)
        moe_block(be, x, router, w1, w3, w2, top_k)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = moe_block(be, x, router, w1, w3, w2, top_k)
            graphs.append((graph, held))
        for step in range(4):
            x.copy_(make(g, tokens, 128))
            want = moe_block(be, x, router, w1, w3, w2, top_k)[-1]
            for graph, held in graphs:
                held[-1].fill_(9)
                graph.replay()
                assert torch.equal(held[-1], want), step
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = moe_block(be, x, router, w1, w3, w2, top_k)[-1]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)


def test_calls_on_two_streams_at_once():
    import llm_compileforge_b200 as pkg

    be, g, top_k = pkg.B200Backend(), gen(14), 2
    router, w1, w3, w2 = make(g, 128, 8, std=0.2), make(g, 8, 128, 200, std=0.1), make(g, 8, 128, 200, std=0.1), make(g, 8, 200, 128, std=0.1)
    xs = [make(g, 400, 128) for _ in range(2)]
    want = [moe_block(be, x, router, w1, w3, w2, top_k)[-1] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(moe_block(be, xs[i], router, w1, w3, w2, top_k)[-1])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_results_behind_other_kernels():
    """A chain of calls with torch kernels that write their inputs right before them, without a pause: each call waits for what it reads."""
    from llm_compileforge_b200 import ops

    g = gen(15)
    x, w = make(g, 64, 512), make(g, 512, 512, std=0.04)
    want = x
    for _ in range(6):
        want = ops.fused_linear((want * 0.5).contiguous(), w, residual=want)
        torch.cuda.synchronize()
    for _ in range(10):
        h = x
        for _ in range(6):
            h = ops.fused_linear((h * 0.5).contiguous(), w, residual=h)
        assert torch.equal(h, want)


def test_offsets_past_32_bits():
    """Rows, experts and results 2^26 elements apart, so that the last lie more than 2^31 elements behind the first."""
    from llm_compileforge_b200 import ops

    g, rows, apart, k, n = gen(50), 40, 2 ** 26, 128, 72
    buffer = torch.empty(rows * apart, dtype=BF16, device="cuda")

    def far(first, columns, fill=None):
        view = buffer.as_strided((rows, columns), (apart, 1), first)
        if fill is not None:
            view.copy_(fill)
        return view

    for odd in (0, 1):  # 1: bases that only the CUDA cores take
        x, r = far(odd, k, make(g, rows, k)), far(1024 + odd, n, make(g, rows, n))
        experts = buffer.as_strided((rows, k, n), (apart, n, 1), 4096)
        experts.copy_(make(g, rows, k, n, std=k ** -0.5))
        out = far(2048 + odd, n)
        want, tol = linear64(x, experts[-1], r=r)
        ops.fused_linear(x, experts[-1], residual=r, out=out)
        assert_rounded(out, want, tol, "dense")
        offsets, index = torch.arange(rows + 1, dtype=torch.int32, device="cuda"), torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda")
        ops.grouped_linear(x, experts, offsets, row_index=index, out=out)
        for e in (0, 20, rows - 1):
            want, tol = linear64(x[rows - 1 - e:rows - e], experts[e])
            assert_rounded(out[e:e + 1], want, tol, f"expert {e}")
        positions, weights = torch.stack([index, index], 1).contiguous(), torch.rand(rows, 2, generator=g, device="cuda")
        ops.moe_combine(x, positions, weights, residual=far(512 + odd, k, make(g, rows, k)), out=far(6144 * 4 + odd, k))
        near = ops.moe_combine(x.contiguous(), positions, weights, residual=far(512 + odd, k).contiguous())
        assert torch.equal(far(6144 * 4 + odd, k), near)
        got, want = ops.moe_route(x, 4), ops.moe_route(x.contiguous(), 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_grouped_operands_written_right_before():
    """Weights, offsets, indices and rows that the kernel right before the call has written, where rows are ordered first (the product
    then starts beside that pass) and where they are gathered."""
    from llm_compileforge_b200 import ops

    g = gen(52)
    for rows, experts, ordered in ((2000, 4, 1), (12000, 8, 1), (40, 8, 0)):
        assert ops.linear_plan(rows, 256, 320, groups=experts, indexed=True)["order"] == ordered
        versions = []
        for _ in range(2):
            x, w = make(g, 300, 256), make(g, experts, 256, 320, std=0.06)
            offsets = offsets_of(torch.full((rows,), 1.0, device="cuda").multinomial(experts - 1, generator=g).sort().values.diff(
                prepend=torch.zeros(1, dtype=torch.int64, device="cuda"), append=torch.tensor([rows], device="cuda")).tolist())
            index = torch.randint(0, 300, (rows,), generator=g, device="cuda", dtype=torch.int32)
            versions.append(((x, w, offsets, index), ops.grouped_linear(x, w, offsets, row_index=index)))
            want, tol = linear64(x[index[:1].long()], w[int((offsets <= 0).sum()) - 1])
            assert_rounded(versions[-1][1][:1], want, tol)
        torch.cuda.synchronize()
        now = [torch.empty_like(t) for t in versions[0][0]]
        for n in range(24):
            operands, want = versions[n % 2]
            order = list(range(4))
            order = order[n % 4:] + order[:n % 4]  # each of them the last one written
            for i in order:
                now[i].copy_(operands[i])
            got = ops.grouped_linear(now[0], now[1], now[2], row_index=now[3])
            assert torch.equal(got, want), (rows, n)


@pytest.mark.parametrize("rows", [3, 200, 700])
def test_captured_behind_copies_joins_and_at_the_start(rows):
    """Calls as a graph's first node, behind a copy and a fill, beside one another and behind a join of two streams."""
    from llm_compileforge_b200 import ops

    g = gen(51)
    x, w, v = make(g, rows, 256), make(g, 256, 256, std=0.06), make(g, 256, 256, std=0.06)
    index, offsets = torch.randperm(rows, generator=g, device="cuda").int(), offsets_of([rows // 3, rows - rows // 3])
    both = torch.stack([w, v])
    side = torch.cuda.Stream()

    def work():
        here = torch.cuda.current_stream()
        a = ops.fused_linear(x, w)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = ops.fused_linear(a, v, activation="silu")
            b2 = ops.grouped_linear(b, both, offsets, row_index=index)
        c = torch.empty_like(a).copy_(a)
        d = ops.fused_linear(c, v)
        here.wait_stream(side)
        e = ops.fused_linear(d, w, residual=b2)
        f = torch.zeros_like(e)
        ops.fused_linear(e, v, residual=f, out=f)
        route = ops.moe_route(f[:, :16], 2)
        y = ops.moe_combine(f, route.positions.clamp(max=rows - 1), route.weights, residual=e)
        return [a, b, b2, d, e, f, *route, y]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for _ in range(3):
        x.copy_(make(g, rows, 256))
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        for t in held:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), n


# ── the two ways from Python into the library ────────────────────────────────
def test_both_ways_into_the_library_agree(monkeypatch):
    from llm_compileforge_b200 import _lib, ops

    g = gen(40)
    x, w, v, b = make(g, 2, 30, 128), make(g, 128, 96, std=0.1), make(g, 128, 96, std=0.1), make(g, 96)
    r, flat = make(g, 2, 30, 96), make(g, 60, 128)
    we, ve, be = make(g, 4, 128, 72, std=0.1), make(g, 72, 4, 128).permute(1, 2, 0), make(g, 4, 72)
    offsets, index = offsets_of([10, 0, 45, 5]), torch.randint(0, 60, (60,), generator=g, device="cuda", dtype=torch.int32)
    logits = make(g, 300, 12, dtype=F32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def every():
        route = ops.moe_route(logits, 3, renormalize=False)
        y = make(gen(41), 900, 64)
        out, out2 = torch.zeros(60, 96, dtype=F32, device="cuda"), torch.zeros(300, 64, dtype=BF16, device="cuda")
        grouped_out = torch.zeros(60, 72, dtype=BF16, device="cuda")
        return [ops.fused_linear(x, w, b, activation="silu", up_weight=v, up_bias=b, residual=r, status=status), ops.fused_linear(flat, w, out=out),
                ops.fused_linear(x, w, out_dtype=F32), ops.fused_linear(flat, w.t().contiguous().t(), b),
                ops.grouped_linear(flat, we, offsets, be, activation="gelu", row_index=index, status=status), ops.grouped_linear(flat, ve, offsets, up_weight=ve),
                ops.grouped_linear(flat, we, offsets, out=grouped_out), ops.grouped_linear(flat, we, offsets, out_dtype=F32), *route,
                ops.moe_combine(y, route.positions, route.weights, residual=out2, out=out2, status=status), out, grouped_out]

    quick = every()
    assert _lib.calls is not _lib._NoCalls, "the extension module is not built"
    monkeypatch.setattr(_lib, "calls", _lib._NoCalls)
    plain = every()
    assert len(quick) == len(plain)
    for a, c in zip(quick, plain):
        assert a.dtype == c.dtype and a.shape == c.shape and a.is_contiguous() == c.is_contiguous() and torch.equal(a, c)
    assert status.item() == 0


def test_refusals_of_cuda_operands():
    """Bad calls with tensors where they belong: refused before a launch, the results' memory untouched."""
    from llm_compileforge_b200 import ops

    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    x, w, we = z(4, 8), z(8, 16), z(2, 8, 16)
    bad = [
        lambda: ops.fused_linear(x, z(9, 16)), lambda: ops.fused_linear(x, z(8, 16, dtype=F16)), lambda: ops.fused_linear(x, z(8, 16, 1)),
        lambda: ops.fused_linear(x, w, z(15)), lambda: ops.fused_linear(x, w, z(16, dtype=F32)), lambda: ops.fused_linear(x, w, z(32)[::2]),
        lambda: ops.fused_linear(x, w, up_bias=z(16)), lambda: ops.fused_linear(x, w, up_weight=z(8, 8)), lambda: ops.fused_linear(x, w, up_weight=z(16, 8).t()),
        lambda: ops.fused_linear(x, w, residual=z(4, 15)), lambda: ops.fused_linear(x, w, residual=z(2, 2, 16)), lambda: ops.fused_linear(x, w, residual=z(4, 16, dtype=F32)),
        lambda: ops.fused_linear(x, w, out=z(5, 16)), lambda: ops.fused_linear(x, w, out=z(4, 16, dtype=F16)), lambda: ops.fused_linear(x, w, out=z(16, 4).t()),
        lambda: ops.fused_linear(x, w, out=z(1, 16).expand(4, 16)), lambda: ops.fused_linear(x, w, activation="SILU"), lambda: ops.fused_linear(x, w, activation=["silu"]),
        lambda: ops.fused_linear(x, w, status=z(1, dtype=torch.int64)), lambda: ops.fused_linear(x, w.cpu()), lambda: ops.fused_linear(x.cpu(), w),
        lambda: ops.fused_linear(x.double(), w.double()), lambda: ops.fused_linear(x, z(8, 32)[:, ::2]), lambda: ops.fused_linear(x, w, out_dtype=F16),
        lambda: ops.grouped_linear(x, we, i(4)), lambda: ops.grouped_linear(x, we, i(3).long()), lambda: ops.grouped_linear(x, we, i(6)[::2]),
        lambda: ops.grouped_linear(x, we, i(3), row_index=i(4).long()), lambda: ops.grouped_linear(x, we, i(3), row_index=i(8)[::2]),
        lambda: ops.grouped_linear(x, we, i(3), z(2, 15)), lambda: ops.grouped_linear(x, we, i(3), z(16)), lambda: ops.grouped_linear(x, we, i(3), out=z(5, 16)),
        lambda: ops.grouped_linear(x, we, i(3), row_index=i(6), out=z(4, 16)), lambda: ops.grouped_linear(x[:0], we, i(3), row_index=i(4)),
        lambda: ops.grouped_linear(x, z(1025, 8, 8), i(1026)), lambda: ops.grouped_linear(x, we, i(3).cpu()), lambda: ops.grouped_linear(x, we, i(3), workspace=z(9).cpu()),
        lambda: ops.moe_route(z(4, 8), 9), lambda: ops.moe_route(z(4, 8), 0), lambda: ops.moe_route(z(4, 64), 33), lambda: ops.moe_route(z(4, 8), -1),
        lambda: ops.moe_route(z(4, 2000), 2), lambda: ops.moe_route(z(4, 8, dtype=torch.float64), 2), lambda: ops.moe_route(z(8), 1), lambda: ops.moe_route(i(4, 8), 1),
        lambda: ops.moe_combine(x, i(3, 2), z(3, 2)), lambda: ops.moe_combine(x, i(3, 2).long(), z(3, 2, dtype=F32)), lambda: ops.moe_combine(x, i(3, 33), z(3, 33, dtype=F32)),
        lambda: ops.moe_combine(x, i(3, 2), z(2, 2, dtype=F32)), lambda: ops.moe_combine(x, i(3, 2), z(3, 2, dtype=F32), residual=z(3, 9)),
        lambda: ops.moe_combine(x, i(3, 2), z(3, 2, dtype=F32), residual=z(3, 8, dtype=F16)), lambda: ops.moe_combine(x, i(3, 2), z(3, 2, dtype=F32), out=z(1, 8).expand(3, 8)),
        lambda: ops.moe_combine(x, i(3, 2), z(2, 3, dtype=F32).t()),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was not refused")
    torch.cuda.synchronize()
