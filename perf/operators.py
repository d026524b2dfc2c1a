"""What the framework's feed-forward operators are measured on: the dense and the routed half of a decoder layer.

Four operators, the calls that follow attention in a serving step:

* ``linear``  ``fused_linear``: ``act(x W + b) [* (x V + c)] [+ residual]``, one product with its whole epilogue;
* ``route``   ``moe_route``: the ``top_k`` experts of every token, their softmax weights, and the token rows sorted by expert;
* ``grouped`` ``grouped_linear``: the same product for rows grouped by expert, every group with its own matrix and a ragged size;
* ``combine`` ``moe_combine``: every token's weighted sum of its experts' rows, plus a residual.

``run`` computes a case in elementary torch operations, or, where ``own`` is true, with the framework's operators.
"""

import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_LARGEST = 1.2e12  # floating-point operations that a drawn product may cost: about the largest listed one's


# ── the cases ────────────────────────────────────────────────────────────────
def listed():
    return [
        # one sequence decoding: the attention output's projection back onto the residual stream, 33 MB of weights for one row
        dict(name="linear_token", op="linear", rows=1, k=4096, n=4096, act="none", gated=False, bias=False, residual=True, layout="kn", dtype="bf16"),
        # a decode batch of 64 through a gated feed-forward's first half: two matrices, one launch
        dict(name="linear_batch_gated", op="linear", rows=64, k=4096, n=14336, act="silu", gated=True, bias=False, residual=False, layout="nk", dtype="bf16"),
        # a ragged prompt through a biased GELU layer of a classic block, weights stored output-major as checkpoints have them
        dict(name="linear_prompt_gelu", op="linear", rows=1001, k=2048, n=8192, act="gelu", gated=False, bias=True, residual=False, layout="nk", dtype="f16"),
        # a full prefill batch: the largest product
        dict(name="linear_prefill", op="linear", rows=8192, k=8192, n=8192, act="none", gated=False, bias=False, residual=True, layout="kn", dtype="bf16"),
        # routing of a small decode batch, where only latency counts
        dict(name="route_decode", op="route", rows=16, experts=64, top_k=8, dtype="f32", masked=0),
        # routing of a long prefill batch with padded rows
        dict(name="route_prefill", op="route", rows=16384, experts=128, top_k=8, dtype="bf16", masked=37),
        # a decode batch of 32 tokens, 4 experts each, over 32 gated experts: a handful of rows for every matrix
        dict(name="grouped_decode_gated", op="grouped", tokens=32, top_k=4, experts=32, k=2048, n=1408, act="silu", gated=True, bias=False, skew=0.0, gather=True, layout="kn", dtype="bf16"),
        # a medium batch with very uneven experts, some of them without a row, biased, weights output-major
        dict(name="grouped_skewed", op="grouped", tokens=517, top_k=2, experts=16, k=1024, n=2816, act="gelu_tanh", gated=False, bias=True, skew=1.5, gather=True, layout="nk", dtype="f16"),
        # prefill through the experts' first half ...
        dict(name="grouped_prefill_gated", op="grouped", tokens=4096, top_k=4, experts=32, k=4096, n=1792, act="silu", gated=True, bias=False, skew=0.5, gather=True, layout="nk", dtype="bf16"),
        # ... and back: rows that already lie in expert order
        dict(name="grouped_prefill_down", op="grouped", tokens=4096, top_k=4, experts=32, k=1792, n=4096, act="none", gated=False, bias=False, skew=0.5, gather=False, layout="kn", dtype="bf16"),
        # the experts' rows of a decode batch back to their tokens
        dict(name="combine_decode", op="combine", tokens=32, top_k=4, h=2048, residual=True, dtype="bf16"),
        # and of a prefill batch
        dict(name="combine_prefill", op="combine", tokens=8192, top_k=8, h=4096, residual=True, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _eights(rng, low, high):
    return max(8, _log(rng, low, high) // 8 * 8)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "route", "grouped", "grouped", "grouped", "combine"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    while op == "linear":
        c = dict(op=op, rows=_log(rng, 1, 8192), k=_eights(rng, 256, 8192), n=_eights(rng, 256, 16384),
                 act=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]), gated=rng.random() < 0.4, bias=rng.random() < 0.4,
                 residual=rng.random() < 0.5, layout=rng.choice(["kn", "nk"]), dtype=dtype)
        if work(c)["flops"] <= _LARGEST:
            return c
    while op == "grouped":
        c = dict(op=op, tokens=_log(rng, 1, 4096), top_k=rng.randint(1, 8), experts=rng.choice([8, 16, 24, 32, 64]), k=_eights(rng, 256, 4096),
                 n=_eights(rng, 256, 4096), act=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]), gated=rng.random() < 0.5,
                 bias=rng.random() < 0.3, skew=rng.choice([0.0, 0.5, 1.5]), gather=rng.random() < 0.6, layout=rng.choice(["kn", "nk"]), dtype=dtype)
        # the plain form multiplies every group padded to the largest one
        padded = c["experts"] * max(_counts(c)) * c["k"] * c["n"] * (4 if c["gated"] else 2)
        if c["top_k"] <= c["experts"] and work(c)["flops"] <= _LARGEST and padded <= _LARGEST:
            return c
    if op == "route":
        experts = _log(rng, 4, 256)
        return dict(op=op, rows=_log(rng, 1, 16384), experts=experts, top_k=rng.randint(1, min(8, experts)), dtype=rng.choice(["f32", "bf16", "f16"]), masked=rng.choice([0, 0, 1, 5]))
    return dict(op=op, tokens=_log(rng, 1, 8192), top_k=rng.randint(1, 8), h=_eights(rng, 256, 4096), residual=rng.random() < 0.5, dtype=dtype)


def _counts(c):
    """Rows of every expert: the case alone decides them; ``skew`` 0 draws the experts evenly, above it by a power law."""
    rng = random.Random("%(tokens)s %(top_k)s %(experts)s %(skew)s" % c)
    weights = [(i + 1.0) ** -c["skew"] for i in range(c["experts"])]
    rng.shuffle(weights)
    counts = [0] * c["experts"]
    for e in rng.choices(range(c["experts"]), weights, k=c["tokens"] * c["top_k"]):
        counts[e] += 1
    if c["skew"]:  # an uneven router leaves experts without a row
        counts[(counts.index(max(counts)) + 1) % len(counts)] += counts[0]
        counts[0] = 0
    return counts


def work(c):
    e = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "linear":
        mats = 2 if c["gated"] else 1
        rows, k, n = c["rows"], c["k"], c["n"]
        return {"bytes": e * (rows * k + mats * (k * n + (n if c["bias"] else 0)) + rows * n * (2 if c["residual"] else 1)), "flops": 2.0 * mats * rows * k * n}
    if c["op"] == "grouped":
        mats = 2 if c["gated"] else 1
        rows, k, n = c["tokens"] * c["top_k"], c["k"], c["n"]
        used = sum(1 for m in _counts(c) if m)
        x_rows = min(rows, c["tokens"]) if c["gather"] else rows
        return {"bytes": e * (x_rows * k + mats * used * (k * n + (n if c["bias"] else 0)) + rows * n) + 4 * (c["experts"] + 1 + (rows if c["gather"] else 0)),
                "flops": 2.0 * mats * rows * k * n}
    if c["op"] == "route":
        rows, top = c["rows"], c["top_k"]
        return {"bytes": e * rows * c["experts"] + 16 * rows * top + 4 * (c["experts"] + 1), "flops": 3.0 * rows * c["experts"]}
    rows, top, h = c["tokens"], c["top_k"], c["h"]
    return {"bytes": e * h * rows * (top + (2 if c["residual"] else 1)) + 8 * rows * top, "flops": 2.0 * rows * top * h}


# ── inputs ───────────────────────────────────────────────────────────────────
def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    dt = _TYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dt)

    def matrix(*lead, k, n):  # [.., k, n]; "nk": stored output-major, as checkpoints store a projection
        if c["layout"] == "nk":
            return normal(*lead, n, k, std=k ** -0.5).transpose(-1, -2)
        return normal(*lead, k, n, std=k ** -0.5)

    s = {"case": c}
    if c["op"] == "linear":
        rows, k, n = c["rows"], c["k"], c["n"]
        s["x"], s["w"] = normal(rows, k), matrix(k=k, n=n)
        s["v"] = matrix(k=k, n=n) if c["gated"] else None
        s["b"] = normal(n, std=0.5) if c["bias"] else None
        s["vb"] = normal(n, std=0.5) if c["bias"] and c["gated"] else None
        s["r"] = normal(rows, n) if c["residual"] else None
    elif c["op"] == "grouped":
        rows, k, n, experts, counts = c["tokens"] * c["top_k"], c["k"], c["n"], c["experts"], _counts(c)
        s["w"] = matrix(experts, k=k, n=n)
        s["v"] = matrix(experts, k=k, n=n) if c["gated"] else None
        s["b"] = normal(experts, n, std=0.5) if c["bias"] else None
        s["vb"] = normal(experts, n, std=0.5) if c["bias"] and c["gated"] else None
        s["x"] = normal(c["tokens"] if c["gather"] else rows, k)
        s["index"] = torch.randint(0, c["tokens"], (rows,), generator=g, device=dev, dtype=torch.int32) if c["gather"] else None
        at = [0]
        for m in counts:
            at.append(at[-1] + m)
        s["offsets"] = torch.tensor(at, dtype=torch.int32, device=dev)
        s["largest"] = max(counts)  # the plain form's padded group size; the operator does not take it
    elif c["op"] == "route":
        # a router's logits: an even spread with a few experts that many tokens prefer
        s["logits"] = (torch.randn((c["rows"], c["experts"]), generator=g, device=dev) * 1.5 + torch.randn((c["experts"],), generator=g, device=dev)).to(dt)
        if c["masked"]:  # rows that pad the batch, and one expert that is switched off
            s["logits"][max(0, c["rows"] - c["masked"]):] = float("-inf")
            s["logits"][:, c["experts"] // 2] = float("-inf")
    else:
        rows, top = c["tokens"], c["top_k"]
        s["y"] = normal(rows * top, c["h"])
        s["positions"] = torch.randperm(rows * top, generator=g, device=dev).to(torch.int32).view(rows, top)
        p = torch.rand((rows, top), generator=g, device=dev) + 0.05
        s["weights"] = p / p.sum(1, keepdim=True)
        s["r"] = normal(rows, c["h"]) if c["residual"] else None
    return s


# ── the operators ────────────────────────────────────────────────────────────
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from llm_compileforge_b200 import ops

    c = s["case"]
    if c["op"] == "linear":
        return ops.fused_linear(s["x"], s["w"], s["b"], activation=c["act"], up_weight=s["v"], up_bias=s["vb"], residual=s["r"])
    if c["op"] == "grouped":
        return ops.grouped_linear(s["x"], s["w"], s["offsets"], s["b"], activation=c["act"], up_weight=s["v"], up_bias=s["vb"], row_index=s["index"])
    if c["op"] == "route":
        return tuple(ops.moe_route(s["logits"], c["top_k"]))
    return ops.moe_combine(s["y"], s["positions"], s["weights"], residual=s["r"])


def _act(h, name):
    if name == "silu":
        return h / (1 + torch.exp(-h))
    if name == "gelu":
        return 0.5 * h * (1 + torch.erf(h * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (h + 0.044715 * h ** 3)))
    return torch.clamp(h, min=0) if name == "relu" else h


def _plain(s):
    c = s["case"]
    if c["op"] == "linear":
        x = s["x"].float()
        h = x @ s["w"].float()
        h = _act(h if s["b"] is None else h + s["b"].float(), c["act"])
        if c["gated"]:
            u = x @ s["v"].float()
            h = h * (u if s["vb"] is None else u + s["vb"].float())
        return (h if s["r"] is None else h + s["r"].float()).to(s["x"].dtype)
    if c["op"] == "grouped":
        # rows into a [experts, largest group, k] box, one batched product, and back
        at = s["offsets"].long()
        row = torch.arange(c["tokens"] * c["top_k"], device=at.device)
        group = torch.searchsorted(at[1:], row, right=True)
        place = row - at[group]
        x = s["x"].float()
        box = torch.zeros((c["experts"], s["largest"], c["k"]), device=x.device)
        box[group, place] = x if s["index"] is None else x[s["index"].long()]
        h = torch.bmm(box, s["w"].float())
        h = _act(h if s["b"] is None else h + s["b"].float()[:, None], c["act"])
        if c["gated"]:
            u = torch.bmm(box, s["v"].float())
            h = h * (u if s["vb"] is None else u + s["vb"].float()[:, None])
        return h[group, place].to(s["x"].dtype)
    if c["op"] == "route":
        l, top = s["logits"].float(), c["top_k"]
        value, ids = torch.sort(l, dim=1, descending=True, stable=True)  # equal logits: the lower index first
        value, ids = value[:, :top], ids[:, :top]
        alive = value > float("-inf")
        p = torch.where(alive, torch.exp(value - torch.where(alive[:, :1], value[:, :1], 0.0)), 0.0)
        p = p / torch.clamp(p.sum(1, keepdim=True), min=1.0)  # the largest logit counts 1: the sum is 0 or at least 1
        key = torch.where(alive, ids, c["experts"]).reshape(-1)
        order = torch.sort(key, stable=True)[1]
        place = torch.empty_like(order)
        place[order] = torch.arange(order.numel(), device=order.device)
        token = torch.where(key[order] < c["experts"], order // top, -1)
        offsets = (key[:, None] < torch.arange(c["experts"] + 1, device=key.device)).sum(0)
        whole = lambda t: t.to(torch.int32)  # noqa: E731
        return (whole(torch.where(alive, ids, -1)), p, whole(offsets), whole(token), whole(torch.where(alive, place.view(-1, top), -1)))
    picked = s["y"][s["positions"].long()].float()
    out = (picked * s["weights"][:, :, None]).sum(1)
    return (out if s["r"] is None else out + s["r"].float()).to(s["y"].dtype)


# ── in 64 bits, from the definitions ─────────────────────────────────────────
def _act64(h, name):
    if name == "silu":
        return h * torch.special.expit(h)
    if name == "gelu":
        return h * torch.special.ndtr(h)
    if name == "gelu_tanh":  # (1 + tanh z) / 2 is the logistic function of 2 z
        return h * torch.special.expit(2 * (2 / torch.pi) ** 0.5 * (h + 0.044715 * h * h * h))
    return torch.where(h > 0, h, torch.zeros_like(h)) if name == "relu" else h


def exact(c, seed):
    s = prepare(c, seed)
    d = lambda t: t.double()  # noqa: E731
    if c["op"] in ("linear", "grouped"):
        def product(x, i):
            pick = (lambda t: t) if i is None else (lambda t: t[i])
            h = torch.einsum("mk,kn->mn", x, d(pick(s["w"])))
            if c["bias"]:
                h += d(pick(s["b"]))
            h = _act64(h, c["act"])
            if c["gated"]:
                u = torch.einsum("mk,kn->mn", x, d(pick(s["v"])))
                if c["bias"]:
                    u += d(pick(s["vb"]))
                h *= u
            return h

        if c["op"] == "linear":
            y = product(d(s["x"]), None)
            return y + d(s["r"]) if c["residual"] else y
        x = s["x"] if s["index"] is None else torch.index_select(s["x"], 0, s["index"])
        at = s["offsets"].tolist()
        return torch.cat([product(d(x[at[i]:at[i + 1]]), i) for i in range(c["experts"])])
    if c["op"] == "route":
        rows = d(s["logits"]).cpu().tolist()
        n, experts, top = len(rows), c["experts"], c["top_k"]
        ids = [[-1] * top for _ in rows]
        value = torch.full((n, top), float("-inf"), dtype=torch.float64)
        groups = [[] for _ in range(experts)]
        for t, row in enumerate(rows):
            best = sorted(((-v, i) for i, v in enumerate(row) if v > float("-inf")))[:top]
            for j, (v, i) in enumerate(best):
                ids[t][j] = i
                value[t, j] = -v
                groups[i].append((t, j))
        weights = torch.nan_to_num(torch.softmax(value, 1), nan=0.0)
        token, place, offsets = [-1] * (n * top), [[-1] * top for _ in rows], [0]
        for members in groups:
            offsets.append(offsets[-1] + len(members))
        at = 0
        for members in groups:
            for t, j in members:
                token[at], place[t][j] = t, at
                at += 1
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        return (i32(ids), weights, i32(offsets), i32(token), i32(place))
    out = torch.zeros((c["tokens"], c["h"]), dtype=torch.float64, device=s["y"].device)
    for j in range(c["top_k"]):
        out += d(s["weights"][:, j:j + 1]) * d(torch.index_select(s["y"], 0, s["positions"][:, j]))
    return out + d(s["r"]) if c["residual"] else out
