"""Timed cases of the operators of a pre-norm block: the norm in front of it, the bias of its attention's scores, its
feed-forward half.

  norm   root-mean-square norm of the rows of x + residual, the sum handed on as the residual stream; with its gradients, or
         with the normalised rows in 8 bits (e4m3) and one scale a row
  bias   learned relative position bias of a sparse attention's edges: the positions of an edge's two ends, their distance's
         bucket, the bucket's row of a table; with the table's gradient
  ffn    gated feed-forward block: act(x Wg^T) * (x Wu^T), times Wd^T, plus the residual; with its gradients

``run`` computes them from elementary operations in 32 bits, or, where ``own`` is set, by the package's entry points.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
CLUSTERS = 8
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
E4M3_MOST, SMALLEST_SCALE = 448.0, 2.0 ** -126
MOST_ROW_VALUES = 16384 * 5120       # of a norm, of the largest listed case
MOST_EDGES = 18214272
MOST_PRODUCTS = 9 * 16384 * 1024 * 2816      # of a feed-forward block


# ---- cases -----------------------------------------------------------------------------------------------------------
def _norm(name, rows, hidden, dtype, mode, residual=True):
    case = {"kind": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "mode": mode, "residual": residual}
    return dict(case, name=name) if name else case


def _bias(name, nodes, random_edges, heads, buckets=32, distance=128, both_ways=True, backward=True, int32=False):
    case = {"kind": "bias", "nodes": nodes, "random_edges": random_edges, "heads": heads, "buckets": buckets,
            "distance": distance, "both_ways": both_ways, "backward": backward, "int32": int32}
    return dict(case, name=name) if name else case


def _ffn(name, rows, hidden, middle, dtype, activation="silu", residual=True, backward=True):
    case = {"kind": "ffn", "rows": rows, "hidden": hidden, "middle": middle, "dtype": dtype, "activation": activation,
            "residual": residual, "backward": backward}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one serving step of four sequences: the norm in front of a product in 8 bits, all latency
        _norm("norm-4-rows-e4m3", 4, 4096, "bf16", "quantise"),
        # the norm between the two halves of an encoder layer, sequence length 64,000 at the models' width of 64
        _norm("norm-64k-train", 64001, 64, "fp32", "train"),
        # a wide model's training step
        _norm("norm-2048-train", 16384, 2048, "bf16", "train"),
        # a long prompt on its way into products in 8 bits
        _norm("norm-5120-e4m3", 16384, 5120, "bf16", "quantise"),
        # serving a small graph: the bias of one attention call, all latency
        _bias("bias-4k", 4096, 8 * 4096, 8, backward=False),
        # a training step on the batch of 64,000 nodes and 526,450 edges
        _bias("bias-64k-train", 64000, 334450, 8),
        # the long-sequence batch of 870,000 nodes and 18.2 M edges
        _bias("bias-870k-train", 870000, 18214272 - 3 * 870000, 8),
        # one token's feed-forward block: the weights are read once and nothing else counts
        _ffn("ffn-1-row", 1, 2048, 5632, "bf16", residual=True, backward=False),
        # a short prompt with an odd number of tokens
        _ffn("ffn-333-rows", 333, 768, 2048, "bf16", activation="gelu", backward=False),
        # an encoder layer's feed-forward half, sequence length 64,000 at the models' width of 64 in fp32
        _ffn("ffn-64k-train", 64001, 64, 128, "fp32"),
        # a prompt of 8,191 tokens
        _ffn("ffn-8191-rows", 8191, 2048, 5632, "bf16", backward=False),
        # a wide model's training step
        _ffn("ffn-1024-train", 16384, 1024, 2816, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "bias", "ffn"])
    if kind == "norm":
        mode = rng.choice(["forward", "train", "train", "quantise"])
        hidden = _log_int(rng, 32, 8192)
        if rng.random() < 0.8:
            hidden = max(8, hidden // 8 * 8)
        rows = _log_int(rng, 1, MOST_ROW_VALUES // (hidden * (2 if mode == "train" else 1)))
        return _norm(None, min(rows, 400000), hidden, rng.choice(["fp32", "bf16", "bf16"]), mode, rng.random() < 0.7)
    if kind == "bias":
        nodes = _log_int(rng, 500, 870000)
        heads = rng.choice([1, 2, 4, 8, 8, 8, 12, 16, 32])
        edges = min(int(nodes * math.exp(rng.uniform(0.0, math.log(17.0)))), MOST_EDGES * 8 // max(heads, 8) - 3 * nodes)
        buckets, distance = rng.choice([(32, 128), (32, 128), (64, 1000), (16, 64), (128, 4096), (10, 50)])
        return _bias(None, nodes, max(edges, 0), heads, buckets, distance, rng.random() < 0.7, rng.random() < 0.7,
                     rng.random() < 0.4)
    backward = rng.random() < 0.6
    activation = rng.choice(["silu", "silu", "gelu", "relu"])
    if rng.random() < 0.3:
        hidden, middle, dtype = 64 * rng.randint(1, 8), 64 * rng.randint(1, 8), "fp32"
    else:
        hidden, middle, dtype = 8 * rng.randint(8, 320), 8 * rng.randint(8, 700), "bf16"
    most = MOST_PRODUCTS // (hidden * middle * (9 if backward else 3))
    if dtype == "fp32":
        most = most // 4
    return _ffn(None, _log_int(rng, 1, min(most, 100000)), hidden, middle, dtype, activation, rng.random() < 0.6, backward)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _prepare_norm(case, gen):
    dtype, shape = TYPES[case["dtype"]], (case["rows"], case["hidden"])
    s = SimpleNamespace(x=_randn(shape, dtype, gen), weight=(1 + _randn(shape[1:], torch.float32, gen, 0.2)).to(dtype),
                        residual=_randn(shape, dtype, gen, 2.0) if case["residual"] else None)
    if case["mode"] == "train":
        s.dy, s.dsum = _randn(shape, dtype, gen), _randn(shape, dtype, gen) if case["residual"] else None
        for t in (s.x, s.weight, s.residual):
            if t is not None:
                t.requires_grad_()
    return s


def _edges(case, gen):
    """[2, 3 nodes + random_edges]: self loops, a global token at row 0 linked both ways with every node, random edges that
    mostly stay inside one of eight clusters; in no particular order."""
    n, m = case["nodes"], case["random_edges"]
    size = max(1, n // CLUSTERS)
    nodes = torch.arange(1, n + 1, device="cuda")
    zeros = torch.zeros_like(nodes)
    src = torch.randint(0, n, (m,), generator=gen, device="cuda")
    cross = torch.rand(m, generator=gen, device="cuda") < 0.315
    near = ((src // size) * size + torch.randint(0, size, (m,), generator=gen, device="cuda")).clamp_(max=n - 1)
    dst = torch.where(cross, torch.randint(0, n, (m,), generator=gen, device="cuda"), near)
    return torch.cat([torch.stack([nodes, nodes]), torch.stack([nodes, zeros]), torch.stack([zeros, nodes]),
                      torch.stack([src + 1, dst + 1])], dim=1)


def _prepare_bias(case, gen):
    edges = _edges(case, gen)
    # a node's place along its cluster, as a reordered batch has it: most ends of an edge are near one another
    rows = case["nodes"] + 1
    positions = torch.randint(0, max(2, 4 * case["distance"]), (rows,), generator=gen, device="cuda")
    if case["int32"]:
        edges, positions = edges.int(), positions.int()
    s = SimpleNamespace(edges=edges, positions=positions, table=_randn((case["buckets"], case["heads"]), torch.float32, gen, 0.1),
                        borders=torch.tensor(_borders(case), device="cuda"))
    if case["backward"]:
        s.dbias = _randn((edges.shape[1], case["heads"]), torch.float32, gen)
        s.table.requires_grad_()
    return s


def _prepare_ffn(case, gen):
    dtype, rows, hidden, middle = TYPES[case["dtype"]], case["rows"], case["hidden"], case["middle"]
    s = SimpleNamespace(x=_randn((rows, hidden), dtype, gen), gate=_randn((middle, hidden), dtype, gen, hidden ** -0.5),
                        up=_randn((middle, hidden), dtype, gen, hidden ** -0.5),
                        down=_randn((hidden, middle), dtype, gen, middle ** -0.5),
                        residual=_randn((rows, hidden), dtype, gen) if case["residual"] else None)
    if case["backward"]:
        s.dy = _randn((rows, hidden), dtype, gen)
        for t in (s.x, s.gate, s.up, s.down, s.residual):
            if t is not None:
                t.requires_grad_()
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "bias": _prepare_bias, "ffn": _prepare_ffn}[case["kind"]](case, _generator(seed))
    s.case = case
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plain_norm(s):
    case, dtype = s.case, s.x.dtype
    v, w = s.x.detach().float(), s.weight.detach().float()
    if s.residual is not None:
        v = v + s.residual.detach().float()
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    y = v * rstd * w
    total = [v.to(dtype)] if s.residual is not None else []
    if case["mode"] == "quantise":
        scale = (y.abs().amax(-1) / E4M3_MOST).clamp(min=SMALLEST_SCALE)
        return [(y * (1 / scale)[:, None]).to(torch.float8_e4m3fn), scale, *total]
    if case["mode"] == "forward":
        return [y.to(dtype), *total]
    dy, unit = s.dy.float(), v * rstd
    g = dy * w
    dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    dw = (dy * unit).sum(0).to(dtype)
    if s.residual is None:
        return [y.to(dtype), dx.to(dtype), dw]
    dx = (dx + s.dsum.float()).to(dtype)
    return [y.to(dtype), *total, dx, dx, dw]


def _borders(case):
    """The smallest distance of every bucket but the first, of one direction.  Half of a direction's buckets are a distance
    each; the others' borders are even steps of the logarithm, the last bucket starting below ``distance``:
    n >= exact * (distance / exact) ** (j / steps), in whole numbers n ** steps >= distance ** j * exact ** (steps - j)."""
    count = case["buckets"] // 2 if case["both_ways"] else case["buckets"]
    exact = count // 2
    steps = count - exact
    borders = list(range(1, exact + 1))
    for j in range(1, steps):
        bound, lo, hi = case["distance"] ** j * exact ** (steps - j), exact, case["distance"]
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** steps >= bound else (mid + 1, hi)
        borders.append(lo)
    return borders


def _plain_bias(s):
    source, destination = s.edges.long()
    offset = s.positions.long()[source] - s.positions.long()[destination]
    if s.case["both_ways"]:
        distance, first = offset.abs(), (offset > 0).long() * (s.case["buckets"] // 2)
    else:
        distance, first = (-offset).clamp(min=0), 0
    bucket = first + torch.bucketize(distance, s.borders, right=True)
    table = s.table.detach()
    bias = table[bucket]
    if not s.case["backward"]:
        return [bias]
    grad = torch.zeros(table.shape, dtype=torch.float64, device="cuda").index_add_(0, bucket, s.dbias.double())   # long sums
    return [bias, grad.to(table.dtype)]


def _activation(name, x):
    """act(x) and its derivative."""
    if name == "relu":
        return x.clamp(min=0), (x > 0).to(x.dtype)
    if name == "silu":
        sigmoid = 1 / (1 + torch.exp(-x))
        return x * sigmoid, sigmoid * (1 + x * (1 - sigmoid))
    cdf = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def _plain_ffn(s):
    dtype = s.x.dtype
    x, wg, wu, wd = (t.detach().float() for t in (s.x, s.gate, s.up, s.down))
    g, u = x @ wg.T, x @ wu.T
    a, slope = _activation(s.case["activation"], g)
    h = a * u
    y = h @ wd.T
    if s.residual is not None:
        y = y + s.residual.detach().float()
    if not s.case["backward"]:
        return [y.to(dtype)]
    dy = s.dy.float()
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    grads = [dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h]
    return [y.to(dtype), *(t.to(dtype) for t in grads), *([s.dy] if s.residual is not None else [])]


# ---- one pass --------------------------------------------------------------------------------------------------------
def _own_norm(s):
    from torchgt_b200.rms_norm import add_rms_norm, rms_norm, rms_norm_quantized
    mode = s.case["mode"]
    if mode == "quantise":
        with torch.no_grad():
            values, scale, total = rms_norm_quantized(s.x, s.weight, EPS, residual=s.residual)
        return [values, scale] + ([total] if s.residual is not None else [])
    if s.residual is None:
        if mode == "forward":
            with torch.no_grad():
                return [rms_norm(s.x, s.weight, EPS)]
        y = rms_norm(s.x, s.weight, EPS)
        return [y.detach(), *torch.autograd.grad(y, [s.x, s.weight], s.dy)]
    if mode == "forward":
        with torch.no_grad():
            return list(add_rms_norm(s.x, s.residual, s.weight, EPS))
    y, total = add_rms_norm(s.x, s.residual, s.weight, EPS)
    grads = torch.autograd.grad([y, total], [s.x, s.residual, s.weight], [s.dy, s.dsum])
    return [y.detach(), total.detach(), *grads]


def _own_bias(s):
    from torchgt_b200.position_bias import edge_position_bias
    call = (s.table, s.edges, s.positions, s.case["distance"], s.case["both_ways"])
    if not s.case["backward"]:
        with torch.no_grad():
            return [edge_position_bias(*call)]
    bias = edge_position_bias(*call)
    return [bias.detach(), *torch.autograd.grad(bias, [s.table], s.dbias)]


def _own_ffn(s):
    from torchgt_b200.gated_ffn import gated_feed_forward
    call = (s.x, s.gate, s.up, s.down, s.case["activation"], s.residual)
    if not s.case["backward"]:
        with torch.no_grad():
            return [gated_feed_forward(*call)]
    y = gated_feed_forward(*call)
    inputs = [s.x, s.gate, s.up, s.down] + ([s.residual] if s.residual is not None else [])
    return [y.detach(), *torch.autograd.grad(y, inputs, s.dy)]


def run(state):
    kind = state.case["kind"]
    if own:
        return {"norm": _own_norm, "bias": _own_bias, "ffn": _own_ffn}[kind](state)
    return {"norm": _plain_norm, "bias": _plain_bias, "ffn": _plain_ffn}[kind](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def _exact_norm(s):
    x, r, w = _leaf(s.x), _leaf(s.residual), _leaf(s.weight)
    total = x if r is None else x + r
    y = w * total / torch.sqrt(torch.sum(total ** 2, -1, keepdim=True) / total.shape[-1] + EPS)
    sums = [] if r is None else [total.detach()]
    if s.case["mode"] == "quantise":
        scale = torch.clamp(torch.max(torch.abs(y), -1, keepdim=True).values / E4M3_MOST, min=SMALLEST_SCALE)
        return [(y / scale).detach(), scale.detach().squeeze(-1), *sums]
    if s.case["mode"] == "forward":
        return [y.detach(), *sums]
    loss = torch.sum(y * s.dy.double())
    if r is not None:
        loss = loss + torch.sum(total * s.dsum.double())
    return [y.detach(), *sums, *torch.autograd.grad(loss, [x, w] if r is None else [x, r, w])]


def _exact_bias(s):
    case = s.case
    where = s.positions.long()
    offset = where.index_select(0, s.edges[0].long()) - where.index_select(0, s.edges[1].long())
    # every distance's bucket, counted border by border
    distance = torch.abs(offset) if case["both_ways"] else torch.where(offset < 0, -offset, torch.zeros_like(offset))
    bucket = torch.zeros_like(distance)
    for border in _borders(case):
        bucket += distance >= border
    if case["both_ways"]:
        bucket = torch.where(offset > 0, bucket + case["buckets"] // 2, bucket)
    table = s.table.detach().double()
    bias = table.index_select(0, bucket)
    if not case["backward"]:
        return [bias]
    d = s.dbias.double()
    return [bias, torch.stack([(d * (bucket == b)[:, None]).sum(0) for b in range(case["buckets"])])]


def _exact_ffn(s):
    x, wg, wu, wd, r = (_leaf(t) for t in (s.x, s.gate, s.up, s.down, s.residual))
    act = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[s.case["activation"]]
    y = torch.matmul(act(torch.matmul(x, wg.t())) * torch.matmul(x, wu.t()), wd.t())
    if r is not None:
        y = r + y
    if not s.case["backward"]:
        return [y.detach()]
    inputs = [x, wg, wu, wd] + ([r] if r is not None else [])
    return [y.detach(), *torch.autograd.grad(y, inputs, s.dy.double())]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "bias": _exact_bias, "ffn": _exact_ffn}[case["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        size = 4 if case["dtype"] == "fp32" else 2
        values, row = case["rows"] * case["hidden"], case["hidden"] * size
        ends = 2 if case["residual"] else 1                   # x and residual in, sum out
        if case["mode"] == "quantise":
            return {"bytes": values * size * (2 * ends - 1) + values + row + 4 * case["rows"], "flops": 8 * values}
        if case["mode"] == "forward":
            return {"bytes": values * size * 2 * ends + row, "flops": 6 * values}
        return {"bytes": values * size * (3 * ends + 2) + 2 * row, "flops": 16 * values}    # and dy, dsum in, dx out
    if case["kind"] == "bias":
        edges = 3 * case["nodes"] + case["random_edges"]
        table = 4 * case["buckets"] * case["heads"]
        ids = (4 if case["int32"] else 8) * (2 * edges + case["nodes"] + 1)
        values = 4 * edges * case["heads"]
        if not case["backward"]:
            return {"bytes": ids + values + table, "flops": 0}
        return {"bytes": ids + 2 * values + 2 * table, "flops": edges * case["heads"]}
    size = 4 if case["dtype"] == "fp32" else 2
    rows, weights = case["rows"] * case["hidden"] * size, 3 * case["hidden"] * case["middle"] * size
    products = 6 * case["rows"] * case["hidden"] * case["middle"]
    tensors = 3 if case["residual"] else 2
    if not case["backward"]:
        return {"bytes": tensors * rows + weights, "flops": products}
    return {"bytes": (tensors + 2) * rows + 2 * weights, "flops": 3 * products}     # and dy in, dx out
