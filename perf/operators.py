"""Measured cases of the row operators: embedding lookup and its gradient, rows sorted by id, and products grouped by
expert with their gradients.

Each is a product with a sparse factor that is given by one id per row: a lookup multiplies by a matrix with a single
nonzero in every row, its gradient by the transposed matrix, a grouped product by a matrix of dense blocks.  Where `own`
is false `run` computes them from elementary torch operations in 32 bits, otherwise through the package's entry points.
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
ID_TYPES = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # one step of a small batch of sequences that are being answered: latency
        {"name": "lookup step", "op": "lookup", "n": 16, "ids": 32768, "width": 1024, "type": "bf16", "id": "i64"},
        # the first layer of a training step: 8 sequences of 4096 tokens over a large vocabulary
        {"name": "lookup batch", "op": "lookup", "n": 32768, "ids": 131072, "width": 4096, "type": "bf16", "id": "i64"},
        # a short batch, odd vocabulary and width, gradients kept in 32 bits
        {"name": "lookup_grad short", "op": "lookup_grad", "n": 1000, "ids": 50001, "width": 771, "type": "f16", "out": "f32", "id": "i32"},
        # the last layer of a backward pass: every row of a large table is written, most of them zero
        {"name": "lookup_grad batch", "op": "lookup_grad", "n": 32768, "ids": 131072, "width": 2048, "type": "bf16", "out": "bf16", "id": "i64"},
        # many tokens over a small vocabulary: the sums are long
        {"name": "lookup_grad long", "op": "lookup_grad", "n": 262144, "ids": 32768, "width": 1024, "type": "bf16", "out": "f32", "id": "i64"},
        # the rows of a small batch sorted by the expert that they go to
        {"name": "group_rows short", "op": "group_rows", "n": 512, "ids": 16, "id": "i32"},
        # eight experts of 64 for each of 65536 tokens
        {"name": "group_rows batch", "op": "group_rows", "n": 524288, "ids": 64, "id": "i64"},
        # answering: a handful of rows, and the weights of the experts that they meet are read once
        {"name": "experts step", "op": "experts", "n": 32, "groups": 64, "k": 2048, "m": 1024, "type": "bf16"},
        # the experts' products of a training step
        {"name": "experts batch", "op": "experts", "n": 32768, "groups": 32, "k": 2048, "m": 4096, "type": "bf16"},
        # odd sizes in 32 bits
        {"name": "experts odd f32", "op": "experts", "n": 1777, "groups": 10, "k": 1001, "m": 519, "type": "f32"},
        # short ragged groups, backward
        {"name": "experts_grad short", "op": "experts_grad", "n": 777, "groups": 8, "k": 512, "m": 1024, "type": "f16", "out": "f16"},
        # the backward pass of the experts' products of a training step, gradients of the weights in 32 bits
        {"name": "experts_grad batch", "op": "experts_grad", "n": 16384, "groups": 16, "k": 2048, "m": 4096, "type": "bf16", "out": "f32"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row length: mostly a multiple of 8 as the layers of models have it, sometimes any number."""
    v = _spread(rng, lo, hi)
    return v if rng.random() < 0.3 else max(8, v // 8 * 8)


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "group_rows", "experts", "experts_grad"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    ids = rng.choice(["i32", "i64"])
    if op == "group_rows":
        return {"op": op, "n": _spread(rng, 1, 524288), "ids": _spread(rng, 1, 65536), "id": ids}
    if op in ("lookup", "lookup_grad"):
        width = _width(rng, 16, 4096)
        table = _spread(rng, 100, min(131072, (1 << 28) // width))
        n = _spread(rng, 1, min(262144, (1 << (27 if op == "lookup" else 28)) // width))
        case = {"op": op, "n": n, "ids": table, "width": width, "type": kind, "id": ids}
        if op == "lookup_grad":
            case["out"] = rng.choice([kind, "f32"])
        return case
    groups = _spread(rng, 1, 64)
    k = _width(rng, 32, 4096)
    m = _width(rng, 32, min(4096, (1 << 28) // (groups * k)))
    most = (1 << 38) // (k * m) // (8 if kind == "f32" else 1) // (2 if op == "experts_grad" else 1)
    case = {"op": op, "n": _spread(rng, 1, max(1, min(32768, most))), "groups": groups, "k": k, "m": m, "type": kind}
    if op == "experts_grad":
        case["out"] = rng.choice([kind, "f32"])
    return case


def _frequencies(ids):
    """Frequencies of the tokens of a vocabulary, the most frequent first: natural text falls off as one over the rank."""
    p = 1.0 / (np.arange(ids, dtype=np.float64) + 3.0)
    return p / p.sum()


def _tokens(case, seed, generator):
    """n ids: natural frequencies over a vocabulary, about even over experts; one place in 64 is padding (-1)."""
    n, ids = case["n"], case["ids"]
    if case["op"] == "group_rows":
        p = np.random.default_rng([seed, n, ids]).uniform(0.25, 1.25, ids)
    else:
        p = _frequencies(ids)
    # (the sums of the frequencies are taken on the host, in one order: the same seed gives the same ids)
    upto = torch.from_numpy(np.cumsum(p / p.sum())).to("cuda")
    u = torch.rand(n, device="cuda", dtype=torch.float64, generator=generator)
    t = torch.searchsorted(upto, u).clamp_(max=ids - 1)
    t = torch.randperm(ids, device="cuda", generator=generator)[t]
    t[torch.rand(n, device="cuda", generator=generator) < 1.0 / 64] = -1
    return t.to(ID_TYPES[case["id"]])


def _sizes(case, seed):
    """Rows of each expert: uneven, some empty; the last rows of a padded batch belong to none."""
    rng = np.random.default_rng([seed, case["n"], case["groups"]])
    n, groups = case["n"], case["groups"]
    return [int(v) for v in rng.multinomial(n - n // 64, rng.dirichlet(np.full(groups, 3.0)))]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], dict(case)

    def normal(kind, *shape, scale=1.0):
        x = torch.empty(shape, dtype=DTYPES[kind], device="cuda")
        return x.normal_(0.0, scale, generator=g)

    if op in ("lookup", "lookup_grad", "group_rows"):
        s["tokens"] = _tokens(case, seed, g)
    if op == "lookup":
        s["table"] = normal(case["type"], case["ids"], case["width"], scale=0.02)
        s["scale"] = math.sqrt(case["width"])
        s["rows"] = torch.zeros(case["n"], case["width"], dtype=DTYPES[case["type"]], device="cuda")
    elif op == "lookup_grad":
        s["d_rows"] = normal(case["type"], case["n"], case["width"])
        s["scale"] = math.sqrt(case["width"])
        s["d_table"] = torch.zeros(case["ids"], case["width"], dtype=DTYPES[case["out"]], device="cuda")
    elif op == "group_rows":
        s["order"] = torch.zeros(case["n"], dtype=torch.int32, device="cuda")
        s["offsets"] = torch.zeros(case["ids"] + 1, dtype=torch.int32, device="cuda")
    else:
        n, groups, k, m = case["n"], case["groups"], case["k"], case["m"]
        s["sizes"] = _sizes(case, seed)
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(s["sizes"])]).astype(np.int32)).to("cuda")
        s["x"] = normal(case["type"], n, k)
        s["w"] = normal(case["type"], groups, m, k, scale=1.0 / math.sqrt(k))
        if op == "experts":
            s["y"] = torch.zeros(n, m, dtype=DTYPES[case["type"]], device="cuda")
        else:
            s["d_y"] = normal(case["type"], n, m)
            s["d_x"] = torch.zeros(n, k, dtype=DTYPES[case["type"]], device="cuda")
            s["d_w"] = torch.zeros(groups, m, k, dtype=DTYPES[case["out"]], device="cuda")
    if own:
        # the workspace that a program makes once and keeps
        s["capi"] = importlib.import_module("hp-spmm-sddmm_amd").capi
        if op in ("lookup_grad", "group_rows"):
            s["plan"] = s["capi"].RowsPlan(case["n"], case["ids"], case.get("width", 0))
        elif op == "experts_grad":
            s["plan"] = s["capi"].RowsPlan(case["n"], case["groups"], 0)
    return s


def _run_own(s):
    capi, op = s["capi"], s["op"]
    if op == "lookup":
        return capi.embedding_lookup(s["table"], s["tokens"], s["rows"], scale=s["scale"])
    if op == "lookup_grad":
        return capi.embedding_grad(s["plan"], s["tokens"], s["d_rows"], s["d_table"], scale=s["scale"])
    if op == "group_rows":
        return capi.group_rows(s["plan"], s["tokens"], s["ids"], s["order"], s["offsets"])
    if op == "experts":
        return capi.grouped_mm(s["x"], s["w"], s["offsets"], s["y"])
    return (capi.grouped_mm_grad_x(s["d_y"], s["w"], s["offsets"], s["d_x"]),
            capi.grouped_mm_grad_w(s["plan"], s["d_y"], s["x"], s["offsets"], s["d_w"]))


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op in ("lookup", "lookup_grad", "group_rows"):
        tokens, ids = s["tokens"], s["ids"]
        here = (tokens >= 0) & (tokens < ids)
    if op == "lookup":
        rows = s["table"][tokens.clamp(0, ids - 1)].float() * s["scale"]
        return torch.where(here[:, None], rows, 0.0).to(s["table"].dtype)
    if op == "lookup_grad":
        total = torch.zeros(ids + 1, s["width"], dtype=torch.float32, device="cuda")
        total.index_add_(0, torch.where(here, tokens, ids), s["d_rows"].float())
        return (total[:ids] * s["scale"]).to(s["d_table"].dtype)
    if op == "group_rows":
        key, order = torch.sort(torch.where(here, tokens, ids), stable=True)
        first = torch.searchsorted(key, torch.arange(ids + 1, dtype=key.dtype, device="cuda"))
        return order.to(torch.int32), first.to(torch.int32)
    begin = 0
    for e, size in enumerate(s["sizes"]):
        rows = slice(begin, begin + size)
        begin += size
        if op == "experts":
            if size:
                s["y"][rows] = (s["x"][rows].float() @ s["w"][e].float().t()).to(s["y"].dtype)
        else:
            if size:
                s["d_x"][rows] = (s["d_y"][rows].float() @ s["w"][e].float()).to(s["d_x"].dtype)
            s["d_w"][e] = (s["d_y"][rows].float().t() @ s["x"][rows].float()).to(s["d_w"].dtype)
    return s["y"] if op == "experts" else (s["d_x"], s["d_w"])


def work(case):
    op, n = case["op"], case["n"]
    if op == "group_rows":
        return {"bytes": n * (8 if case["id"] == "i64" else 4) + 4 * n + 4 * (case["ids"] + 1), "flops": 0}
    if op in ("lookup", "lookup_grad"):
        width, size, id_bytes = case["width"], BYTES[case["type"]], 8 if case["id"] == "i64" else 4
        if op == "lookup":
            # a row of the table is read once however often its id occurs
            met = float(np.sum(-np.expm1(n * np.log1p(-_frequencies(case["ids"])))))
            return {"bytes": n * id_bytes + (n + met) * width * size, "flops": n * width}
        return {"bytes": n * id_bytes + n * width * size + case["ids"] * width * BYTES[case["out"]], "flops": n * width}
    size, groups, k, m = BYTES[case["type"]], case["groups"], case["k"], case["m"]
    used = n - n // 64
    met = groups * (1.0 - (1.0 - 1.0 / groups) ** used)  # experts with at least one row
    if op == "experts":
        return {"bytes": (used * (k + m) + met * k * m) * size, "flops": 2.0 * used * k * m}
    return {"bytes": (used * (2 * k + m) + met * k * m) * size + groups * k * m * BYTES[case["out"]], "flops": 4.0 * used * k * m}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("lookup", "lookup_grad", "group_rows"):
        t = s["tokens"].long()
        kept = torch.nonzero((t >= 0) & (t < case["ids"])).flatten()
    if op == "lookup":
        rows = torch.zeros(case["n"], case["width"], dtype=torch.float64, device="cuda")
        rows[kept] = s["table"].index_select(0, t[kept]).double().mul_(s["scale"])
        return rows
    if op == "lookup_grad":
        total = torch.zeros(case["ids"], case["width"], dtype=torch.float64, device="cuda")
        return total.index_add_(0, t[kept], s["d_rows"][kept].double(), alpha=s["scale"])
    if op == "group_rows":
        key = np.where((t.cpu().numpy() >= 0) & (t.cpu().numpy() < case["ids"]), t.cpu().numpy(), case["ids"])
        order = np.lexsort((np.arange(case["n"]), key))
        counts = np.bincount(key, minlength=case["ids"] + 1)[: case["ids"]]
        return order.astype(np.int32), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    bounds = s["offsets"].tolist()
    parts = [(e, b, c) for e, (b, c) in enumerate(zip(bounds[:-1], bounds[1:]))]
    if op == "experts":
        y = torch.zeros(case["n"], case["m"], dtype=torch.float64, device="cuda")
        for e, b, c in parts:
            y[b:c] = torch.nn.functional.linear(s["x"][b:c].double(), s["w"][e].double())
        return y
    d_x = torch.zeros(case["n"], case["k"], dtype=torch.float64, device="cuda")
    d_w = torch.zeros(case["groups"], case["m"], case["k"], dtype=torch.float64, device="cuda")
    for e, b, c in parts:
        d_x[b:c] = torch.mm(s["d_y"][b:c].double(), s["w"][e].double())
        d_w[e] = torch.mm(s["x"][b:c].double().t(), s["d_y"][b:c].double()).t()
    return d_x, d_w
