"""The operators at the two ends of a training step on learned vertex embeddings, as cases to measure: the scaled
embedding lookup and its gradient, the softmax cross entropy of a linear scorer over many classes or vertices and its
gradient, and the clipping of many gradients by their global norm.

`own` False computes a case in elementary torch operations in 32 bits, rounded once at the end; `own` True calls the
classes of featgraph_amd.module."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a handful of vertices looked up for serving in the 4096-vertex graph: latency
        {"name": "lookup-few", "op": "lookup", "dtype": "float32", "n": 61, "rows": 4096, "d": 64, "ids": "int32"},
        # 1024 seed vertices with 10 and 15 sampled neighbours each, in the 232,965-vertex graph
        {"name": "lookup-sampled", "op": "lookup", "dtype": "bfloat16", "n": 164864, "rows": 232965, "d": 128, "ids": "int64"},
        # the gradients of the same two, and of a million lookups in the 2.45M-vertex graph's table
        {"name": "lookup-grad-few", "op": "lookup_grad", "dtype": "float32", "n": 333, "rows": 4096, "d": 100, "ids": "int32"},
        {"name": "lookup-grad-sampled", "op": "lookup_grad", "dtype": "bfloat16", "n": 164864, "rows": 232965, "d": 128, "ids": "int64"},
        {"name": "lookup-grad-large", "op": "lookup_grad", "dtype": "float32", "n": 1000003, "rows": 2449029, "d": 256, "ids": "int32"},
        # evaluation of a small batch on the small graph: latency
        {"name": "loss-few", "op": "loss", "dtype": "float32", "n": 127, "rows": 4096, "d": 64, "ids": "int64"},
        # link prediction: 1024 queries scored against every vertex of the 232,965-vertex graph
        {"name": "loss-all-vertices", "op": "loss", "dtype": "bfloat16", "n": 1024, "rows": 232965, "d": 128, "ids": "int32"},
        # vertex classification, all vertices at once into a few dozen classes: loss and both gradients
        {"name": "step-classes", "op": "step", "dtype": "bfloat16", "n": 232965, "rows": 41, "d": 256, "ids": "int32"},
        # a training step against a large vocabulary, wide features
        {"name": "step-vocabulary", "op": "step", "dtype": "bfloat16", "n": 4096, "rows": 65536, "d": 1024, "ids": "int64"},
        # the framework's own type, at sizes that divide nothing
        {"name": "step-odd", "op": "step", "dtype": "float32", "n": 1003, "rows": 20011, "d": 100, "ids": "int32"},
        # the weights of a small attention layer
        {"name": "clip-layer", "op": "clip", "dtype": "float32", "tensors": 6, "elements": 24700, "mixed": False},
        # a model with a large embedding table: tensors of very different sizes, some of 16 bits
        {"name": "clip-model", "op": "clip", "dtype": "float32", "tensors": 45, "elements": 330000017, "mixed": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "loss", "step", "clip"])
    if op == "clip":
        return {"op": op, "dtype": rng.choice(["float32", "bfloat16", "float16"]), "tensors": _log(rng, 1, 48),
                "elements": _log(rng, 20000, 300000000), "mixed": rng.random() < 0.5}
    ids = rng.choice(["int32", "int64"])
    if op in ("lookup", "lookup_grad"):
        rows, d = _log(rng, 1000, 2449029), _log(rng, 30, 1024)
        n = _log(rng, 1, 1000003)
        while (n + rows) * d > 880000000:
            d = max(30, d // 2)
            n, rows = (n * 3 // 4, rows) if d == 30 else (n, rows)
        return {"op": op, "dtype": rng.choice(["float32", "bfloat16", "float16"]), "n": n, "rows": rows, "d": d, "ids": ids}
    dtype = rng.choice(["float32", "bfloat16"])
    n, rows, d = _log(rng, 16, 232965), _log(rng, 16, 232965), _log(rng, 30, 1024)
    most = 1 << 29 if dtype == "float32" else 1 << 30
    while n * rows > 1 << 28 or n * rows * d > most * 64:  # logits that the plain form can hold, products of bounded cost
        if n > rows:
            n = n * 2 // 3
        else:
            rows = rows * 2 // 3
    return {"op": op, "dtype": dtype, "n": n, "rows": rows, "d": d, "ids": ids}


def _sizes(case):
    """Element counts of the tensors to clip: one large table, the others falling off by a power."""
    t, total = case["tensors"], case["elements"]
    share = [(i + 1.0) ** -1.5 for i in range(t)]
    sizes = [max(1, int(total * s / sum(share))) for s in share]
    return [s + (i % 3) for i, s in enumerate(sizes)]


def _type_of(case, i):
    if case["mixed"] and i % 3 == 1:
        return torch.bfloat16
    return TYPES[case["dtype"]]


def _ids(g, n, rows, dtype, padding):
    """Vertices met in proportion to a power law, spread over the ids; a share of them padding (-1)."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    i = (u * u * u * rows).long().clamp_(max=rows - 1)
    i = (i * 1000003 + 17) % rows
    i[torch.rand(n, generator=g, device="cuda") < padding] = -1
    return i.to(getattr(torch, dtype))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or TYPES[case["dtype"]])

    op, s = case["op"], {"case": dict(case)}
    if op == "clip":
        s["grads"] = [normal(n, scale=10.0 ** -(i % 4), dtype=_type_of(case, i)) for i, n in enumerate(_sizes(case))]
        norm = math.sqrt(sum(n * 100.0 ** -(i % 4) for i, n in enumerate(_sizes(case))))
        s["max_norm"] = norm * (0.25 if seed % 2 else 0.5)
    else:
        n, rows, d = case["n"], case["rows"], case["d"]
        s["ids"] = _ids(g, n, rows, case["ids"], 0.02)
        s["scale"] = math.sqrt(d)
        if op == "lookup":
            s["table"] = normal(rows, d, scale=0.1)
        elif op == "lookup_grad":
            s["dout"] = normal(n, d, scale=1.0 / n)
        else:
            s["hidden"] = normal(n, d)
            s["weight"] = normal(rows, d, scale=1.5 / math.sqrt(d))
            s["dloss"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    if own:
        s["modules"] = _modules(case, s)
    return s


def _modules(case, s):
    """The built operators that a user's program keeps over its steps."""
    from featgraph_amd import module, placeholder
    op = case["op"]
    if op == "clip":
        m = module.ClipGradNormhip(s["max_norm"])
        m.build([placeholder(tuple(x.shape), str(x.dtype).replace("torch.", "")) for x in s["grads"]])
        return (m,)
    ids = placeholder((case["n"],), case["ids"])
    table = placeholder((case["rows"], case["d"]), case["dtype"])
    if op in ("lookup", "lookup_grad"):
        m = (module.EmbeddingLookuphip if op == "lookup" else module.EmbeddingLookupGradhip)(scale=s["scale"])
        m.build([table, ids])
        return (m,)
    hidden = placeholder((case["n"], case["d"]), case["dtype"])
    loss = module.LinearCrossEntropyhip()
    loss.build([hidden, table, ids])
    if op == "loss":
        return (loss,)
    grad = module.LinearCrossEntropyGradhip()
    grad.build([hidden, table, ids])
    return (loss, grad)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        m = state["modules"]
        if op == "clip":
            norm, clipped = m[0].run(state["grads"])
            return {"norm": norm.tensor, "clipped": [x.tensor for x in clipped]}
        if op == "lookup":
            return m[0].run([state["table"], state["ids"]]).tensor
        if op == "lookup_grad":
            return m[0].run([state["ids"], state["dout"]]).tensor
        loss, lse = m[0].run([state["hidden"], state["weight"], state["ids"]])
        if op == "loss":
            return {"loss": loss.tensor, "lse": lse.tensor}
        dhidden, dweight = m[1].run([state["hidden"], state["weight"], state["ids"], lse, state["dloss"]])
        return {"loss": loss.tensor, "lse": lse.tensor, "dhidden": dhidden.tensor, "dweight": dweight.tensor}
    if op == "clip":
        squares = torch.stack([x.float().square().sum() for x in state["grads"]])
        norm = squares.sum().sqrt()
        c = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        return {"norm": norm, "clipped": [(x.float() * c).to(x.dtype) for x in state["grads"]]}
    ids = state["ids"].long()
    there = ids >= 0
    safe = ids.clamp(min=0)
    if op == "lookup":
        rows = state["table"][safe].float() * state["scale"]
        return torch.where(there[:, None], rows, 0.0).to(TYPES[case["dtype"]])
    if op == "lookup_grad":
        grad = torch.zeros(case["rows"], case["d"], device="cuda")
        grad.index_add_(0, safe, torch.where(there[:, None], state["dout"].float(), 0.0))
        return (grad * state["scale"]).to(TYPES[case["dtype"]])
    h, w = state["hidden"].float(), state["weight"].float()
    logits = h @ w.T
    top = logits.amax(1, keepdim=True)
    p = (logits - top).exp()
    total = p.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    loss = torch.where(there, lse - logits.gather(1, safe[:, None])[:, 0], 0.0)
    if op == "loss":
        return {"loss": loss, "lse": lse}
    p = p / total
    p[torch.arange(case["n"], device="cuda"), safe] -= 1.0
    p = p * torch.where(there, state["dloss"], 0.0)[:, None]
    kind = TYPES[case["dtype"]]
    return {"loss": loss, "lse": lse, "dhidden": (p @ w).to(kind), "dweight": (p.T @ h).to(kind)}


def work(case):
    op = case["op"]
    if op == "clip":
        size = sum(n * _type_of(case, i).itemsize for i, n in enumerate(_sizes(case)))
        return {"bytes": 2 * size, "flops": 3 * sum(_sizes(case))}
    n, rows, d, es = case["n"], case["rows"], case["d"], TYPES[case["dtype"]].itemsize
    ids = n * (4 if case["ids"] == "int32" else 8)
    if op == "lookup":
        return {"bytes": ids + (n + min(n, rows)) * d * es, "flops": n * d}
    if op == "lookup_grad":
        return {"bytes": ids + (n + rows) * d * es, "flops": 2 * n * d}
    if op == "loss":
        return {"bytes": ids + (n + rows) * d * es + 8 * n, "flops": 2 * n * rows * d}
    return {"bytes": ids + 2 * (n + rows) * d * es + 12 * n, "flops": 6 * n * rows * d}


def exact(case, seed):
    global own
    kept, own = own, False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "clip":
        norm = math.sqrt(sum(float(torch.dot(x.double(), x.double())) for x in s["grads"]))
        c = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "clipped": [x.double() * c for x in s["grads"]]}
    ids = s["ids"].to(torch.int64)
    valid = torch.nonzero(ids != -1)[:, 0]
    at = ids[valid]
    n, rows, d = case["n"], case["rows"], case["d"]
    if op == "lookup":
        out = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        out[valid] = torch.index_select(s["table"], 0, at).double().mul_(s["scale"])
        return out
    if op == "lookup_grad":
        out = torch.zeros(rows, d, dtype=torch.float64, device="cuda")
        return out.index_put_((at,), s["dout"][valid].double() * s["scale"], accumulate=True)
    h, w = s["hidden"].double(), s["weight"].double()
    scores = torch.mm(h, w.t().contiguous())
    lse = torch.logsumexp(scores, 1)
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    loss[valid] = lse[valid] - scores[valid, at]
    if op == "loss":
        return {"loss": loss, "lse": lse}
    scores = torch.exp(scores.sub_(lse[:, None]))
    weight = torch.zeros(n, dtype=torch.float64, device="cuda")
    weight[valid] = s["dloss"][valid].double()
    scores *= weight[:, None]
    scores[valid, at] -= weight[valid]
    return {"loss": loss, "lse": lse, "dhidden": torch.mm(scores, w), "dweight": torch.mm(scores.t().contiguous(), h)}
