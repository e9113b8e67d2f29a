"""Products grouped by ragged sets of rows, embeddings with the gradient of their table, and the norm and clipping of gradients: calls that
stand for the use of these operators.

The framework routes per-atom rows to groups (elements, fine-tuned variants, experts) and trains small parts of a model. What a program does with
the routed rows is a linear of every group's own; what it starts from is an embedding of elements, or of (variant, element) pairs; what it does
with all gradients before a step is clip them by their common norm.

* ``grouped``: rows in the order of the groups times each group's own matrices, all degrees.
* ``grouped_train``: forward and backward pass of such a linear, the matrices' gradients clipped.
* ``embed``: the rows of a table that a batch's tokens name, weighted.
* ``embed_train``: a batch's tokens sorted, the lookup, the gradients of the table and of the weights.
* ``clip``: the norm over many tensors, and the tensors scaled to at most that norm.

A row of the arrays is an atom (or one of its slots): the (2l+1) components of degree 0, then those of degree 1, and so on, with their channels.
``paths`` counts the channel blocks that each degree's input rows concatenate, as in the linears of an evaluator (2+3+3+2: behind the tensor
product of 16 harmonics with scalars and vectors).
"""
import math
import random

import torch

own = False


def listed():
    return [
        # two molecules, each atom with two of seven groups: what a call costs at least
        {"name": "grouped_molecule_f64", "op": "grouped", "dtype": "float64", "atoms": 18, "slots": 2, "groups": 7, "paths": "1+1", "channels": 128,
         "out": 128, "request": 9},
        # a batch of small structures, one variant each
        {"name": "grouped_batch_f32", "op": "grouped", "dtype": "float32", "atoms": 4001, "slots": 1, "groups": 16, "paths": "1+1", "channels": 128,
         "out": 128, "request": 37},
        # a large box, every atom with a linear of its element (as many as the periodic table's models have)
        {"name": "grouped_elements_f32", "op": "grouped", "dtype": "float32", "atoms": 98304, "slots": 1, "groups": 89, "paths": "1+1", "channels": 128,
         "out": 128, "request": 1},
        # one step of training behind the tensor product, two experts an atom
        {"name": "train_batch_f32", "op": "grouped_train", "dtype": "float32", "atoms": 8001, "slots": 2, "groups": 8, "paths": "2+3+3+2", "channels": 128,
         "out": 128, "request": 99, "max_norm": 1.0},
        # wide features in double precision, odd sizes
        {"name": "train_odd_f64", "op": "grouped_train", "dtype": "float64", "atoms": 1029, "slots": 1, "groups": 5, "paths": "1+1+1", "channels": 131,
         "out": 97, "request": 21, "max_norm": 1.0},
        # one molecule's elements
        {"name": "embed_molecule_f64", "op": "embed", "dtype": "float64", "atoms": 18, "slots": 1, "table": 10, "width": 128, "skew": 0.5},
        # a large box, rows of scalars and vectors
        {"name": "embed_large_f32", "op": "embed", "dtype": "float32", "atoms": 98304, "slots": 1, "table": 89, "width": 512, "skew": 0.5},
        # (variant, element) pairs, two a row, of sixteen variants of a model with 89 elements
        {"name": "embed_train_pairs_f32", "op": "embed_train", "dtype": "float32", "atoms": 49152, "slots": 2, "table": 1424, "width": 512, "skew": 0.5},
        # water: two tokens, one of them twice as often; wide rows
        {"name": "embed_train_water_f64", "op": "embed_train", "dtype": "float64", "atoms": 4001, "slots": 1, "table": 2, "width": 2304, "skew": 1.0},
        # gradients of one linear's adapters
        {"name": "clip_adapters_f64", "op": "clip", "dtype": "float64", "tensors": 6, "values": 40960, "shape": 1, "max_norm": 1.0},
        # gradients of all adapters of a few models in training, ragged
        {"name": "clip_many_f32", "op": "clip", "dtype": "float32", "tensors": 407, "values": 6000001, "shape": 2, "max_norm": 1.0},
        # a whole model's gradients, some of them kept in double precision
        {"name": "clip_model_mixed", "op": "clip", "dtype": "mixed", "tensors": 96, "values": 64000000, "shape": 3, "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    most = {}
    for c in listed():
        kind = c["op"].split("_")[0]
        for k, v in work(c).items():
            most[kind, k] = max(most.get((kind, k), 0), v)
    while True:
        op = rng.choice(["grouped", "grouped_train", "embed", "embed_train", "clip"])
        kind = op.split("_")[0]
        case = {"op": op, "dtype": rng.choice(["float32", "float64"])}
        if kind == "clip":
            case["dtype"] = rng.choice(["float32", "float64", "mixed"])
            case.update(tensors=_log_int(rng, 1, 2000), values=_log_int(rng, 4096, 64000000), shape=rng.randint(0, 10 ** 6),
                        max_norm=rng.choice([0.5, 1.0, 1.0, 10.0, 1e6]))
        elif kind == "embed":
            case.update(atoms=_log_int(rng, 18, 98304), slots=rng.choice([1, 1, 2, 3]), table=_log_int(rng, 1, 20000),
                        width=rng.choice([1, 4, 9]) * _log_int(rng, 15, 256), skew=rng.choice([0.0, 0.5, 1.0]))
        else:
            case.update(atoms=_log_int(rng, 18, 98304), slots=rng.choice([1, 1, 2, 3]), groups=_log_int(rng, 1, 128), request=_log_int(rng, 1, 1500),
                        paths=rng.choice(["1", "1+1", "1+1+1", "2+3+3+2"]), channels=rng.choice([64, 128, 256, _log_int(rng, 15, 256)]),
                        out=rng.choice([64, 128, 256, _log_int(rng, 15, 256)]))
            if op == "grouped_train":
                case["max_norm"] = rng.choice([1.0, 100.0, 1e6])
        w = work(case)
        limit = 0.25 if case["dtype"] == "float64" and kind == "grouped" else 1.0      # double precision costs more an operation
        if all(w[k] <= limit * most[kind, k] for k in w):
            return case


# ------------------------------------------------------------------------------------------- sizes

def _degrees(case):
    """(components, input channels, output channels) of every degree."""
    return [(2 * l + 1, int(p) * case["channels"], case["out"]) for l, p in enumerate(case["paths"].split("+"))]


def _lengths(case):
    """Values of every tensor of a ``clip`` case: from single numbers to a fifth of all."""
    rng = random.Random(case["shape"])
    share = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["values"] * s / sum(share))) for s in share]


def _types(case):
    """The type of every tensor of a ``clip`` case: in ``mixed`` ones every eighth is kept in double precision."""
    wide = {"float32": lambda i: False, "float64": lambda i: True, "mixed": lambda i: i % 8 == 5}[case["dtype"]]
    return [torch.float64 if wide(i) else torch.float32 for i in range(case["tensors"])]


def _starts(case):
    """Where every tensor of a ``clip`` case starts in the buffer of its type: on a multiple of 16 bytes."""
    at, starts = {torch.float32: 0, torch.float64: 0}, []
    for n, t in zip(_lengths(case), _types(case)):
        starts.append(at[t])
        at[t] += -(-n // 4) * 4
    return starts, at


def _flat_sizes(case):
    return {t: n for t, n in _starts(case)[1].items() if n}


def _views(case, flat):
    return [flat[t][a:a + n] for n, t, a in zip(_lengths(case), _types(case), _starts(case)[0])]


def work(case):
    size = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "clip":
        bytes_ = sum(n * (8 if t is torch.float64 else 4) for n, t in zip(_lengths(case), _types(case)))
        return {"bytes": 2 * bytes_ + 8, "flops": 3 * sum(_lengths(case))}
    n, s = case["atoms"], case["slots"]
    if case["op"].startswith("embed"):
        w, used = case["width"], min(case["table"], n * s)
        if case["op"] == "embed":
            return {"bytes": 4 * n * s + size * (n * s + used * w + n * w), "flops": 2 * n * s * w}
        return {"bytes": 8 * n * s + size * (2 * n * s + used * w + 2 * n * w + case["table"] * w), "flops": 6 * n * s * w}
    pairs = n * s
    wide_in, wide_out = (sum(c * d[i] for c, *d in _degrees(case)) for i in (0, 1))
    weights = min(case["groups"], pairs) * sum(i * o for _, i, o in _degrees(case))
    product = sum(2 * pairs * c * i * o for c, i, o in _degrees(case))
    if case["op"] == "grouped":
        return {"bytes": size * (pairs * (wide_in + wide_out) + weights), "flops": product}
    grads = case["groups"] * sum(i * o for _, i, o in _degrees(case))
    return {"bytes": size * (pairs * 2 * (wide_in + wide_out) + weights + grads), "flops": 3 * product}


# ------------------------------------------------------------------------------------------- inputs

def _ids(case, gen):
    """Groups of every (atom, slot): one draw a request; a few groups serve most of them, and one slot in twelve is empty."""
    n, s, g = case["atoms"], case["slots"], case["groups"]
    requests = -(-n // case["request"])
    score = torch.rand(requests, g, generator=gen, device="cuda") ** (1.0 / (1.0 + torch.arange(g, device="cuda")) ** -0.5)
    chosen = score.topk(min(s, g), dim=1).indices.to(torch.int32)
    if s > g:
        chosen = torch.cat([chosen, chosen[:, :1].expand(requests, s - g)], dim=1)
    chosen[torch.rand(requests, s, generator=gen, device="cuda") < 1.0 / 12.0] = -1
    return chosen.repeat_interleave(case["request"], dim=0)[:n].contiguous()


def _arrays(case, seed):
    """All inputs, drawn on the GPU from the seed."""
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = torch.float64 if case["dtype"] == "float64" else torch.float32

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype) * scale

    if case["op"] == "clip":
        # layers differ in the size of their gradients by some orders of magnitude
        scales = (torch.rand(case["tensors"], generator=gen, device="cuda") * 6.0 - 4.0).tolist()
        return {"grads": [normal(n, scale=10.0 ** e, dtype=t) for n, t, e in zip(_lengths(case), _types(case), scales)]}
    n, s = case["atoms"], case["slots"]
    if case["op"].startswith("embed"):
        v = case["table"]
        share = (1.0 + torch.arange(v, device="cuda", dtype=torch.float64)) ** -case["skew"]
        bounds = share.cumsum(0) / share.sum()
        names = torch.randperm(v, generator=gen, device="cuda").to(torch.int32)       # which tokens are the frequent ones
        ids = names[torch.searchsorted(bounds, torch.rand(n, s, generator=gen, device="cuda", dtype=torch.float64)).clamp(max=v - 1)]
        ids[torch.rand(n, s, generator=gen, device="cuda") < 0.02] = -1               # rows that pad a batch
        weights = torch.softmax(normal(n, s), dim=1) if s > 1 else 0.5 + torch.rand(n, 1, generator=gen, device="cuda", dtype=dt)
        out = {"ids": ids.contiguous(), "weights": weights.contiguous(), "table": normal(v, case["width"])}
        if case["op"] == "embed_train":
            out["grad_y"] = normal(n, case["width"])
        return out
    deg = _degrees(case)
    out = {"ids": _ids(case, gen), "rows": normal(n * s, sum(c * i for c, i, _ in deg)),
           "matrices": [normal(case["groups"], i, o, scale=i ** -0.5) for _, i, o in deg]}
    if case["op"] == "grouped_train":
        out["grad_y"] = normal(n * s, sum(c * o for c, _, o in deg))
    return out


def prepare(case, seed):
    state = _arrays(case, seed)
    state["case"] = case
    kind = case["op"].split("_")[0]
    if kind == "clip":
        # a buffer for each type, as programs keep them that hand all gradients on at once
        state["flat"] = {t: torch.zeros(n, dtype=t, device="cuda") for t, n in _flat_sizes(case).items()}
        state["out"] = _views(case, state["flat"])
    if own:
        from symmetrix_b200 import Embedding, GradientSet, GroupedLinear, RowRouting
        if kind == "grouped":
            state["routing"] = RowRouting(state["ids"], case["groups"])
            state["layer"] = GroupedLinear(state["matrices"])
        elif kind == "embed":
            state["embedding"] = Embedding(state["table"])
        else:
            state["set"] = GradientSet(state["grads"], out=state["out"])
    elif kind == "grouped":
        flat = state["ids"].reshape(-1)
        counts = torch.bincount(flat[flat >= 0], minlength=case["groups"])
        state["bounds"] = [0] + counts.cumsum(0).tolist()
    return state


# ------------------------------------------------------------------------------------------- plain forms

def _norm_and_factor(tensors, max_norm):
    """The common norm, in 64 bits since the sum is long, and what the tensors are multiplied by."""
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in tensors:
        d = t.double()
        total = total + (d * d).sum()
    norm = total.sqrt()
    return norm, torch.where(norm > max_norm, max_norm / norm, torch.ones_like(norm))


def _plain_grouped(st):
    """Each group's rows times its matrices, one after the other."""
    case, rows, bounds = st["case"], st["rows"], st["bounds"]
    train = case["op"] == "grouped_train"
    deg = _degrees(case)
    y = rows.new_zeros(rows.shape[0], sum(c * o for c, _, o in deg))
    grad_x, grad_w = torch.zeros_like(rows) if train else None, [torch.zeros_like(w) for w in st["matrices"]] if train else None
    at_x = at_y = 0
    for d, ((c, i, o), w) in enumerate(zip(deg, st["matrices"])):
        for g in range(case["groups"]):
            a, b = bounds[g], bounds[g + 1]
            if a == b:
                continue
            x = rows[a:b, at_x:at_x + c * i].reshape(-1, i)
            y[a:b, at_y:at_y + c * o] = (x @ w[g]).reshape(b - a, c * o)
            if train:
                gy = st["grad_y"][a:b, at_y:at_y + c * o].reshape(-1, o)
                grad_x[a:b, at_x:at_x + c * i] = (gy @ w[g].T).reshape(b - a, c * i)
                grad_w[d][g] = x.T @ gy
        at_x += c * i
        at_y += c * o
    if not train:
        return {"y": y}
    _, factor = _norm_and_factor(grad_w, case["max_norm"])
    return {"y": y, "grad_x": grad_x, "grad_w": [t * factor.to(t.dtype) for t in grad_w]}


def _plain_embed(st):
    ids, weights, table = st["ids"], st["weights"], st["table"]
    live = (ids >= 0).to(table.dtype) * weights
    at = ids.clamp(min=0).long()
    y = live[:, 0, None] * table[at[:, 0]]
    for q in range(1, ids.shape[1]):
        y += live[:, q, None] * table[at[:, q]]
    if st["case"]["op"] == "embed":
        return {"y": y}
    grad_y = st["grad_y"]
    sums = torch.zeros(table.shape, dtype=torch.float64, device="cuda")      # long sums
    grad_w = torch.zeros_like(weights)
    for q in range(ids.shape[1]):
        sums.index_add_(0, at[:, q], (live[:, q, None] * grad_y).double())
        grad_w[:, q] = (ids[:, q] >= 0) * (table[at[:, q]] * grad_y).sum(1)
    v = table.shape[0]
    key = torch.where(ids < 0, torch.full_like(ids, v), ids).reshape(-1)
    return {"order": torch.sort(key, stable=True).indices.to(torch.int32), "y": y, "grad_table": sums.to(table.dtype), "grad_weights": grad_w}


def _plain_clip(st):
    norm, factor = _norm_and_factor(st["grads"], st["case"]["max_norm"])
    for t, to in zip(st["grads"], st["out"]):
        torch.mul(t, factor.to(t.dtype), out=to)
    return {"norm": norm, "grads": list(st["flat"].values())}


# ------------------------------------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    kind = case["op"].split("_")[0]
    if not own:
        return {"grouped": _plain_grouped, "embed": _plain_embed, "clip": _plain_clip}[kind](state)
    from symmetrix_b200 import EmbeddingPlan, clip_gradients
    if kind == "clip":
        return {"norm": state["set"].clip(case["max_norm"]), "grads": list(state["flat"].values())}
    if kind == "embed":
        embedding = state["embedding"]
        y = embedding.forward(state["ids"], state["weights"])
        if case["op"] == "embed":
            return {"y": y}
        plan = EmbeddingPlan(state["ids"], case["table"])
        grads = embedding.backward(state["grad_y"], plan, state["weights"])
        return {"order": plan.order, "y": y, "grad_table": grads.table, "grad_weights": grads.weights}
    layer, routing = state["layer"], state["routing"]
    y = layer.forward(state["rows"], routing)
    if case["op"] == "grouped":
        return {"y": y}
    grads = layer.backward(state["rows"], state["grad_y"], routing)
    clip_gradients(grads.weights, case["max_norm"])
    return {"y": y, "grad_x": grads.x, "grad_w": list(grads.weights)}


# ------------------------------------------------------------------------------------------- definition in 64 bits

def exact(case, seed):
    """The same outputs from the definitions, in 64 bits."""
    data = _arrays(case, seed)
    if case["op"] == "clip":
        wide = [t.double() for t in data["grads"]]
        norm = torch.sqrt(torch.stack([torch.dot(t, t) for t in wide]).sum())
        scale = min(1.0, case["max_norm"] / float(norm))
        flat = {t: torch.zeros(n, dtype=torch.float64, device="cuda") for t, n in _flat_sizes(case).items()}
        for t, to in zip(wide, _views(case, flat)):
            to.copy_(t * scale)
        return {"norm": norm, "grads": list(flat.values())}
    if case["op"].startswith("embed"):
        ids, v = data["ids"].reshape(-1).long(), case["table"]
        n, s = case["atoms"], case["slots"]
        live = torch.nonzero(ids >= 0)[:, 0]
        atoms, names, w = live // s, ids[live], data["weights"].double().reshape(-1)[live]
        table = data["table"].double()
        y = torch.zeros(n, case["width"], dtype=torch.float64, device="cuda").index_add_(0, atoms, w[:, None] * table[names])
        if case["op"] == "embed":
            return {"y": y}
        gy = data["grad_y"].double()[atoms]
        grad_table = torch.zeros_like(table).index_add_(0, names, w[:, None] * gy)
        grad_weights = torch.zeros(n * s, dtype=torch.float64, device="cuda")
        grad_weights[live] = torch.einsum("pw,pw->p", table[names], gy)
        # by token, equal ones and those without a token in the order of the list
        place = torch.where(ids < 0, torch.full_like(ids, v), ids) * (n * s) + torch.arange(n * s, device="cuda")
        return {"order": place.argsort().to(torch.int32), "y": y, "grad_table": grad_table, "grad_weights": grad_weights.reshape(n, s)}
    n, s = case["atoms"], case["slots"]
    key = data["ids"].reshape(-1)
    sorted_groups = key[key >= 0].sort().values                              # of the rows, which are in the groups' order
    last = sorted_groups.numel()
    train = case["op"] == "grouped_train"
    ys, gxs, gws = [], [], []
    at_x = at_y = 0
    for (c, i, o), w in zip(_degrees(case), data["matrices"]):
        w = w.double()
        x = data["rows"][:, at_x:at_x + c * i].double().reshape(n * s, c, i)
        y = torch.zeros(n * s, c, o, dtype=torch.float64, device="cuda")
        if train:
            gy = data["grad_y"][:, at_y:at_y + c * o].double().reshape(n * s, c, o)
            gx, gw = torch.zeros_like(x), torch.zeros_like(w)
        for g in range(case["groups"]):
            mine = torch.nonzero(sorted_groups == g)[:, 0]
            if mine.numel() == 0:
                continue
            y[mine] = torch.einsum("pci,io->pco", x[mine], w[g])
            if train:
                gx[mine] = torch.einsum("pco,io->pci", gy[mine], w[g])
                gw[g] = torch.einsum("pci,pco->io", x[mine], gy[mine])
        assert last == n * s or not y[last:].any()
        ys.append(y.reshape(n * s, c * o))
        if train:
            gxs.append(gx.reshape(n * s, c * i))
            gws.append(gw)
        at_x += c * i
        at_y += c * o
    if not train:
        return {"y": torch.cat(ys, dim=1)}
    norm = math.sqrt(sum(float((t * t).sum()) for t in gws))
    scale = min(1.0, case["max_norm"] / norm) if norm > 0 else 1.0
    return {"y": torch.cat(ys, dim=1), "grad_x": torch.cat(gxs, dim=1), "grad_w": [t * scale for t in gws]}
