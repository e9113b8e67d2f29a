"""Rows routed to groups and back, and linears with low-rank adapters: calls that stand for the use of these operators.

The framework evaluates one model on many structures. Fine-tuned variants of the model are low-rank adapters of its channel-mixing
linears; every structure (a request) names its adapter, or several with mixing weights. A row of the arrays is an atom: all (2l+1)
components of all degrees with their channels.

* ``route``: atoms sorted by group, their rows copied to sorted order, and the groups' results brought back with weights.
* ``route_grad``: the gradients of both directions, with a plan kept from the forward pass.
* ``adapter``: a linear of all degrees with every atom's adapter beside the shared weights, on a kept plan.
* ``adapter_train``: one step of fine-tuning at such a linear: new adapters laid out, forward and backward pass.

``paths`` counts the channel blocks that each degree's input rows concatenate: one for a block's features (``compute_H1``), several for
the tensor product's outputs (``compute_A1``; 2+3+3+2 is the product of 16 harmonics with scalars and vectors).
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # two molecules, each atom with two of seven variants: what a call costs at least
        {"name": "route_molecule_f64", "op": "route", "dtype": "float64", "atoms": 18, "slots": 2, "groups": 7, "width": 512, "request": 9},
        # a batch of small structures, one variant each
        {"name": "route_batch_f32", "op": "route", "dtype": "float32", "atoms": 4001, "slots": 1, "groups": 16, "width": 512, "request": 37},
        # every atom chooses two of sixty-four groups by itself: no runs of equal groups, the largest box
        {"name": "route_scattered_f32", "op": "route", "dtype": "float32", "atoms": 98304, "slots": 2, "groups": 64, "width": 512, "request": 1},
        # wide features in double precision, three groups an atom
        {"name": "route_grad_wide_f64", "op": "route_grad", "dtype": "float64", "atoms": 1029, "slots": 3, "groups": 11, "width": 2304, "request": 21},
        # the backward pass of a large batch
        {"name": "route_grad_large_f32", "op": "route_grad", "dtype": "float32", "atoms": 49152, "slots": 2, "groups": 64, "width": 512, "request": 1},
        # one molecule of each of two variants: latency of a linear
        {"name": "adapter_molecule_f64", "op": "adapter", "dtype": "float64", "atoms": 18, "slots": 1, "groups": 2, "paths": "1+1", "channels": 128,
         "rank": 4, "request": 9},
        # sixteen variants on a batch of small liquids, first block's features
        {"name": "adapter_batch_f32", "op": "adapter", "dtype": "float32", "atoms": 4001, "slots": 1, "groups": 16, "paths": "1+1", "channels": 128,
         "rank": 16, "request": 37},
        # the same atoms in double precision, a mixture of two variants each, the linear behind the tensor product
        {"name": "adapter_mixture_f64", "op": "adapter", "dtype": "float64", "atoms": 2003, "slots": 2, "groups": 8, "paths": "2+3+3+2", "channels": 128,
         "rank": 8, "request": 100},
        # a large box cut into many requests
        {"name": "adapter_large_f32", "op": "adapter", "dtype": "float32", "atoms": 98304, "slots": 1, "groups": 48, "paths": "1+1", "channels": 128,
         "rank": 32, "request": 1500},
        # fine-tuning one variant on a handful of cells
        {"name": "train_small_f64", "op": "adapter_train", "dtype": "float64", "atoms": 207, "slots": 1, "groups": 1, "paths": "1+1+1", "channels": 64,
         "rank": 5, "request": 23},
        # fine-tuning eight variants side by side, behind the tensor product
        {"name": "train_batch_f32", "op": "adapter_train", "dtype": "float32", "atoms": 8001, "slots": 1, "groups": 8, "paths": "2+3+3+2",
         "channels": 128, "rank": 16, "request": 99},
        # mixtures with trained weights on wide features
        {"name": "train_mixture_f32", "op": "adapter_train", "dtype": "float32", "atoms": 2664, "slots": 2, "groups": 5, "paths": "1+1+1", "channels": 256,
         "rank": 24, "request": 72},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    top = [work(c) for c in listed()]
    most = {k: max(t[k] for t in top) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["route", "route_grad", "adapter", "adapter", "adapter_train"])
        case = {"op": op, "dtype": rng.choice(["float32", "float64"]), "atoms": _log_int(rng, 18, 98304), "slots": rng.choice([1, 1, 2, 3]),
                "groups": _log_int(rng, 1, 64), "request": _log_int(rng, 1, 1500)}
        if op.startswith("route"):
            case["width"] = rng.choice([1, 4, 9]) * _log_int(rng, 15, 256)
        else:
            case["paths"] = rng.choice(["1", "1+1", "1+1+1", "2+3+3+2"])
            case["channels"] = rng.choice([64, 128, 256, _log_int(rng, 15, 256)])
            case["rank"] = rng.choice([4, 8, 16, 32, rng.randint(1, 64)])
        w = work(case)
        limit = 1.0 if case["dtype"] == "float32" else 0.25      # double precision costs more a byte and an operation
        if all(w[k] <= limit * most[k] for k in w):
            return case


# ------------------------------------------------------------------------------------------- sizes

def _degrees(case):
    """(components, input channels, output channels) of every degree."""
    return [(2 * l + 1, int(p) * case["channels"], case["channels"]) for l, p in enumerate(case["paths"].split("+"))]


def work(case):
    size = 4 if case["dtype"] == "float32" else 8
    n, s, g = case["atoms"], case["slots"], case["groups"]
    if case["op"] == "route":
        w = case["width"]       # ids; x in, rows out; rows, weights, base in, y out; the plan's order and offsets out
        return {"bytes": 4 * n * s + size * w * (n + n * s) + size * (w * (n * s + 2 * n) + n * s) + 4 * (n * s + g + 1), "flops": 2 * n * s * w}
    if case["op"] == "route_grad":
        w = case["width"]       # gradient of rows in, of x out; gradient of y, rows, weights in, both gradients out; the plan in
        return {"bytes": size * w * (n * s + n) + size * (w * (n + 2 * n * s) + 2 * n * s) + 4 * n * s, "flops": 4 * n * s * w}
    wide_in, wide_out = (sum(c * d[i] for c, *d in _degrees(case)) for i in (0, 1))
    shared = sum(i * o for _, i, o in _degrees(case))
    adapters = g * case["rank"] * sum(i + o for _, i, o in _degrees(case))
    product = sum(2 * n * c * (i * o + s * case["rank"] * (i + o)) for c, i, o in _degrees(case))
    if case["op"] == "adapter":
        return {"bytes": size * (n * (wide_in + wide_out) + shared + adapters + n * s) + 4 * n * s, "flops": product}
    grads = sum(2 * n * c * s * case["rank"] * (i + o) for c, i, o in _degrees(case))
    return {"bytes": size * (n * (2 * wide_in + 2 * wide_out) + shared + 2 * adapters + 2 * n * s) + 4 * n * s, "flops": 2 * product + grads}


# ------------------------------------------------------------------------------------------- inputs

def _arrays(case, seed):
    """All inputs, drawn on the GPU from the seed (on the host the largest would take seconds)."""
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = torch.float32 if case["dtype"] == "float32" else torch.float64

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dt) * scale

    n, s, g = case["atoms"], case["slots"], case["groups"]
    requests = -(-n // case["request"])
    # groups by popularity: a few variants serve most requests; distinct ones for the slots of a request where there are enough
    score = torch.rand(requests, g, generator=gen, device="cuda") ** (1.0 / (1.0 + torch.arange(g, device="cuda")) ** -0.5)
    chosen = score.topk(min(s, g), dim=1).indices.to(torch.int32)
    if s > g:
        chosen = torch.cat([chosen, chosen[:, :1].expand(requests, s - g)], dim=1)
    # one request in twelve runs the model as it is, or uses a slot less
    chosen[torch.rand(requests, s, generator=gen, device="cuda") < 1.0 / 12.0] = -1
    ids = chosen.repeat_interleave(case["request"], dim=0)[:n].contiguous()
    mix = torch.softmax(normal(requests, s), dim=1) if s > 1 else 0.5 + torch.rand(requests, 1, generator=gen, device="cuda", dtype=dt)
    weights = mix.repeat_interleave(case["request"], dim=0)[:n].contiguous()
    out = {"ids": ids, "weights": weights}
    if case["op"] == "route":
        out.update(x=normal(n, case["width"]), rows=normal(n * s, case["width"]), base=normal(n, case["width"]))
    elif case["op"] == "route_grad":
        out.update(grad_rows=normal(n * s, case["width"]), grad_y=normal(n, case["width"]), rows=normal(n * s, case["width"]))
    else:
        deg, r = _degrees(case), case["rank"]
        out["x"] = normal(n, sum(c * i for c, i, _ in deg))
        out["shared"] = [normal(i, o, scale=i ** -0.5) for _, i, o in deg]
        out["down"] = [normal(g, i, r, scale=i ** -0.5) for _, i, _ in deg]
        out["up"] = [normal(g, r, o, scale=0.5 * r ** -0.5) for _, _, o in deg]
        if case["op"] == "adapter_train":
            out["grad_y"] = normal(n, sum(c * o for c, _, o in deg))
    return out


def prepare(case, seed):
    state = _arrays(case, seed)
    state["case"] = case
    if own:
        from symmetrix_b200 import AdapterLinear, RowRouting
        if case["op"] != "route":
            state["routing"] = RowRouting(state["ids"], case["groups"])
        if case["op"].startswith("adapter"):
            state["layer"] = AdapterLinear(state["shared"], state["down"], state["up"])
    elif case["op"] == "route_grad":
        state["plan"] = _plain_plan(state["ids"], case["groups"])
    return state


# ------------------------------------------------------------------------------------------- plain forms

def _plain_plan(ids, groups):
    """order: pairs (atom, slot) by group, empty slots last; position: where each pair went; offsets of the groups."""
    flat = ids.reshape(-1)
    key = torch.where(flat < 0, torch.full_like(flat, groups), flat).long()
    order = torch.sort(key, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(groups + 1, dtype=torch.long, device=order.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:groups].cumsum(0)])
    return order, position.reshape(ids.shape), offsets


def _plain_route(st):
    ids, s = st["ids"], st["ids"].shape[1]
    order, position, offsets = _plain_plan(ids, st["case"]["groups"])
    live = (ids >= 0)
    rows = st["x"][order // s] * (ids.reshape(-1)[order] >= 0).to(st["x"].dtype)[:, None]
    y = st["base"].clone()
    for q in range(s):
        y += (st["weights"][:, q] * live[:, q])[:, None] * st["rows"][position[:, q]]
    return {"order": order.to(torch.int32), "offsets": offsets.to(torch.int32), "rows": rows, "y": y}


def _plain_route_grad(st):
    ids, s = st["ids"], st["ids"].shape[1]
    order, position, _ = st["plan"]
    live = (ids >= 0).to(st["grad_y"].dtype)
    grad_x = torch.zeros_like(st["grad_y"])
    grad_w = torch.zeros_like(st["weights"])
    for q in range(s):
        grad_x += live[:, q, None] * st["grad_rows"][position[:, q]]
        grad_w[:, q] = live[:, q] * (st["grad_y"] * st["rows"][position[:, q]]).sum(1)
    grad_rows = (st["weights"] * live).reshape(-1)[order][:, None] * st["grad_y"][order // s]
    return {"grad_x": grad_x, "grad_rows": grad_rows, "grad_weights": grad_w}


def _plain_linear(case, x, ids, weights, shared, first, second, grad_y=None):
    """All adapters' products of every row, of which each row's own are taken. `first` and `second` are [groups, in, rank] and
    [groups, rank, out] of each degree. With `grad_y` also the gradients."""
    n, s, g, r = case["atoms"], case["slots"], case["groups"], case["rank"]
    live = (ids >= 0).to(x.dtype) * weights
    pick = ids.clamp(min=0).long()
    # mix[n, g]: what adapter g counts for in atom n
    mix = torch.zeros(n, g, dtype=x.dtype, device=x.device).scatter_add_(1, pick, live)
    ys, gxs, g_first, g_second = [], [], [], []
    g_mix = torch.zeros_like(mix)
    at_x = at_y = 0
    for (c, i, o), w, a, b in zip(_degrees(case), shared, first, second):
        xd = x[:, at_x:at_x + c * i].reshape(n * c, i)
        at_x += c * i
        hidden = (xd @ a.permute(1, 0, 2).reshape(i, g * r)).reshape(n, c, g, r)
        scaled = (hidden * mix[:, None, :, None]).reshape(n * c, g * r)
        ys.append((xd @ w + scaled @ b.reshape(g * r, o)).reshape(n, c * o))
        if grad_y is None:
            continue
        gy = grad_y[:, at_y:at_y + c * o].reshape(n * c, o)
        at_y += c * o
        back = (gy @ b.reshape(g * r, o).T).reshape(n, c, g, r)
        g_mix += (hidden * back).sum(dim=(1, 3))
        back = (back * mix[:, None, :, None]).reshape(n * c, g * r)
        gxs.append((gy @ w.T + back @ a.permute(0, 2, 1).reshape(g * r, i)).reshape(n, c * i))
        g_first.append((xd.T @ back).reshape(i, g, r).permute(1, 0, 2).contiguous())
        g_second.append((scaled.T @ gy).reshape(g, r, o))
    y = torch.cat(ys, dim=1)
    if grad_y is None:
        return {"y": y}
    return {"y": y, "grad_x": torch.cat(gxs, dim=1), "grad_down": g_first, "grad_up": g_second,
            "grad_weights": torch.gather(g_mix, 1, pick) * (ids >= 0).to(x.dtype)}


# ------------------------------------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "route":
            return _plain_route(state)
        if case["op"] == "route_grad":
            return _plain_route_grad(state)
        return _plain_linear(case, state["x"], state["ids"], state["weights"], state["shared"], state["down"], state["up"], state.get("grad_y"))
    from symmetrix_b200 import RowRouting
    if case["op"] == "route":
        routing = RowRouting(state["ids"], case["groups"])
        rows = routing.dispatch(state["x"])
        y = routing.combine(state["rows"], state["weights"], state["base"])
        return {"order": routing.order, "offsets": routing.offsets, "rows": rows, "y": y}
    routing = state["routing"]
    if case["op"] == "route_grad":
        grad_x = routing.dispatch_backward(state["grad_rows"])
        grad_rows, grad_weights = routing.combine_backward(state["grad_y"], state["rows"], state["weights"])
        return {"grad_x": grad_x, "grad_rows": grad_rows, "grad_weights": grad_weights}
    layer = state["layer"]
    if case["op"] == "adapter":
        return {"y": layer.forward(state["x"], routing, state["weights"])}
    layer.set_adapters(state["down"], state["up"])
    y, hidden = layer.forward(state["x"], routing, state["weights"], keep_hidden=True)
    grads = layer.backward(state["x"], state["grad_y"], routing, state["weights"], hidden=hidden)
    return {"y": y, "grad_x": grads.x, "grad_down": list(grads.down), "grad_up": list(grads.up), "grad_weights": grads.weights}


# ------------------------------------------------------------------------------------------- definition in 64 bits

def exact(case, seed):
    """The same outputs from the definitions, group by group and slot by slot, in 64 bits."""
    data = _arrays(case, seed)
    ids = data["ids"].cpu().numpy()
    n, s = ids.shape
    g = case["groups"]
    f64 = {k: v.double() for k, v in data.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    members = [np.flatnonzero(ids.reshape(-1) == q) for q in range(g)]       # pairs of every group, in pair order
    empty = np.flatnonzero(ids.reshape(-1) < 0)

    def pairs(p):
        p = torch.as_tensor(p, device="cuda")
        return p // s, p % s

    if case["op"].startswith("route"):
        order = np.concatenate(members + [empty])
        starts = np.concatenate([[0], np.cumsum([m.size for m in members])])
        atoms, slots = pairs(order[:starts[-1]])
        last = int(starts[-1])
        if case["op"] == "route":
            rows = torch.zeros(n * s, case["width"], dtype=torch.float64, device="cuda")
            rows[:last] = f64["x"][atoms]
            y = f64["base"].clone()
            y.index_add_(0, atoms, f64["weights"][atoms, slots][:, None] * f64["rows"][:last])
            return {"order": torch.as_tensor(order.astype(np.int32), device="cuda"), "offsets": torch.as_tensor(starts.astype(np.int32), device="cuda"),
                    "rows": rows, "y": y}
        grad_x = torch.zeros(n, case["width"], dtype=torch.float64, device="cuda").index_add_(0, atoms, f64["grad_rows"][:last])
        grad_rows = torch.zeros(n * s, case["width"], dtype=torch.float64, device="cuda")
        grad_rows[:last] = f64["weights"][atoms, slots][:, None] * f64["grad_y"][atoms]
        grad_w = torch.zeros(n, s, dtype=torch.float64, device="cuda")
        grad_w[atoms, slots] = torch.einsum("pw,pw->p", f64["grad_y"][atoms], f64["rows"][:last])
        return {"grad_x": grad_x, "grad_rows": grad_rows, "grad_weights": grad_w}

    train = case["op"] == "adapter_train"
    ys, gxs, g_down, g_up = [], [], [], []
    grad_w = torch.zeros(n, s, dtype=torch.float64, device="cuda")
    at_x = at_y = 0
    for (c, i, o), w, a, b in zip(_degrees(case), data["shared"], data["down"], data["up"]):
        w, a, b = w.double(), a.double(), b.double()
        xd = f64["x"][:, at_x:at_x + c * i].reshape(n, c, i)
        y = torch.einsum("nci,io->nco", xd, w)
        gy = f64["grad_y"][:, at_y:at_y + c * o].reshape(n, c, o) if train else None
        gx = torch.einsum("nco,io->nci", gy, w) if train else None
        ga, gb = torch.zeros_like(a), torch.zeros_like(b)
        for q in range(g):
            if members[q].size == 0:
                continue
            atoms, slots = pairs(members[q])
            scale = f64["weights"][atoms, slots][:, None, None]
            hidden = xd[atoms] @ a[q]
            y.index_add_(0, atoms, scale * (hidden @ b[q]))
            if train:
                back = gy[atoms] @ b[q].T
                gx.index_add_(0, atoms, scale * (back @ a[q].T))
                ga[q] = torch.einsum("pci,pcr->ir", xd[atoms], scale * back)
                gb[q] = torch.einsum("pcr,pco->ro", scale * hidden, gy[atoms])
                grad_w[atoms, slots] += (hidden * back).sum(dim=(1, 2))
        at_x += c * i
        at_y += c * o
        ys.append(y.reshape(n, c * o))
        if train:
            gxs.append(gx.reshape(n, c * i))
            g_down.append(ga)
            g_up.append(gb)
    if not train:
        return {"y": torch.cat(ys, dim=1)}
    return {"y": torch.cat(ys, dim=1), "grad_x": torch.cat(gxs, dim=1), "grad_down": g_down, "grad_up": g_up, "grad_weights": grad_w}
