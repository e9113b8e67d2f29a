"""Rows routed to groups and back, and linears with low-rank adapters, against plain definitions in 64 bits on the host.

Tolerances are elementwise bounds: a sum of n products computed in a type with unit roundoff u is off by at most n u sum |terms| (first order),
whatever the order of its additions. float32 products on the tensor cores are made of operands x = hi + lo + e with hi and lo rounded to
11 bits (|e| <= 2^-22 |x|) and leave out lo lo (2^-22): 3 x 2^-22 a product, and their sums may be cut instead of rounded: one step,
2^-23, an addition. A value that passes through a second product carries the first one's error along. EPS is that step, twice the unit
roundoff, also in float64, where it covers the reference's own roundings; 24 further steps cover the splits of two products in a row
(2 x 3 x 2^-22 = 12 x 2^-23) and the roundings of weights and inputs.
"""
import itertools

import numpy as np
import pytest
import torch

from symmetrix_b200 import AdapterLinear, RowRouting

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.float64: 2.0 ** -52}


def host(t):
    return t.detach().double().cpu().numpy()


def make_ids(rng, n, slots, groups, kind="random"):
    if kind == "empty":
        return torch.full((n, slots), -1, dtype=torch.int32, device="cuda")
    ids = rng.integers(0, groups, size=(n, slots))
    if kind == "random":
        ids[rng.random((n, slots)) < 0.15] = -1
    elif kind == "skewed":                       # nearly all in one group, a few elsewhere
        ids = np.where(rng.random((n, slots)) < 0.97, groups // 2, ids)
    elif kind == "outside":                      # anything outside the groups is an empty slot
        ids[rng.random((n, slots)) < 0.3] = groups
        ids[rng.random((n, slots)) < 0.3] = 2 ** 31 - 1
        ids[rng.random((n, slots)) < 0.3] = -(2 ** 31)
    return torch.as_tensor(ids.astype(np.int32)).cuda()


def plan_of(ids, groups):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    key = np.where((flat < 0) | (flat >= groups), groups, flat)
    order = np.argsort(key, kind="stable")
    position = np.empty_like(order)
    position[order] = np.arange(order.size)
    position[key == groups] = -1
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=groups + 1)[:groups])])
    return order, position.reshape(ids.shape), offsets


def same_plan(routing, ids):
    order, position, offsets = plan_of(ids, routing.num_groups)
    np.testing.assert_array_equal(routing.order.cpu().numpy(), order)
    np.testing.assert_array_equal(routing.position.cpu().numpy().reshape(-1), position.reshape(-1))
    np.testing.assert_array_equal(routing.offsets.cpu().numpy(), offsets)
    return order, position, offsets


# ------------------------------------------------------------------------------------------- plan

@pytest.mark.parametrize("n,slots,groups", [
    (0, 1, 1), (0, 2, 7), (1, 1, 1), (1, 64, 1024), (31, 1, 2), (32, 1, 2), (33, 3, 5), (1000, 1, 1), (129, 2, 1024), (4096, 2, 3), (8192, 1, 1000),
    (8193, 1, 1), (4097, 2, 65), (20000, 3, 1024), (70001, 1, 33), (300000, 2, 64),
])
@pytest.mark.parametrize("kind", ["random", "skewed", "outside", "empty"])
def test_plan(n, slots, groups, kind):
    rng = np.random.default_rng(n + slots + groups)
    ids = make_ids(rng, n, slots, groups, kind)
    routing = RowRouting(ids, groups)
    same_plan(routing, ids)
    other = make_ids(rng, n, slots, groups, "random")
    routing.update(other)
    same_plan(routing, other)


def test_plan_of_strided_ids_and_one_dimension():
    ids = make_ids(np.random.default_rng(0), 500, 4, 9)
    routing = RowRouting(ids[:, 1], 9)
    same_plan(routing, ids[:, 1:2])
    same_plan(RowRouting(ids[::3, :2], 9), ids[::3, :2].contiguous())


# ------------------------------------------------------------------------------------------- rows

SIZES = [(1, 1, 1, 1), (1, 1, 1, 4), (5, 3, 2, 7), (37, 2, 100, 33), (64, 1, 3, 512), (100, 5, 8, 130), (257, 9, 4, 36), (3000, 2, 17, 20), (33, 2, 4, 2304)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("n,slots,groups,width", SIZES)
@pytest.mark.parametrize("kind", ["random", "empty", "outside"])
def test_rows(dtype, n, slots, groups, width, kind):
    rng = np.random.default_rng(width)
    gen = torch.Generator("cuda").manual_seed(n)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    ids = make_ids(rng, n, slots, groups, kind)
    routing = RowRouting(ids, groups)
    order, position, offsets = plan_of(ids, groups)
    live = position >= 0
    last = offsets[-1]
    x, base, rows, weights, grad_y = rand(n, width), rand(n, width), rand(n * slots, width), rand(n, slots), rand(n, width)
    rows[last:] = float("nan")                   # behind the last group nothing is read
    weights[torch.as_tensor(~live).cuda()] = float("inf")

    sorted_rows = routing.dispatch(x)
    expect = np.zeros((n * slots, width))
    expect[:last] = host(x)[order[:last] // slots]
    np.testing.assert_array_equal(host(sorted_rows), expect)
    kept = torch.full_like(sorted_rows, 7.0)
    assert routing.dispatch(x, out=kept) is kept
    expect[last:] = 7.0
    np.testing.assert_array_equal(host(kept), expect)

    w, r, gy = np.where(live, host(weights), 0.0), host(rows), host(grad_y)
    gathered = np.where(live[..., None], r[np.where(live, position, 0)], 0.0)
    for use_w, use_b in itertools.product([True, False], repeat=2):
        y = routing.combine(rows, weights if use_w else None, base if use_b else None)
        terms = gathered * (w if use_w else live)[..., None]
        add = host(base) if use_b else 0.0
        bound = (slots + 1) * EPS[dtype] * (np.abs(terms).sum(1) + np.abs(add))
        assert (np.abs(host(y) - terms.sum(1) - add) <= bound).all()
    np.testing.assert_array_equal(host(routing.dispatch_backward(rows)), host(routing.combine(rows)))

    grad_rows, grad_weights = routing.combine_backward(grad_y, rows, weights)
    expect = np.zeros((n * slots, width))
    expect[:last] = (w.reshape(-1)[order[:last]])[:, None] * gy[order[:last] // slots]
    assert (np.abs(host(grad_rows) - expect) <= EPS[dtype] * np.abs(expect)).all()
    terms = gathered * gy[:, None, :]
    assert (np.abs(host(grad_weights) - terms.sum(2)) <= width * EPS[dtype] * np.abs(terms).sum(2)).all()
    ones, none = routing.combine_backward(grad_y)
    assert none is None
    np.testing.assert_array_equal(host(ones)[:last], gy[order[:last] // slots])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_rows_of_any_stride_and_alignment(dtype):
    ids = make_ids(np.random.default_rng(3), 50, 2, 6)
    routing = RowRouting(ids, 6)
    big = torch.randn(50, 100, device="cuda", dtype=dtype)
    rows, w = torch.randn(100, 40, device="cuda", dtype=dtype), torch.rand(50, 2, device="cuda", dtype=dtype)
    for start, step in [(0, 1), (1, 1), (3, 1), (4, 1), (0, 2)]:
        x = big[:, start:start + 40 * step:step]
        plain = x.contiguous()
        assert torch.equal(routing.dispatch(x), routing.dispatch(plain))
        assert torch.equal(routing.combine(rows, w, x), routing.combine(rows, w, plain))
        a, b = routing.combine_backward(x, rows, w), routing.combine_backward(plain, rows, w)
        assert torch.equal(a[0], b[0])
        # rows that start on no 16-byte boundary are walked value by value, so the 40 products add up in another order: each sum is off by
        # at most 40 u sum |products|, so two of them differ by at most 40 EPS sum |products|
        size = routing.combine_backward(plain.abs(), rows.abs(), w)[1]
        assert ((a[1] - b[1]).abs() <= 40 * EPS[dtype] * size).all()
    one = torch.randn(1, 40, device="cuda", dtype=dtype).expand(50, 40)
    assert torch.equal(routing.dispatch(one), routing.dispatch(one.contiguous()))
    view = torch.full((50, 100), 5.0, device="cuda", dtype=dtype)
    routing.combine(rows, w, out=view[:, 7:47])
    assert torch.equal(view[:, 7:47], routing.combine(rows, w))
    assert (view[:, :7] == 5).all() and (view[:, 47:] == 5).all()
    base = big[:, :40].contiguous()
    expect = routing.combine(rows, w, base)
    assert routing.combine(rows, w, base, out=base) is base and torch.equal(base, expect)


def test_row_refusals():
    routing = RowRouting(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 3)
    x, rows = torch.randn(4, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    for bad in (lambda: RowRouting(torch.zeros(4, dtype=torch.int64, device="cuda"), 3),
                lambda: RowRouting(torch.zeros(4, 2, 2, dtype=torch.int32, device="cuda"), 3),
                lambda: RowRouting(torch.zeros(4, dtype=torch.int32, device="cuda"), 0),
                lambda: RowRouting(torch.zeros(4, dtype=torch.int32, device="cuda"), 1025),
                lambda: RowRouting(torch.zeros(4, 65, dtype=torch.int32, device="cuda"), 3),
                lambda: routing.update(torch.zeros(5, 2, dtype=torch.int32, device="cuda")),
                lambda: routing.update(torch.zeros(8, dtype=torch.int32, device="cuda")),
                lambda: routing.dispatch(x.half()), lambda: routing.dispatch(x[:3]), lambda: routing.dispatch(x.cpu()), lambda: routing.dispatch(x[0]),
                lambda: routing.dispatch(x, out=torch.empty(8, 9, device="cuda")), lambda: routing.dispatch(x, out=torch.empty(8, 16, device="cuda")[:, ::2]),
                lambda: routing.dispatch(x, out=torch.empty(8, 8, device="cuda", dtype=torch.float64)),
                lambda: routing.combine(rows[:7]), lambda: routing.combine(rows, torch.ones(4, 3, device="cuda")),
                lambda: routing.combine(rows, torch.ones(4, 2, device="cuda").double()), lambda: routing.combine(rows, base=x[:, :4]),
                lambda: routing.combine(rows, out=rows[:4]), lambda: routing.combine(rows, out=x[:1].expand(4, 8)),
                lambda: routing.combine(rows, base=x[:, :], out=torch.as_strided(x, (4, 8), (8, 1), 0).view(-1)[0:32].view(4, 8).t()),
                lambda: routing.combine_backward(x, rows[:, :4]),
                lambda: routing.dispatch(x.clone().requires_grad_())):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        routing.dispatch(x.clone().requires_grad_())


# ------------------------------------------------------------------------------------------- linears

class Case:
    def __init__(self, dtype, components, in_channels, out_channels, n, slots, groups, rank, kind="random", shared=True, seed=0, weights=True):
        rng = np.random.default_rng(seed + n + rank)
        gen = torch.Generator("cuda").manual_seed(seed + n)
        rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
        self.dtype, self.components, self.n, self.slots, self.groups, self.rank = dtype, components, n, slots, groups, rank
        self.in_channels, self.out_channels = in_channels, out_channels
        self.ids = make_ids(rng, n, slots, groups, kind)
        self.weights = rand(n, slots) if weights else None
        self.shared = [rand(i, o) * i ** -0.5 for i, o in zip(in_channels, out_channels)] if shared else None
        self.down = [rand(groups, i, rank) * i ** -0.5 for i in in_channels]
        self.up = [rand(groups, rank, o) * rank ** -0.5 for o in out_channels]
        self.x = rand(n, sum(c * i for c, i in zip(components, in_channels)))
        self.gy = rand(n, sum(c * o for c, o in zip(components, out_channels)))

    def layer(self):
        return AdapterLinear(self.shared, self.down, self.up, self.components)

    def reference(self, absolute=False):
        """Outputs and gradients in 64 bits pair by group; with `absolute` of the operands' absolute values: what the bounds are made of."""
        f = (lambda t: np.abs(host(t))) if absolute else host
        ids = self.ids.cpu().numpy()
        live = (ids >= 0) & (ids < self.groups)
        w_all = np.where(live, f(self.weights) if self.weights is not None else 1.0, 0.0)
        x, gy = f(self.x), f(self.gy)
        ys, gxs, gds, gus = [], [], [], []
        gw = np.zeros(ids.shape)
        at_x = at_y = 0
        for q, (c, i, o) in enumerate(zip(self.components, self.in_channels, self.out_channels)):
            xd, gd = x[:, at_x:at_x + c * i].reshape(-1, c, i), gy[:, at_y:at_y + c * o].reshape(-1, c, o)
            at_x, at_y = at_x + c * i, at_y + c * o
            w = f(self.shared[q]) if self.shared is not None else np.zeros((i, o))
            a, b = f(self.down[q]), f(self.up[q])
            y, gx, ga, gb = xd @ w, gd @ w.T, np.zeros_like(a), np.zeros_like(b)
            for s in range(self.slots):
                for g in range(self.groups):
                    sel = np.flatnonzero(live[:, s] & (ids[:, s] == g))
                    if sel.size == 0:
                        continue
                    ws = w_all[sel, s][:, None, None]
                    t, h = xd[sel] @ a[g], gd[sel] @ b[g].T
                    y[sel] += ws * (t @ b[g])
                    gx[sel] += ws * (h @ a[g].T)
                    ga[g] += np.einsum("pci,pcr->ir", xd[sel], ws * h)
                    gb[g] += np.einsum("pcr,pco->ro", ws * t, gd[sel])
                    gw[sel, s] += (t * h).sum((1, 2))
            ys.append(y.reshape(self.n, -1)); gxs.append(gx.reshape(self.n, -1)); gds.append(ga); gus.append(gb)
        return np.concatenate(ys, 1), np.concatenate(gxs, 1), gds, gus, gw

    def check(self, y, grads):
        ref, mag = self.reference(), self.reference(absolute=True)
        eps, most_i, most_o = EPS[self.dtype], max(self.in_channels), max(self.out_channels)
        terms = self.n * self.slots * max(self.components)
        steps = {"y": most_i + self.rank + self.slots + 24, "x": most_o + self.rank + self.slots + 24,
                 "down": terms + most_o + 24, "up": terms + most_i + 24, "weights": sum(self.components) * self.rank + most_i + most_o + 24}

        def close(name, got, want, size):
            assert got.shape == want.shape, name
            excess = np.abs(got - want) - steps[name] * eps * size
            assert excess.size == 0 or excess.max() <= 0, f"{name}: {np.abs(got - want).max()} off, {excess.max()} beyond the bound"
        if y is not None:
            close("y", host(y), ref[0], mag[0])
        if grads is None:
            return
        if grads.x is not None:
            close("x", host(grads.x), ref[1], mag[1])
        if grads.down is not None:
            for q in range(len(self.components)):
                close("down", host(grads.down[q]), ref[2][q], mag[2][q])
                close("up", host(grads.up[q]), ref[3][q], mag[3][q])
        if grads.weights is not None:
            close("weights", host(grads.weights), ref[4], mag[4])


def everything(case):
    layer, routing = case.layer(), RowRouting(case.ids, case.groups)
    y, hidden = layer.forward(case.x, routing, case.weights, keep_hidden=True)
    grads = layer.backward(case.x, case.gy, routing, case.weights, hidden=hidden)
    return layer, routing, y, grads


SHAPES = [
    # components, in, out, atoms, slots, adapters, rank
    ([1], [1], [1], 1, 1, 1, 1),
    ([1], [8], [8], 5, 1, 2, 3),
    ([1, 3], [128, 128], [128, 128], 18, 1, 2, 4),
    ([1, 3, 5], [64, 64, 64], [64, 64, 64], 41, 1, 3, 16),
    ([1, 3], [33, 33], [33, 33], 65, 1, 4, 5),
    ([1, 3, 5, 7], [256, 384, 384, 256], [128, 128, 128, 128], 40, 1, 5, 8),
    ([1, 3, 5, 7], [10, 15, 15, 10], [5, 5, 5, 5], 19, 2, 3, 2),
    ([1], [130], [70], 129, 1, 2, 64),
    ([1], [70], [130], 300, 1, 1, 33),
    ([2], [257], [255], 63, 1, 7, 17),
    ([1, 3], [128, 128], [128, 128], 700, 2, 9, 16),
    ([1, 3, 5], [96, 96, 96], [96, 96, 96], 111, 3, 4, 24),
    ([1, 3], [128, 128], [128, 128], 2500, 1, 40, 32),
    ([1], [256], [256], 513, 1, 1000, 16),
    ([9], [16], [16], 1000, 1, 3, 4),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(str(v).replace(" ", "") for v in s))
def test_linear(dtype, shape):
    case = Case(dtype, *shape)
    _, _, y, grads = everything(case)
    case.check(y, grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("slots", [1, 2])
@pytest.mark.parametrize("kind", ["empty", "skewed", "outside"])
@pytest.mark.parametrize("shared,weights", [(True, True), (False, False)])
def test_linear_masks(dtype, slots, kind, shared, weights):
    """No adapter at all, nearly one adapter, ids that are no adapters; without shared weights and without mixing weights."""
    case = Case(dtype, [1, 3], [72, 40], [40, 56], 150, slots, 6, 7, kind=kind, shared=shared, weights=weights)
    if weights:
        outside = ((case.ids < 0) | (case.ids >= 6))
        case.weights[outside] = float("nan")
    _, _, y, grads = everything(case)
    if weights:
        case.weights[outside] = 0.0
        assert (grads.weights[outside] == 0).all()
    case.check(y, grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("slots", [1, 2])
def test_linear_without_rows(dtype, slots):
    case = Case(dtype, [1, 3], [16, 16], [16, 16], 0, slots, 3, 4)
    _, _, y, grads = everything(case)
    assert y.shape == (0, 64) and grads.x.shape == (0, 64) and grads.weights.shape == (0, slots)
    assert all((g == 0).all() for g in (*grads.down, *grads.up))


MANY_SLOTS = [
    # plans of one CTA and of several, rows that are aligned and not, more than one block of columns, the most slots
    ([1], [221], [221], 6000, 2, 1, 38),
    ([1, 3], [44, 44], [44, 44], 3100, 3, 40, 14),
    ([1, 3], [128, 128], [192, 192], 4500, 2, 5, 24),
    ([1], [72], [264], 70, 64, 9, 4),
    ([2], [64], [64], 200, 64, 3, 64),
    ([1], [19], [3], 1, 64, 2, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("shape", MANY_SLOTS, ids=lambda s: "x".join(str(v).replace(" ", "") for v in s))
@pytest.mark.parametrize("kind", ["random", "same", "outside"])
def test_linear_with_many_slots(dtype, shape, kind):
    """Every slot adds to what the slots before it left; "same" gives a row's slots one adapter, which counts as often as it is listed."""
    for shared in (True, False):
        case = Case(dtype, *shape, kind="random" if kind == "same" else kind, shared=shared)
        if kind == "same":
            case.ids = case.ids[:, :1].expand(-1, case.slots).contiguous()
        _, _, y, grads = everything(case)
        case.check(y, grads)
        _, _, again, other = everything(case)
        assert torch.equal(y, again) and torch.equal(grads.x, other.x) and torch.equal(grads.weights, other.weights)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_unused_adapters_and_other_requests_do_not_matter(dtype):
    """Adapters that nobody names may hold anything; an atom's result does not depend on the batch it is in beyond its roundings."""
    case = Case(dtype, [1, 3], [64, 64], [64, 64], 90, 1, 5, 8)
    case.ids[case.ids == 3] = 1
    for m in (*case.down, *case.up):
        m[3] = float("nan")
    _, routing, y, grads = everything(case)
    assert torch.isfinite(y).all() and torch.isfinite(grads.x).all() and all((g[3] == 0).all() for g in (*grads.down, *grads.up))
    case2 = Case(dtype, [1, 3], [64, 64], [64, 64], 90, 1, 5, 8)
    case2.ids = case.ids.clone()
    poisoned = case2.x.clone()
    poisoned[case2.ids[:, 0] == 2] = float("nan")
    layer = case2.layer()
    out = layer.forward(poisoned, routing, case2.weights)
    clean = layer.forward(case2.x, routing, case2.weights)
    keep = case2.ids[:, 0] != 2
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[~keep]).all()


def test_gradients_against_differences():
    """float64: every gradient against central differences of a random linear functional of the output. The function is linear in x and in
    the weights and bilinear in the two adapter matrices, so central differences have no error but rounding: with a step of 2^-10,
    about 2^-52 x 2^10 x the size of the functional's terms (here a few thousand of order one)."""
    for slots in (1, 2):
        case = Case(torch.float64, [1, 3], [12, 9], [10, 11], 14, slots, 3, 4)
        layer, routing, _, grads = everything(case)
        value = lambda: float((layer.forward(case.x, routing, case.weights) * case.gy).sum())  # noqa: E731
        rng = np.random.default_rng(1)
        step = 2.0 ** -10
        for tensor, grad in [(case.x, grads.x), (case.weights, grads.weights), *zip(case.down, grads.down), *zip(case.up, grads.up)]:
            for _ in range(6):
                at = tuple(int(rng.integers(0, n)) for n in tensor.shape)
                old = tensor[at].item()
                diff = []
                for sign in (1, -1):
                    tensor[at] = old + sign * step
                    layer.set_adapters(case.down, case.up)
                    diff.append(value())
                tensor[at] = old
                layer.set_adapters(case.down, case.up)
                assert abs((diff[0] - diff[1]) / (2 * step) - grad[at].item()) <= 1e-8


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("slots", [1, 2])
def test_same_bits_and_parts(dtype, slots):
    """Repeated calls, with and without the kept products, all gradients at once or one kind alone."""
    case = Case(dtype, [1, 3], [128, 128], [128, 128], 1500, slots, 6, 16)
    layer, routing, y, grads = everything(case)
    _, _, y2, grads2 = everything(case)
    assert torch.equal(y, y2) and torch.equal(grads.x, grads2.x) and torch.equal(grads.weights, grads2.weights)
    assert all(torch.equal(a, b) for a, b in zip((*grads.down, *grads.up), (*grads2.down, *grads2.up)))
    again = layer.backward(case.x, case.gy, routing, case.weights)
    case.check(None, again)
    only = layer.backward(case.x, case.gy, routing, case.weights, want_adapters=False, want_weights=False)
    assert torch.equal(only.x, grads.x) and only.down is None and only.up is None and only.weights is None
    only = layer.backward(case.x, case.gy, routing, case.weights, want_x=False, want_weights=False)
    assert only.x is None
    case.check(None, only)
    only = layer.backward(case.x, case.gy, routing, case.weights, want_x=False, want_adapters=False)
    assert only.down is None
    case.check(None, only)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("slots", [1, 2])
def test_strided_rows(dtype, slots):
    case = Case(dtype, [1, 3], [40, 24], [24, 40], 77, slots, 4, 6)
    layer, routing, y, grads = everything(case)
    wide_x, wide_y = torch.zeros(77, case.x.shape[1] + 9, device="cuda", dtype=dtype), torch.full((77, case.gy.shape[1] + 5), 3.0, device="cuda", dtype=dtype)
    for start in (0, 1, 4):
        x = wide_x[:, start:start + case.x.shape[1]]
        x.copy_(case.x)
        out = layer.forward(x, routing, case.weights, out=wide_y[:, 1:1 + case.gy.shape[1]])
        case.check(out, None)
        assert (wide_y[:, 0] == 3).all() and (wide_y[:, 1 + case.gy.shape[1]:] == 3).all()
        gy = wide_y[:, 1:1 + case.gy.shape[1]]
        gy.copy_(case.gy)
        case.check(None, layer.backward(x, gy, routing, case.weights))
        wide_y.fill_(3.0)


def test_matrices_are_those_of_the_last_set_call():
    case = Case(torch.float32, [1, 3], [64, 64], [64, 64], 60, 1, 3, 8)
    layer, routing, y, _ = everything(case)
    new = Case(torch.float32, [1, 3], [64, 64], [64, 64], 60, 1, 3, 8, seed=5)
    kept = [m.clone() for m in case.down]
    for m in case.down:
        m.mul_(-3.0)                              # in place: not seen before the next set call
    assert torch.equal(layer.forward(case.x, routing, case.weights), y)
    for m, k in zip(case.down, kept):
        m.copy_(k)
    layer.set_adapters(new.down, new.up)
    layer.set_shared(new.shared)
    new.x, new.gy, new.ids, new.weights = case.x, case.gy, case.ids, case.weights
    new.check(layer.forward(new.x, routing, new.weights), layer.backward(new.x, new.gy, routing, new.weights))


def test_linear_refusals():
    case = Case(torch.float32, [1, 3], [16, 16], [16, 16], 12, 1, 3, 4)
    layer, routing = case.layer(), RowRouting(case.ids, 3)
    x, gy = case.x, case.gy
    many = RowRouting(case.ids, 4)
    for bad in (lambda: AdapterLinear(case.shared, case.down, case.up[:1]), lambda: AdapterLinear(case.shared[:1], case.down, case.up),
                lambda: AdapterLinear(case.shared, [d.double() for d in case.down], case.up),
                lambda: AdapterLinear(case.shared, [d[:2] for d in case.down], case.up),
                lambda: AdapterLinear(case.shared, [d.repeat(1, 1, 17) for d in case.down], [u.repeat(1, 17, 1) for u in case.up]),
                lambda: AdapterLinear(case.shared, case.down, case.up, components=[1]), lambda: AdapterLinear(case.shared, case.down, case.up, components=[1, 0]),
                lambda: AdapterLinear(None, case.down, case.up).set_shared(case.shared), lambda: layer.set_adapters(case.down[:1], case.up),
                lambda: layer.set_adapters([d[:, :8] for d in case.down], case.up), lambda: layer.set_shared([w.t()[:8] for w in case.shared]),
                lambda: layer.forward(x[:, :60], routing), lambda: layer.forward(x[:11], routing), lambda: layer.forward(x.double(), routing),
                lambda: layer.forward(x, many), lambda: layer.forward(x, case.ids), lambda: layer.forward(x, routing, torch.ones(12, 2, device="cuda")),
                lambda: layer.forward(x, routing, out=x), lambda: layer.forward(x, routing, out=torch.empty(12, 128, device="cuda")[:, ::2]),
                lambda: layer.forward(x.clone().requires_grad_(), routing), lambda: layer.backward(x, gy[:, :3], routing),
                lambda: layer.backward(x, gy, routing, hidden=torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


def test_offsets_beyond_32_bits():
    """Arrays of more than 2^32 bytes and 2^31 values: rows at both ends against their definition."""
    n, width = 270_001, 8192
    ids = (torch.arange(n, device="cuda", dtype=torch.int32) * 7) % 5
    ids[::11] = -1
    routing = RowRouting(ids, 5)
    order, position, offsets = plan_of(ids[:, None], 5)
    x = torch.randn(n, width, device="cuda")
    rows = routing.dispatch(x)
    probe = [0, 1, n // 2, n - 2, n - 1]
    for r in probe:
        p = int(position[r, 0])
        if p >= 0:
            assert torch.equal(rows[p], x[r])
    assert (rows[int(offsets[-1]):] == 0).all()
    y = routing.combine(rows, base=x)
    grad_rows, grad_weights = routing.combine_backward(x, rows)
    for r in probe:
        assert torch.equal(y[r], 2 * x[r] if position[r, 0] >= 0 else x[r])
        if position[r, 0] >= 0:
            assert torch.equal(grad_rows[int(position[r, 0])], x[r])
            exact = (x[r].double() ** 2).sum().item()
            assert abs(grad_weights[r, 0].item() - exact) <= width * 2.0 ** -23 * exact
    del x, rows, y, grad_rows
    n = 2 ** 31 // 128 + 5
    for dtype in (torch.float32, torch.float64):
        gen = torch.Generator("cuda").manual_seed(1)
        rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
        ids = torch.arange(n, device="cuda", dtype=torch.int32) % 3
        shared, down, up = rand(128, 32), rand(3, 128, 4) / 11, rand(3, 4, 32)
        x = rand(n, 128)
        y = AdapterLinear([shared], [down], [up]).forward(x, RowRouting(ids, 3))
        for r in (0, n // 2, n - 1):
            g = int(ids[r])
            v, w, a, b = host(x[r]), host(shared), host(down[g]), host(up[g])
            size = np.abs(v) @ np.abs(w) + np.abs(v) @ np.abs(a) @ np.abs(b)
            assert (np.abs(host(y[r]) - v @ w - v @ a @ b) <= (128 + 4 + 24) * EPS[dtype] * size).all()
        del x, y


# ------------------------------------------------------------------------------------------- used together

@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_routing_and_linears_together(dtype):
    """Dispatch, one linear without shared weights on the sorted rows, combine: the mixture that the linear makes itself; and the way back."""
    case = Case(dtype, [1, 3], [48, 48], [32, 32], 200, 2, 5, 6)
    layer, routing, y, grads = everything(case)
    order, _, offsets = plan_of(case.ids, 5)
    groups = np.full(400, -1, dtype=np.int32)
    groups[:offsets[-1]] = np.repeat(np.arange(5), np.diff(offsets))
    inner = RowRouting(torch.as_tensor(groups).cuda(), 5)
    experts = AdapterLinear(None, case.down, case.up, case.components)
    base = AdapterLinear(case.shared, case.down, case.up, case.components).forward(case.x, RowRouting(torch.full_like(case.ids, -1), 5))
    rows = routing.dispatch(case.x)
    products = experts.forward(rows, inner)
    case.check(routing.combine(products, case.weights, base), None)
    grad_products, grad_weights = routing.combine_backward(case.gy, products, case.weights)
    g = experts.backward(rows, grad_products, inner)
    back = AdapterLinear(case.shared, case.down, case.up, case.components).backward(case.x, case.gy, RowRouting(torch.full_like(case.ids, -1), 5))
    together = grads._replace(x=routing.combine(g.x, base=back.x), down=g.down, up=g.up, weights=None)
    case.check(None, together)
    # <gy, products> of a whole row instead of sums over the hidden rows: out_width terms
    ref, mag = case.reference(), case.reference(absolute=True)
    assert (np.abs(host(grad_weights) - ref[4]) <= (case.gy.shape[1] + 48 + 6 + 24) * EPS[dtype] * mag[4]).all()


def test_captured_and_replayed_next_to_eager_calls():
    """A captured plan, forward and backward pass, replayed with other ids and values while the same linear is called eagerly."""
    case = Case(torch.float32, [1, 3], [128, 128], [128, 128], 5000, 2, 6, 16)
    layer, routing, _, _ = everything(case)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    static = {k: getattr(case, k).clone() for k in ("x", "gy", "ids", "weights")}
    with torch.cuda.stream(stream):
        inner = RowRouting(static["ids"], 6)
        layer.forward(static["x"], inner, static["weights"])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            inner.update(static["ids"])
            y, hidden = layer.forward(static["x"], inner, static["weights"], keep_hidden=True)
            grads = layer.backward(static["x"], static["gy"], inner, static["weights"], hidden=hidden)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (1, 2):
        new = Case(torch.float32, [1, 3], [128, 128], [128, 128], 5000, 2, 6, 16, seed=seed)
        for k in static:
            static[k].copy_(getattr(new, k))
        new.shared, new.down, new.up = case.shared, case.down, case.up
        graph.replay()
        eager = layer.forward(case.x, routing, case.weights)
        torch.cuda.synchronize()
        new.check(y, grads)
        case.check(eager, None)


def test_two_streams_at_once():
    """Two streams use one linear and one plan at the same time: outputs, workspaces and kept products are each call's own."""
    case = Case(torch.float32, [1, 3], [128, 128], [128, 128], 4000, 2, 6, 16)
    layer, routing, y, grads = everything(case)
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                out, hidden = layer.forward(case.x, routing, case.weights, keep_hidden=True)
                results.append((out, layer.backward(case.x, case.gy, routing, case.weights, hidden=hidden)))
    torch.cuda.synchronize()
    for out, g in results:
        assert torch.equal(out, y) and torch.equal(g.x, grads.x) and torch.equal(g.weights, grads.weights)
        assert all(torch.equal(a, b) for a, b in zip((*g.down, *g.up), (*grads.down, *grads.up)))
