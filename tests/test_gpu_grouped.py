"""Linears of routed rows against their definition in 64 bits on the host.

Tolerances are elementwise bounds. A sum of n products computed with unit roundoff u is off by at most n u sum |terms| (first order), in whatever order it
is added. float32 products on the tensor cores are made of operands x = hi + lo + e with hi and lo rounded to 11 bits (|e| <= 2^-22 |x|)
and leave out lo lo (2^-22): 3 x 2^-22 = 6 x 2^-23 a product; their sums may be cut instead of rounded: 2^-23 an addition. EPS is that step, twice the
unit roundoff, also in float64, where it covers the reference's own roundings. Three parts of a product and the sums of parts are
further additions of small numbers: 24 steps cover them all.
"""
import itertools
import threading

import numpy as np
import pytest
import torch

from symmetrix_b200 import Embedding, EmbeddingPlan, GroupedLinear, RowRouting, SymmetrixError, clip_gradients

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.float64: 2.0 ** -52}
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.float64])


def host(t):
    return t.detach().double().cpu().numpy()


def ids_of(counts, tail, seed=0):
    """Ids in random order with `counts[g]` rows of group g and `tail` empty ones."""
    flat = np.concatenate([np.full(c, g) for g, c in enumerate(counts)] + [np.full(tail, -1)]).astype(np.int32)
    return torch.as_tensor(np.random.default_rng(seed).permutation(flat)).cuda()


class Case:
    def __init__(self, dtype, counts, comps, ins, outs, tail=3, seed=0):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)
        self.dtype, self.counts, self.comps, self.ins, self.outs = dtype, counts, comps, ins, outs
        self.routing = RowRouting(ids_of(counts, tail, seed), len(counts))
        self.live, self.n = sum(counts), sum(counts) + tail
        self.weights = [self.rand(len(counts), i, o) for i, o in zip(ins, outs)]
        self.layer = GroupedLinear(self.weights, comps)
        self.x, self.gy = self.rand(self.n, self.layer.in_width), self.rand(self.n, self.layer.out_width)

    def blocks(self, a, widths):
        at, out = 0, []
        for c, w in zip(self.comps, widths):
            out.append(a[:, at:at + c * w].reshape(a.shape[0], c, w))
            at += c * w
        return out

    def expect(self, weights=None):
        """y, grad_x, grad_w and for each the sums of the terms' sizes with the numbers of terms."""
        ws = [host(w) for w in (weights or self.weights)]
        x, gy = host(self.x), host(self.gy)
        groups = np.repeat(np.arange(len(self.counts)), self.counts)
        bounds = np.concatenate([[0], np.cumsum(self.counts)])
        y, gx, gw = [], [], []
        for xd, gd, w in zip(self.blocks(x[:self.live], self.ins), self.blocks(gy[:self.live], self.outs), ws):
            both = []
            for f in (lambda v: v, np.abs):
                a = np.zeros(gd.shape), np.zeros(xd.shape), np.zeros(w.shape)
                for g in range(len(self.counts)):
                    s = slice(bounds[g], bounds[g + 1])
                    a[0][s] = f(xd[s]) @ f(w[g])
                    a[1][s] = f(gd[s]) @ f(w[g]).T
                    a[2][g] = np.einsum("pci,pco->io", f(xd[s]), f(gd[s]))
                both.append(a)
            eps = EPS[self.dtype]
            rows = np.array(self.counts) * xd.shape[1]
            y.append((both[0][0], both[1][0] * eps * (w.shape[1] + 24)))
            gx.append((both[0][1], both[1][1] * eps * (w.shape[2] + 24)))
            gw.append((both[0][2], both[1][2] * eps * (rows[:, None, None] + 24)))
        assert groups.size == self.live
        return y, gx, gw

    def check_rows(self, got, expect, widths, tail=0.0):
        got = host(got)
        for a, (want, tol) in zip(self.blocks(got[:self.live], widths), expect):
            assert np.all(np.abs(a - want) <= tol), np.max(np.abs(a - want) / (tol + 1e-300))
        np.testing.assert_array_equal(got[self.live:], tail)

    def check(self):
        y, gx, gw = self.expect()
        self.x[self.live:] = float("nan")            # behind the last group nothing is read
        self.gy[self.live:] = float("inf")
        self.check_rows(self.layer.forward(self.x, self.routing), y, self.outs)
        kept = torch.full((self.n, self.layer.out_width), 7.0, device="cuda", dtype=self.dtype)
        assert self.layer.forward(self.x, self.routing, out=kept) is kept
        self.check_rows(kept, y, self.outs, tail=7.0)
        grads = self.layer.backward(self.x, self.gy, self.routing)
        self.check_rows(grads.x, gx, self.ins)
        for a, (want, tol) in zip(grads.weights, gw):
            assert np.all(np.abs(host(a) - want) <= tol), np.max(np.abs(host(a) - want) / (tol + 1e-300))
        for want_x, want_w in [(True, False), (False, True), (False, False)]:
            part = self.layer.backward(self.x if want_w else None, self.gy, self.routing, want_x=want_x, want_weights=want_w)
            assert (part.x is None) == (not want_x) and (part.weights is None) == (not want_w)
            if want_x:
                assert torch.equal(part.x, grads.x)
            if want_w:
                assert all(torch.equal(a, b) for a, b in zip(part.weights, grads.weights))
        self.layer.check()


SHAPES = [
    ([1], [1], [1], [1]), ([1], [1], [3], [5]), ([2, 0, 1], [1, 3], [8, 8], [8, 4]), ([0, 0, 7, 0], [1], [33], [65]), ([0, 0], [1], [16], [16]),
    ([127, 128, 129], [1], [32], [128]), ([64, 0, 65, 63], [3], [64], [64]), ([5, 300, 1, 44], [1, 3], [128, 128], [128, 128]),
    ([40, 41], [2, 1, 4], [31, 1, 130], [7, 129, 1]), ([1000], [1], [768], [96]), ([17, 90], [1, 3, 5, 7], [48, 72, 72, 48], [24, 24, 24, 24]),
    ([3] * 70, [1], [20], [36]), ([700, 2, 700], [5], [36], [132]), ([9, 0, 2500], [1, 3], [66, 258], [130, 62]), ([6] * 1024, [1], [4], [4]),
    ([140, 1, 77], [1, 3], [96, 40], [40, 96]), ([300, 20], [1], [72], [136]), ([200], [3, 1], [8, 24], [24, 200]),
    ([3, 0, 9], [40, 1], [36, 64], [64, 33]), ([2, 5], [1000], [7], [64]), ([1, 3], [1024, 33], [8, 64], [64, 8]), ([130], [31, 32], [64, 1], [1, 64]),
]


@BOTH
@pytest.mark.parametrize("counts,comps,ins,outs", SHAPES)
def test_products_and_gradients(dtype, counts, comps, ins, outs):
    Case(dtype, counts, comps, ins, outs, tail=len(counts) % 5).check()


@BOTH
@pytest.mark.parametrize("k,n", list(itertools.product([1, 4, 31, 32, 33, 64, 96, 127, 128, 129, 160, 256, 300], [1, 16, 63, 64, 128, 129, 200, 257])))
def test_sizes_of_matrices(dtype, k, n):
    Case(dtype, [130, 3, 0, 60], [1], [k], [n], tail=1, seed=k + n).check()


@BOTH
def test_no_rows(dtype):
    case = Case(dtype, [0, 0], [1, 3], [4, 5], [6, 7], tail=0)
    assert case.layer.forward(case.x, case.routing).shape == (0, 27)
    grads = case.layer.backward(case.x, case.gy, case.routing)
    assert grads.x.shape == (0, 19) and all(not g.any() and g.shape == w.shape for g, w in zip(grads.weights, case.weights))


@BOTH
def test_only_empty_slots(dtype):
    case = Case(dtype, [0, 0, 0], [1, 3], [40, 5], [6, 70], tail=200)
    case.check()


@BOTH
@pytest.mark.parametrize("shift,extra", [(0, 5), (1, 0), (1, 3), (2, 2), (3, 1)])
def test_rows_of_any_stride_and_start(dtype, shift, extra):
    case = Case(dtype, [70, 1, 150], [1, 3], [36, 64], [64, 30], seed=shift)
    y, gx, gw = case.expect()

    def place(t):
        flat = torch.full((shift + t.shape[0] * (t.shape[1] + extra) + 8,), float("nan"), dtype=dtype, device="cuda")
        view = flat.as_strided(t.shape, (t.shape[1] + extra, 1), shift)
        view.copy_(t)
        return flat, view

    flat_x, x = place(case.x)
    _, gy = place(case.gy)
    flat_y, out = place(torch.zeros_like(case.gy))
    before = flat_y.clone()
    case.layer.forward(x, case.routing, out=out)
    case.check_rows(out, y, case.outs)
    written = torch.zeros_like(flat_y, dtype=torch.bool)
    written.as_strided(out.shape, out.stride(), shift).fill_(True)
    assert torch.equal(flat_y[~written].isnan(), before[~written].isnan())           # nothing between the rows
    grads = case.layer.backward(x, gy, case.routing)
    case.check_rows(grads.x, gx, case.ins)
    for a, (want, tol) in zip(grads.weights, gw):
        assert np.all(np.abs(host(a) - want) <= tol)


@BOTH
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_matrices_of_any_start(dtype, shift):
    case = Case(dtype, [70, 1, 150], [1], [36], [64])
    flat = torch.empty(shift + case.weights[0].numel(), dtype=dtype, device="cuda")
    w = flat[shift:].view_as(case.weights[0])
    w.copy_(case.weights[0])
    case.layer = GroupedLinear([w], [1])
    case.check()
    w.mul_(2.0)                                      # values changed in place count
    case.x, case.gy = torch.nan_to_num(case.x), torch.nan_to_num(case.gy, posinf=0.0)
    case.check_rows(case.layer.forward(case.x, case.routing), case.expect([w])[0], case.outs)


@BOTH
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_stay_in_their_rows_and_groups(dtype, value):
    case = Case(dtype, [130, 20, 50], [1, 3], [70, 36], [40, 130])
    clean_y, clean = case.layer.forward(case.x, case.routing), case.layer.backward(case.x, case.gy, case.routing)
    case.x[131, 69] = value                          # group 1, degree 0
    y = case.layer.forward(case.x, case.routing)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[131, :40] = True
    assert not y[bad].isfinite().any() and torch.equal(y[~bad], clean_y[~bad])
    grads = case.layer.backward(case.x, case.gy, case.routing)
    assert torch.equal(grads.x, clean.x) and torch.equal(grads.weights[1], clean.weights[1])
    bad = torch.zeros_like(grads.weights[0], dtype=torch.bool)
    bad[1, 69] = True
    assert not grads.weights[0][bad].isfinite().any() and torch.equal(grads.weights[0][~bad], clean.weights[0][~bad])
    case.x[131, 69] = 0.0
    case.weights[1][2, 3, 129] = value               # group 2, degree 1
    y = case.layer.forward(case.x, case.routing)
    column = y[150:200, 40:].view(50, 3, 130)[:, :, 129]
    assert not column.isfinite().any() and int((~y.isfinite()).sum()) == 150
    if dtype is torch.float64:
        want = torch.full_like(column, value) * torch.sign(case.x[150:200, 70:].view(50, 3, 36)[:, :, 3])
        assert torch.equal(column.isnan(), want.isnan()) and torch.equal(column.nan_to_num(), want.nan_to_num())


def test_large_and_small_magnitudes():
    # the remainder of a split must neither overflow nor be lost where the type still holds the products
    for size in (1e30, 1e-18):
        case = Case(torch.float32, [40, 100], [1], [50], [70])
        case.x *= size
        case.gy *= 1.0 / size
        case.check()


@BOTH
def test_the_same_call_gives_the_same_bits(dtype):
    case = Case(dtype, [3000, 0, 4100, 17], [1, 3], [128, 72], [64, 130])
    y, grads = case.layer.forward(case.x, case.routing), case.layer.backward(case.x, case.gy, case.routing)
    for _ in range(3):
        assert torch.equal(case.layer.forward(case.x, case.routing), y)
        again = case.layer.backward(case.x, case.gy, case.routing)
        assert torch.equal(again.x, grads.x) and all(torch.equal(a, b) for a, b in zip(again.weights, grads.weights))


@BOTH
def test_many_tiles(dtype):
    # more tiles than CTAs, groups that end inside tiles, several column blocks
    case = Case(dtype, [1, 9000, 127, 5, 12000, 300], [1, 3], [40, 130], [136, 24], seed=5)
    case.check()


@BOTH
def test_gradients_are_differences(dtype):
    # a product is linear in x and in every matrix, so a central difference of any step is its derivative up to roundings: those of two sums of
    # all outputs, which the step divides
    case = Case(dtype, [7, 12], [1, 3], [5, 6], [4, 3], tail=0)
    grads = case.layer.backward(case.x, case.gy, case.routing)

    def loss():
        return float((case.layer.forward(case.x, case.routing).double() * case.gy.double()).sum())

    size = float((case.x.double().abs().sum() * case.gy.double().abs().sum() * max(w.abs().max() for w in case.weights)))
    step = 1.0
    for t, g in [(case.x, grads.x), (case.weights[0], grads.weights[0]), (case.weights[1], grads.weights[1])]:
        for at in (0, t.numel() // 2, t.numel() - 1):
            flat, old = t.view(-1), float(t.view(-1)[at])
            flat[at] = old + step
            up, plus = loss(), float(flat[at])
            flat[at] = old - step
            down, minus = loss(), float(flat[at])
            flat[at] = old
            assert abs((up - down) / (plus - minus) - float(g.reshape(-1)[at])) <= 30 * EPS[dtype] * size / step


@BOTH
def test_other_streams_and_graphs(dtype):
    case = Case(dtype, [300, 0, 170], [1, 3], [64, 40], [48, 56])
    y, grads = case.layer.forward(case.x, case.routing), case.layer.backward(case.x, case.gy, case.routing)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = case.layer.forward(case.x, case.routing)
        others = case.layer.backward(case.x, case.gy, case.routing)
    here = case.layer.forward(case.x, case.routing)
    torch.cuda.synchronize()
    assert torch.equal(other, y) and torch.equal(here, y) and torch.equal(others.x, grads.x)
    x, gy = torch.zeros_like(case.x), torch.zeros_like(case.gy)
    graphs, results = [], []
    for _ in range(2):                               # two graphs of the same layer, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append((case.layer.forward(x, case.routing), case.layer.backward(x, gy, case.routing)))
        graphs.append(graph)
    x.copy_(case.x)
    gy.copy_(case.gy)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for got_y, got in results:
        assert torch.equal(got_y, y) and torch.equal(got.x, grads.x) and all(torch.equal(a, b) for a, b in zip(got.weights, grads.weights))
    case.routing.update(ids_of([170, 130, 170], 3, seed=9))          # another plan in the same memory: the graphs use it
    y2 = case.layer.forward(case.x, case.routing)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], y2) and not torch.equal(y2, y)


@BOTH
def test_threads_share_the_operators(dtype):
    """Four threads, each on a stream of its own, with the same linear, embedding, plan and inputs; the sets of gradients are each thread's own."""
    case = Case(dtype, [300, 0, 170, 5], [1, 3], [64, 40], [48, 56])
    ids = torch.as_tensor(np.random.default_rng(3).integers(-1, 40, (9000, 2)).astype(np.int32)).cuda()
    table, gy = case.rand(40, 64), case.rand(9000, 64)
    embedding, plan = Embedding(table), EmbeddingPlan(ids, 40)

    def step():
        y, grads = case.layer.forward(case.x, case.routing), case.layer.backward(case.x, case.gy, case.routing)
        back = embedding.backward(gy, plan)
        mine = [g.clone() for g in grads.weights] + [back.table.clone()]
        norm = clip_gradients(mine, 0.5)
        return [y, grads.x, *grads.weights, embedding.forward(ids), EmbeddingPlan(ids, 40).order, back.table, back.weights, norm, *mine]

    want = step()
    torch.cuda.synchronize()
    results = [[] for _ in range(4)]

    def work(q):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                results[q].append(step())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(q,)) for q in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    case.layer.check()
    for runs in results:
        assert len(runs) == 5 and all(torch.equal(a, b) for got in runs for a, b in zip(got, want))


@BOTH
def test_rows_beyond_32_bit_offsets(dtype):
    size = torch.empty(0, dtype=dtype).element_size()
    case = Case(dtype, [2, 3], [1, 3], [8, 4], [4, 8], tail=1)
    y, gx, gw = case.expect()
    stride = 2 ** 31 // 4 + 64                       # the last rows start beyond 2^31 values
    n = stride * 5 + 64
    if torch.cuda.mem_get_info()[0] < 2.5 * n * size:
        pytest.skip("too little memory")
    far = torch.empty(n, dtype=dtype, device="cuda")
    x = far.as_strided((case.n, case.layer.in_width), (stride, 1), 0)
    gy = far.as_strided((case.n, case.layer.out_width), (stride, 1), case.layer.in_width)
    x.copy_(case.x)
    gy.copy_(case.gy)
    out = torch.empty(n, dtype=dtype, device="cuda").as_strided((case.n, case.layer.out_width), (stride, 1), 0)
    out[case.live:] = 0.0
    case.layer.forward(x, case.routing, out=out)
    case.check_rows(out, y, case.outs)
    grads = case.layer.backward(x, gy, case.routing)
    case.check_rows(grads.x, gx, case.ins)
    for a, (want, tol) in zip(grads.weights, gw):
        assert np.all(np.abs(host(a) - want) <= tol)


@BOTH
def test_experts_of_an_atom(dtype):
    """Dispatch, the experts' products, combine and back, the gradients clipped: the whole as it is used, against autograd in 64 bits."""
    gen = torch.Generator("cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    n, slots, groups, comps, i, o = 333, 2, 5, [1, 3], 40, 24
    ids = torch.randint(-1, groups, (n, slots), generator=gen, device="cuda", dtype=torch.int32)
    x, mix, gy = rand(n, 4 * i), rand(n, slots), rand(n, 4 * o)
    weights = [rand(groups, i, o) for _ in comps]
    routing, layer = RowRouting(ids, groups), GroupedLinear(weights)
    rows = routing.dispatch(x)
    hidden = layer.forward(rows, routing)
    y = routing.combine(hidden, mix)
    grad_hidden, grad_mix = routing.combine_backward(gy, hidden, mix)
    grads = layer.backward(rows, grad_hidden, routing)
    grad_x = routing.dispatch_backward(grads.x)
    norm = clip_gradients(grads.weights, 1.0)

    leaves = [t.double().detach().requires_grad_() for t in (x, mix, *weights)]
    bx, bm, *bw = leaves
    live = (ids >= 0).double()
    at = ids.clamp(min=0).long()
    want, at_x = [], 0
    for c, w in zip(comps, bw):
        xd = bx[:, at_x:at_x + c * i].reshape(n, c, i)
        want.append(sum((bm[:, s] * live[:, s])[:, None, None] * torch.bmm(xd, w[at[:, s]]) for s in range(slots)).reshape(n, c * o))
        at_x += c * i
    want = torch.cat(want, dim=1)
    (want * gy.double()).sum().backward()
    want_norm = torch.sqrt(sum((w.grad ** 2).sum() for w in bw))
    # sums of at most 333 x 3 x 2 terms through three steps; the terms' sizes are bounded by the largest values' product
    rel = EPS[dtype] * 64
    for got, ref in [(y, want), (grad_x, bx.grad), (grad_mix, bm.grad), *[(g, w.grad / want_norm) for g, w in zip(grads.weights, bw)]]:
        err = (got.double() - ref.detach()).norm() / ref.detach().norm()
        assert float(err) <= rel, float(err)
    assert abs(float(norm) - float(want_norm)) <= rel * float(want_norm)


def test_matrices_that_change():
    case = Case(torch.float32, [30, 40], [1], [36], [64])
    w = case.weights[0]
    w.data = torch.randn_like(w)                     # other memory
    case.check_rows(case.layer.forward(case.x, case.routing), case.expect([w])[0], case.outs)
    w.requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        case.layer.forward(case.x, case.routing)
    with torch.no_grad():
        case.layer.forward(case.x, case.routing)
        for other, text in [(torch.randn(2, 36, 65, device="cuda"), "shape"), (torch.randn(2, 64, 36, device="cuda").transpose(1, 2), "contiguous")]:
            w.data = other
            with pytest.raises(ValueError, match=text):
                case.layer.forward(case.x, case.routing)


def test_refusals():
    case = Case(torch.float32, [3, 4], [1, 3], [4, 5], [6, 7])
    layer, routing, x, gy = case.layer, case.routing, case.x, case.gy
    for bad, text in [(lambda: layer.forward(x[:-1], routing), "shape"), (lambda: layer.forward(x.double(), routing), "dtype"), (lambda: layer.forward(x.cpu(), routing), "CUDA"),
                      (lambda: layer.forward(x, None), "RowRouting"), (lambda: layer.forward(x, RowRouting(routing.order.clone(), 3)), "groups"),
                      (lambda: layer.forward(x, routing, out=gy[:, :-1]), "shape"), (lambda: layer.forward(x, routing, out=gy.t().contiguous().t()), "unit stride"),
                      (lambda: layer.forward(x.requires_grad_(), routing), "autograd"), (lambda: layer.backward(x, gy[:, 1:], routing), "shape"),
                      (lambda: layer.backward(x.detach()[1:], gy, routing), "shape"), (lambda: GroupedLinear([case.weights[0], case.weights[1][:1]]), "shape"),
                      (lambda: GroupedLinear([case.weights[0].transpose(1, 2)]), "contiguous"), (lambda: GroupedLinear(case.weights, [1]), "components"),
                      (lambda: GroupedLinear(case.weights, [1, 2000]), "components"), (lambda: GroupedLinear(case.weights * 5), "degrees"),
                      (lambda: GroupedLinear([torch.zeros(1025, 1, 1, device="cuda")]), "groups"), (lambda: GroupedLinear([torch.zeros(2, 0, 3, device="cuda")]), "channels"),
                      (lambda: GroupedLinear([case.weights[0].half()]), "dtype")]:
        with pytest.raises(ValueError, match=text):
            bad()
        x.requires_grad_(False)
    shared = torch.zeros(case.n, 30, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        GroupedLinear([torch.zeros(2, 4, 4, device="cuda")]).forward(shared[:, :4], routing, out=shared[:, 2:6])


def test_waits_that_run_out_are_reported():
    """The test switch makes every CTA lose the matrices behind its first step of inner values and give up after a few hundred polls: what is lost holds NaN, the
    rest is right, and the next calls are."""
    case = Case(torch.float32, [1500, 0, 2700, 40], [1, 3], [70, 200], [136, 64])
    y, gx, gw = case.expect()
    layer = case.layer
    layer.check()
    layer._fixed.expire_polls = 300
    lost_y = layer.forward(case.x, case.routing)
    with pytest.raises(SymmetrixError, match="ran out"):
        layer.check()
    lost = layer.backward(case.x, case.gy, case.routing)
    with pytest.raises(SymmetrixError, match="ran out"):
        layer.check()
    layer._fixed.expire_polls = 0
    layer.check()
    for got, expect, widths in [(lost_y, y, case.outs), (lost.x, gx, case.ins)]:
        got = host(got)
        gone = 0
        for a, (want, tol) in zip(case.blocks(got[:case.live], widths), expect):
            missing = np.isnan(a)
            gone += missing.sum()
            assert np.all(missing | (np.abs(a - want) <= tol))
        assert gone > 0
        np.testing.assert_array_equal(got[case.live:], 0.0)
    for a, (want, tol) in zip(lost.weights, gw):
        assert np.all(np.isnan(host(a)) | (np.abs(host(a) - want) <= tol))
    case.check()
