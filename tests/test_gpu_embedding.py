"""Embeddings against their definition in 64 bits on the host. A sum of n products computed with unit roundoff u is off by at most (n + 2) u sum |terms|
(the two more: a factor in front, and a weight times it), in whatever order it is added; EPS is twice the unit roundoff."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import Embedding, EmbeddingPlan, GradientSet

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.float64: 2.0 ** -52}
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.float64])


def host(t):
    return t.detach().double().cpu().numpy()


def tokens_of(rng, n, slots, rows, kind):
    ids = rng.integers(0, rows, size=(n, slots))
    if kind == "skewed":
        ids = np.where(rng.random((n, slots)) < 0.95, rows // 2, ids)
    elif kind == "one":
        ids[:] = rows - 1
    elif kind == "empty":
        ids[:] = -1
    elif kind == "outside":
        ids[rng.random((n, slots)) < 0.3] = rows
        ids[rng.random((n, slots)) < 0.2] = 2 ** 31 - 1
        ids[rng.random((n, slots)) < 0.2] = -2 ** 31
    return torch.as_tensor(ids.astype(np.int32)).cuda()


def sorted_pairs(ids, rows):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    key = np.where((flat < 0) | (flat >= rows), rows, flat)
    order = np.argsort(key, kind="stable")
    return key, order


def expect(table, ids, weights, gy, scale):
    """y, grad_table, grad_weights with bounds of their errors."""
    n, slots = ids.shape
    rows, width = table.shape
    key, _ = sorted_pairs(ids, rows)
    live = np.flatnonzero(key < rows)
    w = (host(weights) if weights is not None else np.ones((n, slots))).reshape(-1)
    t, g = host(table), host(gy)
    eps = EPS[table.dtype]
    out = []
    for f in (lambda v: v, np.abs):
        y, gt, gw = np.zeros((n, width)), np.zeros((rows, width)), np.zeros(n * slots)
        np.add.at(y, live // slots, f(scale * w[live])[:, None] * f(t[key[live]]))
        np.add.at(gt, key[live], f(scale * w[live])[:, None] * f(g[live // slots]))
        gw[live] = f(np.float64(scale)) * (f(t[key[live]]) * f(g[live // slots])).sum(1)
        out.append((y, gt, gw.reshape(n, slots)))
    counts = np.bincount(key, minlength=rows + 1)[:rows, None]
    return [(a, b * eps * k) for a, b, k in zip(out[0], out[1], (slots + 2, counts + 2, width + 2))]


def check(got, want):
    assert np.all(np.abs(host(got) - want[0]) <= want[1]), np.max(np.abs(host(got) - want[0]) / (want[1] + 1e-300))


@pytest.mark.parametrize("n,slots,rows", [
    (0, 1, 1), (1, 1, 1), (1, 64, 5), (33, 1, 3), (100, 3, 1022), (100, 3, 1023), (100, 3, 1024), (500, 2, 1025), (1000, 1, 5000), (8192, 1, 1023), (8193, 1, 1023),
    (8193, 1, 1024), (4097, 2, 20000), (30000, 3, 1424), (70001, 1, 1048575), (200000, 2, 89), (300, 1, 1048575),
    (5000, 1, 4095), (9000, 1, 4094), (9000, 1, 4095), (9000, 1, 4096), (30000, 2, 4097), (303105, 1, 2499), (303105, 1, 2500), (303104, 1, 4095), (75776, 1, 7), (75777, 1, 7), (151552, 1, 40), (50519, 3, 40),
])
@pytest.mark.parametrize("kind", ["random", "skewed", "one", "outside", "empty"])
def test_plan(n, slots, rows, kind):
    rng = np.random.default_rng(n + rows)
    ids = tokens_of(rng, n, slots, rows, kind)
    plan = EmbeddingPlan(ids, rows)
    for q in range(2):
        key, order = sorted_pairs(ids, rows)
        np.testing.assert_array_equal(plan.order.cpu().numpy(), order)
        np.testing.assert_array_equal(plan.tokens.cpu().numpy(), key[order])
        ids = tokens_of(rng, n, slots, rows, "random")
        plan.update(ids)


SIZES = [(1, 1, 1, 1), (1, 1, 1, 4), (5, 3, 2, 7), (18, 1, 10, 128), (37, 2, 100, 33), (100, 5, 8, 130), (257, 9, 4, 36), (3000, 2, 1700, 20), (33, 2, 4, 2304), (2000, 1, 2, 520),
         (9000, 1, 3, 12), (3, 64, 40, 8)]


@BOTH
@pytest.mark.parametrize("n,slots,rows,width", SIZES)
@pytest.mark.parametrize("kind", ["random", "skewed", "one", "outside", "empty"])
@pytest.mark.parametrize("weighted", [True, False])
def test_lookup_and_gradients(dtype, n, slots, rows, width, kind, weighted):
    gen = torch.Generator("cuda").manual_seed(n + width)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    ids = tokens_of(np.random.default_rng(width), n, slots, rows, kind)
    table, weights, gy = rand(rows, width), rand(n, slots) if weighted else None, rand(n, width)
    scale = 1.75 if weighted else 1.0
    want = expect(table, ids, weights, gy, scale)
    empty = (ids < 0) | (ids >= rows)
    if weighted:
        weights[empty] = float("nan")                # of empty slots nothing is read
    gy[empty.all(dim=1)] = float("inf")
    embedding, plan = Embedding(table, scale), EmbeddingPlan(ids, rows)
    check(embedding.forward(ids, weights), want[0])
    grads = embedding.backward(gy, plan, weights)
    check(grads.table, want[1])
    check(grads.weights, want[2])
    assert not host(grads.weights)[empty.cpu().numpy()].any()
    only = embedding.backward(gy, plan, weights, want_weights=False)
    assert only.weights is None and torch.equal(only.table, grads.table)
    only = embedding.backward(gy, plan, weights, want_table=False)
    assert only.table is None and torch.equal(only.weights, grads.weights)
    again = embedding.backward(gy, plan, weights)
    assert torch.equal(again.table, grads.table) and torch.equal(again.weights, grads.weights)


@BOTH
def test_long_runs(dtype):
    # runs over many chunks, that begin and end at and between the chunks' borders
    gen = torch.Generator("cuda").manual_seed(1)
    for n, borders in [(40000, [1, 64, 65, 20000, 39999]), (16 * 50, [16, 32, 33, 200, 784]), (700000, [3, 300000, 300001])]:
        ids = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
        for b in borders:
            ids[b:] += 1
        ids = ids[torch.randperm(n, generator=gen, device="cuda")].contiguous()
        table = torch.randn(len(borders) + 1, 8, generator=gen, device="cuda", dtype=dtype)
        gy = torch.randn(n, 8, generator=gen, device="cuda", dtype=dtype)
        want = expect(table, ids, None, gy, 1.0)
        check(Embedding(table).backward(gy, EmbeddingPlan(ids, table.shape[0])).table, want[1])


@BOTH
@pytest.mark.parametrize("shift,extra", [(0, 4), (1, 0), (1, 3), (2, 6)])
def test_strides_and_starts(dtype, shift, extra):
    gen = torch.Generator("cuda").manual_seed(2)

    def rows_of(n, w):
        t = torch.randn(shift + n * (w + extra) + 8, generator=gen, device="cuda", dtype=dtype)
        return t.as_strided((n, w), (w + extra, 1), shift)

    ids = tokens_of(np.random.default_rng(0), 300, 2, 40, "outside")
    table, gy, out, weights = rows_of(40, 36), rows_of(300, 36), rows_of(300, 36), rows_of(300, 2)
    want = expect(table, ids, weights, gy, 0.5)
    embedding = Embedding(table, 0.5)
    assert embedding.forward(ids, weights, out=out) is out
    check(out, want[0])
    grads = embedding.backward(gy, EmbeddingPlan(ids, 40), weights)
    check(grads.table, want[1])
    check(grads.weights, want[2])
    check(embedding.backward(gy.t().contiguous().t(), EmbeddingPlan(ids, 40), weights).table, want[1])
    wide = torch.full((300, 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 1:3] = ids
    check(embedding.forward(wide[:, 1:3], weights), want[0])
    table.mul_(2.0)                                  # values changed in place count
    check(embedding.forward(ids, weights), expect(table, ids, weights, gy, 0.5)[0])


@BOTH
def test_one_dimension(dtype):
    ids = torch.tensor([2, 0, -1, 2], dtype=torch.int32, device="cuda")
    table = torch.arange(12, device="cuda", dtype=dtype).view(3, 4)
    embedding, plan = Embedding(table), EmbeddingPlan(ids, 3)
    weights = torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda", dtype=dtype)
    assert embedding.forward(ids).tolist() == [[8, 9, 10, 11], [0, 1, 2, 3], [0] * 4, [8, 9, 10, 11]]
    assert embedding.forward(ids, weights).tolist() == [[8, 9, 10, 11], [0, 2, 4, 6], [0] * 4, [32, 36, 40, 44]]
    grads = embedding.backward(torch.ones(4, 4, device="cuda", dtype=dtype), plan, weights)
    assert grads.table.tolist() == [[2] * 4, [0] * 4, [5] * 4] and grads.weights.tolist() == [[38], [6], [0], [38]]


@BOTH
def test_values_that_are_not_finite(dtype):
    ids = tokens_of(np.random.default_rng(4), 500, 2, 30, "random")
    table, gy = torch.ones(30, 40, device="cuda", dtype=dtype), torch.ones(500, 40, device="cuda", dtype=dtype)
    table[7, 3], gy[11, 5] = float("inf"), float("nan")
    embedding, plan = Embedding(table), EmbeddingPlan(ids, 30)
    y = embedding.forward(ids)
    named = (ids == 7).any(dim=1)
    assert torch.equal(~y.isfinite(), named[:, None] & (torch.arange(40, device="cuda") == 3))
    grads = embedding.backward(gy, plan)
    bad = torch.zeros(30, 40, dtype=torch.bool, device="cuda")
    bad[ids[11].long(), 5] = True
    assert torch.equal(grads.table.isnan(), bad)
    expect_w = (ids == 7) | (torch.arange(500, device="cuda") == 11)[:, None]
    assert torch.equal(~grads.weights.isfinite(), expect_w)


@BOTH
def test_streams_and_graphs(dtype):
    gen = torch.Generator("cuda").manual_seed(5)
    n, rows, width = 9000, 2000, 24
    ids = tokens_of(np.random.default_rng(5), n, 2, rows, "skewed")
    table, weights, gy = (torch.randn(*s, generator=gen, device="cuda", dtype=dtype) for s in ((rows, width), (n, 2), (n, width)))
    embedding, plan = Embedding(table), EmbeddingPlan(ids, rows)
    y, grads = embedding.forward(ids, weights), embedding.backward(gy, plan, weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan2 = EmbeddingPlan(ids, rows)
        got = embedding.forward(ids, weights), embedding.backward(gy, plan2, weights), embedding.backward(gy, plan, weights)
    torch.cuda.synchronize()
    assert torch.equal(got[0], y) and all(torch.equal(g.table, grads.table) and torch.equal(g.weights, grads.weights) for g in got[1:])
    static, graphs, results = torch.zeros_like(ids), [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p = EmbeddingPlan(static, rows)
            results.append((embedding.forward(static, weights), embedding.backward(gy, p, weights), p))
        graphs.append(graph)
    static.copy_(ids)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for got_y, got, p in results:
        assert torch.equal(got_y, y) and torch.equal(got.table, grads.table) and torch.equal(got.weights, grads.weights) and torch.equal(p.order, plan.order)


@BOTH
def test_rows_beyond_32_bit_offsets(dtype):
    size = torch.empty(0, dtype=dtype).element_size()
    stride = 2 ** 31 // 3 + 16
    n = 4 * stride + 16
    if torch.cuda.mem_get_info()[0] < 1.5 * n * size:
        pytest.skip("too little memory")
    far = torch.empty(n, dtype=dtype, device="cuda")
    table = far.as_strided((5, 8), (stride, 1), 0)
    gy = far.as_strided((4, 8), (stride, 1), 8)
    gen = torch.Generator("cuda").manual_seed(6)
    table.copy_(torch.randn(5, 8, generator=gen, device="cuda", dtype=dtype))
    gy.copy_(torch.randn(4, 8, generator=gen, device="cuda", dtype=dtype))
    ids = torch.tensor([[4], [3], [4], [0]], dtype=torch.int32, device="cuda")
    want = expect(table, ids, None, gy, 1.0)
    embedding = Embedding(table)
    check(embedding.forward(ids), want[0])
    grads = embedding.backward(gy, EmbeddingPlan(ids, 5))
    check(grads.table, want[1])
    check(grads.weights, want[2])


@BOTH
def test_gradients_are_differences(dtype):
    # linear in the table and in the weights: a difference of any step is the derivative, up to the roundings of two sums
    gen = torch.Generator("cuda").manual_seed(7)
    ids = tokens_of(np.random.default_rng(7), 20, 3, 6, "outside")
    table, weights, gy = (torch.randn(*s, generator=gen, device="cuda", dtype=dtype) for s in ((6, 5), (20, 3), (20, 5)))
    embedding = Embedding(table, 1.5)
    grads = embedding.backward(gy, EmbeddingPlan(ids, 6), weights)
    size = float(table.abs().max() * weights.abs().sum() * gy.abs().sum())

    def loss():
        return float((embedding.forward(ids, weights).double() * gy.double()).sum())

    for t, g in [(table, grads.table), (weights, grads.weights)]:
        for at in range(0, t.numel(), 7):
            flat, old = t.view(-1), float(t.view(-1)[at])
            flat[at] = old + 1.0
            up, plus = loss(), float(flat[at])
            flat[at] = old - 1.0
            down, minus = loss(), float(flat[at])
            flat[at] = old
            assert abs((up - down) / (plus - minus) - float(g.view(-1)[at])) <= 10 * EPS[dtype] * size


def test_a_step_of_training():
    """Lookup, gradients, clipping in buffers of their own, twice: the table moves against its gradient by the clipped length."""
    gen = torch.Generator("cuda").manual_seed(8)
    ids = tokens_of(np.random.default_rng(8), 400, 1, 50, "random")
    table, gy = torch.randn(50, 16, generator=gen, device="cuda"), torch.randn(400, 16, generator=gen, device="cuda")
    embedding, plan, buffer = Embedding(table), EmbeddingPlan(ids, 50), torch.zeros(50, 16, device="cuda")
    together = GradientSet([buffer])
    for _ in range(2):
        before = table.clone()
        buffer.copy_(embedding.backward(gy, plan).table)
        norm = together.clip(0.25)
        assert float(norm) > 0.25 and abs(float(buffer.double().norm()) - 0.25) <= 0.25 * 2.0 ** -22
        table -= buffer
        moved = embedding.forward(ids) - before[ids[:, 0].long()]
        assert torch.allclose(moved, -buffer[ids[:, 0].long()], rtol=0.0, atol=2.0 ** -22 * float(before.abs().max()))


def test_a_table_that_changes():
    table = torch.randn(5, 8, device="cuda")
    ids = torch.tensor([4, 0], dtype=torch.int32, device="cuda")
    embedding = Embedding(table)
    table.data = torch.randn(5, 8, device="cuda")            # other memory
    assert torch.equal(embedding.forward(ids), table[[4, 0]])
    table.requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        embedding.forward(ids)
    with torch.no_grad():
        assert torch.equal(embedding.forward(ids), table[[4, 0]])
        table.data = torch.randn(6, 8, device="cuda")
        with pytest.raises(ValueError, match="shape"):
            embedding.forward(ids)


def test_refusals():
    table = torch.zeros(4, 6, device="cuda")
    ids = torch.zeros(5, 2, dtype=torch.int32, device="cuda")
    embedding, plan, gy = Embedding(table), EmbeddingPlan(ids, 4), torch.zeros(5, 6, device="cuda")
    for bad, text in [(lambda: Embedding(table.half()), "dtype"), (lambda: Embedding(table[:0]), "rows"), (lambda: Embedding(table.t()), "unit stride"), (lambda: Embedding(table[0]), "shape"),
                      (lambda: Embedding(torch.empty(1 << 20, 1, device="cuda")), "rows"), (lambda: EmbeddingPlan(ids.long(), 4), "dtype"), (lambda: EmbeddingPlan(ids, 0), "limits"),
                      (lambda: EmbeddingPlan(ids, 1 << 20), "limits"), (lambda: EmbeddingPlan(ids, 2 ** 32 + 4), "limits"), (lambda: EmbeddingPlan(ids[:, :0], 4), "limits"), (lambda: EmbeddingPlan(ids[None], 4), "shape"),
                      (lambda: plan.update(ids[1:]), "rows"), (lambda: embedding.forward(ids.cpu()), "CUDA"), (lambda: embedding.forward(ids.float()), "dtype"),
                      (lambda: embedding.forward(ids[:, :0]), "slots"), (lambda: embedding.forward(ids, torch.zeros(5, 3, device="cuda")), "shape"),
                      (lambda: embedding.forward(ids, torch.zeros(5, 2, device="cuda").double()), "dtype"), (lambda: embedding.forward(ids, out=gy[1:]), "shape"),
                      (lambda: embedding.forward(ids[:4], out=table), "shares memory"), (lambda: embedding.backward(gy, ids), "EmbeddingPlan"),
                      (lambda: embedding.backward(gy, EmbeddingPlan(ids, 5)), "table"), (lambda: embedding.backward(gy[1:], plan), "shape"),
                      (lambda: embedding.backward(gy.clone().requires_grad_(), plan), "autograd")]:
        with pytest.raises(ValueError, match=text):
            bad()
