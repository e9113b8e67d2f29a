"""The common norm and clipping against their definition in 64 bits. Squares, sums and products are float64, so the norm is off by at most
(n + 3) 2^-53 of itself in whatever order n squares are added (EPS is twice that step), and a float32 output by one rounding more, 2^-24 of itself."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import GradientSet, clip_gradients, gradient_norm

pytestmark = pytest.mark.gpu

EPS64 = 2.0 ** -52


def make(lengths, types, seed=0, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return [torch.randn(n, generator=gen, device="cuda", dtype=t) * scale for n, t in zip(lengths, types)]


def expect(tensors, max_norm):
    wide = [t.detach().double().cpu().numpy().reshape(-1) for t in tensors]
    norm = np.sqrt(sum(float(np.dot(w, w)) for w in wide))
    return norm, [w * (max_norm / norm if norm > max_norm else 1.0) for w in wide]


def check(outs, want, count):
    for o, w in zip(outs, want):
        tol = np.abs(w) * (EPS64 * (count + 4) + (2.0 ** -24 if o.dtype == torch.float32 else 0.0)) + (2.0 ** -150 if o.dtype == torch.float32 else 0.0)
        assert np.all(np.abs(o.double().cpu().numpy().reshape(-1) - w) <= tol)


F, D = torch.float32, torch.float64
LISTS = [
    ([1], [F]), ([1], [D]), ([0, 3], [F, D]), ([5, 0, 7], [F, F, D]), ([4096], [F]), ([2048, 4097], [D, F]), ([4095, 1, 2049], [F, D, D]), ([100000, 3, 77777], [F, F, D]),
    ([13] * 32, [F] * 32), ([13] * 33, [F, D, F] * 11), ([3] * 256, [D] * 256), ([3] * 257, [F] * 257), ([17] * 1000, [F] * 1000), ([5] * 2333, [F] * 2333), ([6000000, 9], [F, D]),
]


@pytest.mark.parametrize("lengths,types", LISTS)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("in_place", [True, False])
def test_norm_and_clipping(lengths, types, max_norm, in_place):
    tensors = make(lengths, types)
    count = sum(lengths)
    norm, want = expect(tensors, max_norm)
    got = gradient_norm(tensors)
    assert got.dtype == torch.float64 and got.dim() == 0 and abs(float(got) - norm) <= norm * EPS64 * (count + 3)
    before = [t.clone() for t in tensors]
    out = None if in_place else [torch.full_like(t, 7.0) for t in tensors]
    same = clip_gradients(tensors, max_norm, out=out)
    assert float(same) == float(got)
    check(tensors if in_place else out, want, count)
    if not in_place or norm <= max_norm:
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))


@pytest.mark.parametrize("dtype", [F, D])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_starts_and_neighbours(dtype, shift):
    # parts of one buffer, next to one another and on no boundary; what lies between and around them stays
    flat = torch.randn(60000, device="cuda", dtype=dtype)
    spans = [(shift, shift + 20001), (shift + 20001, shift + 20002), (shift + 20005, 50000)]
    parts = [flat[a:b] for a, b in spans]
    norm, want = expect(parts, 1.0)
    before = flat.clone()
    clip_gradients(parts, 1.0)
    check(parts, want, 50000)
    keep = torch.ones(60000, dtype=torch.bool, device="cuda")
    for a, b in spans:
        keep[a:b] = False
    assert torch.equal(flat[keep], before[keep])


def test_out_on_another_boundary():
    t = make([5000], [F])[0]
    out = torch.zeros(5003, device="cuda")
    clip_gradients([t], 1.0, out=[out[3:]])
    check([out[3:]], expect([t], 1.0)[1], 5000)
    assert not out[:3].any()


@pytest.mark.parametrize("dtype,size", [(F, 1e38), (F, 1e-38), (F, 1e-44), (D, 1e150), (D, 1e-150)])
def test_sizes_at_the_types_limits(dtype, size):
    tensors = make([3000, 17], [dtype, dtype], scale=1.0)
    tensors = [(t.clamp(-2.0, 2.0) * size).to(dtype) for t in tensors]
    norm, want = expect(tensors, size)
    assert np.isfinite(norm) and norm > 0
    assert abs(float(gradient_norm(tensors)) - norm) <= norm * EPS64 * 3020
    clip_gradients(tensors, size)
    check(tensors, want, 3017)


def test_values_that_are_not_finite():
    for value, wide in [(float("nan"), False), (float("nan"), True), (float("inf"), False), (-float("inf"), True)]:
        tensors = make([5000, 300], [F, D])
        tensors[int(wide)][250] = value
        norm = clip_gradients(tensors, 1.0)
        if np.isnan(value):
            assert norm.isnan() and all(t.isnan().all() for t in tensors)
        else:
            assert norm.isinf() and tensors[int(wide)][250].isnan() and sum(int((t != 0).sum()) for t in tensors) == 1
        tensors = make([5000, 300], [F, D])
        tensors[int(wide)][250] = value
        before = [t.clone() for t in tensors]
        clip_gradients(tensors, float("inf"))
        if not np.isnan(value):
            assert all(torch.equal(a, b) for a, b in zip(tensors, before))


def test_nothing_and_zero():
    zero = torch.zeros(10, device="cuda")
    assert float(clip_gradients([zero], 0.0)) == 0.0 and not zero.any()
    empty = torch.zeros(0, device="cuda")
    assert float(gradient_norm([empty])) == 0.0 and float(clip_gradients([empty], 1.0)) == 0.0
    t = torch.ones(10, device="cuda")
    assert float(clip_gradients([t], 0.0)) == np.sqrt(10.0) and not t.any()


def test_a_norm_at_the_limit_changes_nothing():
    t = torch.zeros(9, device="cuda")
    t[3], t[5] = 3.0, 4.0
    before = t.clone()
    assert float(clip_gradients([t], 5.0)) == 5.0 and torch.equal(t, before)
    assert float(clip_gradients([t], 2.5)) == 5.0 and torch.equal(t, before / 2)


def test_the_same_call_gives_the_same_bits():
    tensors = make([3000001, 700, 50001], [F, F, D])
    norms = {float(gradient_norm(tensors)) for _ in range(5)}
    outs = [torch.empty_like(t) for t in tensors], [torch.empty_like(t) for t in tensors]
    for out in outs:
        norms.add(float(clip_gradients(tensors, 1.0, out=out)))
    assert len(norms) == 1 and all(torch.equal(a, b) for a, b in zip(*outs))


def test_sets_streams_and_graphs():
    tensors = make([100000, 3, 5000], [F, D, D])
    outs = [torch.empty_like(t) for t in tensors]
    both = GradientSet(tensors, out=outs)
    norm, want = expect(tensors, 1.0)
    first = both.clip(1.0)
    check(outs, want, 105003)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both.norm()
    torch.cuda.synchronize()
    assert float(other) == float(first)
    graphs, norms = [], []
    alone = GradientSet(tensors)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(alone.norm())
        graphs.append(graph)
    for t in tensors:
        t.mul_(2.0)                                  # the set's tensors are read when the graph runs
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert all(float(n) == 2.0 * float(first) for n in norms)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clipped = both.clip(1.0)
    for t in tensors:
        t.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert float(clipped) == float(first)
    check(outs, want, 105003)


def test_a_set_keeps_its_memory():
    t = torch.full((1000,), 3.0, device="cuda")
    kept, old = GradientSet([t]), t.detach()
    t.data = torch.zeros(1000, device="cuda")
    torch.empty(1000, device="cuda").fill_(7.0)      # would take the old memory, were it free
    assert abs(float(kept.clip(1.0)) - 3.0 * np.sqrt(1000.0)) < 1e-10 and abs(float(old.norm()) - 1.0) < 1e-6 and not t.any()


def test_a_long_tensor():
    n = 2 ** 31 + 4099
    if torch.cuda.mem_get_info()[0] < 1.2 * 4 * n:
        pytest.skip("too little memory")
    t = torch.zeros(n, device="cuda")
    t[0], t[2 ** 31 - 1], t[2 ** 31 + 1], t[n - 1] = 1.0, 2.0, -2.0, 4.0
    assert float(clip_gradients([t], 2.5)) == 5.0
    assert [float(t[i]) for i in (0, 2 ** 31 - 1, 2 ** 31 + 1, n - 1)] == [0.5, 1.0, -1.0, 2.0] and int(torch.count_nonzero(t)) == 4


def test_refusals():
    a, b = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    for bad, text in [(lambda: gradient_norm([]), "at least one"), (lambda: gradient_norm([a.half()]), "dtype"), (lambda: gradient_norm([a.cpu()]), "CUDA"),
                      (lambda: gradient_norm([a[::2]]), "contiguous"), (lambda: gradient_norm([a[:1].expand(4)]), "contiguous"), (lambda: clip_gradients([a, a], 1.0), "share memory"),
                      (lambda: clip_gradients([a[:6], a[5:]], 1.0), "share memory"), (lambda: clip_gradients([a[:5]], 1.0, out=[a[1:6]]), "share memory"),
                      (lambda: clip_gradients([a, b], 1.0, out=[b, a]), "share memory"), (lambda: clip_gradients([a], 1.0, out=[b[:5]]), "shape"),
                      (lambda: clip_gradients([a], 1.0, out=[b.double()]), "dtype"), (lambda: clip_gradients([a], -1.0), "negative"), (lambda: clip_gradients([a], float("nan")), "NaN"),
                      (lambda: clip_gradients([a.clone().requires_grad_()], 1.0), "autograd")]:
        with pytest.raises(ValueError, match=text):
            bad()
    assert float(clip_gradients([a, b], 1.0, out=[a, b])) == 0.0          # an output may be its own tensor
