"""Gradients of an evaluator's energy by its adapters, against their formula in 64 bits.

The evaluator's own arrays (a linear's input x, the adjoint gy of its output) stand for the rest of the model, so what is compared is
gA_g = sum w x^T (gy B^T), gB_g = sum w (x A)^T gy and gw = <x A, gy B^T>; bounds as in ``tests/test_gpu_adapters.py``.
"""
import numpy as np
import pytest
import torch

from symmetrix_b200 import MACE, structures as st
from tests.test_gpu_adapted_model import adapters_of
from tests.test_gpu_adapters import EPS

pytestmark = pytest.mark.gpu

INPUT = {"H1": "M0", "A1": "Phi1", "Hm": "Mm", "Am": "Phim"}


def formula(x, gy, shapes, down, up, ids, weights, absolute):
    f = np.abs if absolute else np.asarray
    n, slots = ids.shape
    gds, gus, gw, at_x, at_y = [], [], np.zeros(ids.shape), 0, 0
    for l, ((i, o), a, b) in enumerate(zip(shapes, down, up)):
        c = 2 * l + 1
        xd, gd = f(x[:, at_x:at_x + c * i]).reshape(n, c, i), f(gy[:, at_y:at_y + c * o]).reshape(n, c, o)
        at_x, at_y = at_x + c * i, at_y + c * o
        ga, gb = np.zeros(a.shape), np.zeros(b.shape)
        for s in range(slots):
            for g in range(a.shape[0]):
                sel = np.flatnonzero(ids[:, s] == g)
                w = f(weights[sel, s])[:, None, None]
                t, h = xd[sel] @ f(a[g]), gd[sel] @ f(b[g]).T
                ga[g] += np.tensordot(xd[sel], w * h, axes=([0, 1], [0, 1]))
                gb[g] += np.tensordot(w * t, gd[sel], axes=([0, 1], [0, 1]))
                gw[sel, s] += (t * h).sum((1, 2))
        gds.append(ga); gus.append(gb)
    return gds, gus, gw


def check_gradients(ev, linear, down, up, ids, weights, dtype):
    """`ids` outside the adapters are empty slots."""
    shapes = ev._adapter_shapes(linear)
    n, slots = ids.shape
    value = np.float32 if dtype == "float32" else np.float64
    exact = lambda a: np.asarray(a, dtype=value).astype(np.float64)  # noqa: E731
    down, up, weights = [exact(a) for a in down], [exact(b) for b in up], exact(weights)
    x, gy = ev.get(INPUT[linear]).reshape(n, -1), ev.get(linear + "_adj")
    gy = gy[:n * sum((2 * l + 1) * o for l, (_, o) in enumerate(shapes))].reshape(n, -1)
    assert np.abs(gy).max() > 0 and np.isfinite(gy).all()
    got = ev.adapter_gradients(linear)
    want, size = (formula(x, gy, shapes, down, up, ids, weights, absolute) for absolute in (False, True))
    eps, rank = EPS[torch.float32 if dtype == "float32" else torch.float64], down[0].shape[2]
    most_i, most_o, terms = max(i for i, _ in shapes), max(o for _, o in shapes), n * slots * (2 * len(shapes) - 1)
    steps = {"down": terms + most_o + 24, "up": terms + most_i + 24, "weights": len(shapes) ** 2 * rank + most_i + most_o + 24}
    for name, g, r, m in zip(steps, got, want, size):
        for a, b, c in (zip(g, r, m) if name != "weights" else [(g, r, m)]):
            assert a.shape == b.shape and (np.abs(a - b) <= steps[name] * eps * c).all(), (linear, name)


@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("channels", [16, 32])
def test_gradients_of_many_atoms(model_file, dtype, channels):
    """Up to 32 channels and rows enough for five tiles of 128 on each of 148 CTAs, in both linears."""
    path, model, spec = model_file("fcc128", num_channels=channels, num_spline_points=32, r_cut=4.0)
    ev = MACE(path, dtype=dtype)
    s = st.fcc_box(18, 3.6, model["atomic_numbers"], seed=4)
    n, types = s.num_atoms, np.array([list(model["atomic_numbers"]).index(z) for z in s.numbers])
    assert 4 * n > 4.8 * 148 * 128
    rng = np.random.default_rng(1)
    sets = {name: adapters_of(ev, name, 3, 4, q) for q, name in enumerate(("H1", "A1"))}
    for name, (down, up) in sets.items():
        ev.set_adapters(name, down, up)
    for slots in (1, 2):
        ids, weights = rng.integers(-1, 3, size=(n, slots)), rng.uniform(0.5, 1.5, size=(n, slots))
        ev.assign_adapters(ids, weights)
        ev.evaluate(s.positions, types, s.cell, s.pbc)
        for name, (down, up) in sets.items():
            check_gradients(ev, name, down, up, ids, weights, dtype)
