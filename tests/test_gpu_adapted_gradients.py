"""Gradients of an evaluator's energy by its adapters, against their formula in 64 bits.

The evaluator's own arrays (a linear's input x, the adjoint gy of its output) stand for the rest of the model, so what is compared is
gA_g = sum w x^T (gy B^T), gB_g = sum w (x A)^T gy and gw = <x A, gy B^T>; bounds as in ``tests/test_gpu_adapters.py``.
"""
import numpy as np
import pytest
import torch

from symmetrix_b200 import MACE, SymmetrixError, structures as st
from symmetrix_b200.domain import SlabRank, evaluate_decomposed, make_slab_plan
from tests.test_gpu_adapted_model import adapters_of, box, run
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


def molecules(spec, model):
    s = st.molecular_liquid(3, seed=3)
    return st.evaluator_inputs(s, st.neighbor_list(s, spec.r_cut), model["atomic_numbers"])


def three_blocks(model_file, dtype, channels=16):
    path, model, spec = model_file("deep256", num_channels=channels, num_spline_points=32)
    ev = MACE(path, dtype=dtype)
    inp = molecules(spec, model)
    sets = {name: adapters_of(ev, name, 2, 3, q) for q, name in enumerate(("H1", "Am", "Hm", "A1"))}
    n = int(inp["num_nodes"])
    ids = np.array([[0, 1], [1, -1], [0, 0], [-1, -1]])[np.arange(n) % 4]
    return ev, inp, sets, ids, np.random.default_rng(3).uniform(0.5, 1.5, size=(n, 2))


@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("channels", [16, 33, 64])
def test_gradients_of_three_blocks(model_file, dtype, channels):
    ev, inp, sets, ids, weights = three_blocks(model_file, dtype, channels)
    for name, (down, up) in sets.items():
        ev.set_adapters(name, down, up)
    ev.assign_adapters(ids, weights)
    run(ev, inp)
    for name, (down, up) in sets.items():
        check_gradients(ev, name, down, up, ids, weights, dtype)


def test_gradients_of_three_blocks_against_differences(model_file):
    """float64, all four linears; the bound is that of ``tests/test_gpu_adapted_model.py`` for two blocks: with a step h = 1e-4 a central
    difference is off by about h^2 of the gradient's size and by the energy's rounding over h."""
    ev, inp, sets, ids, weights = three_blocks(model_file, "float64")

    def energy():
        for name, (down, up) in sets.items():
            ev.set_adapters(name, down, up)
        ev.assign_adapters(ids, weights)
        return run(ev, inp)[0].sum()

    total = energy()
    grads = {name: ev.adapter_gradients(name) for name in sets}
    h, rng = 1e-4, np.random.default_rng(5)

    def check(array, grad):
        scale = np.abs(grad).max()
        for _ in range(3):
            at = tuple(int(rng.integers(0, m)) for m in array.shape)
            old, d = array[at], []
            for sign in (1, -1):
                array[at] = old + sign * h
                d.append(energy())
            array[at] = old
            assert abs((d[0] - d[1]) / (2 * h) - grad[at]) <= 1e-6 * scale + 1e-11 * abs(total)

    for name, (down, up) in sets.items():
        for q in range(len(down)):
            check(down[q], grads[name][0][q])
            check(up[q], grads[name][1][q])
    check(weights, sum(g[2] for g in grads.values()))


@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("mode", ["message_passing", "recompute"])
def test_decomposed_evaluations(model_file, dtype, mode):
    """Two ranks (emulated on one GPU), each with the adapters of its own rows, owned atoms and ghosts: energies, forces and the ranks' sum of
    gradients are those of one domain, to the evaluator's bounds. With recomputed ghosts a linear's gradients are to be had while the
    receivers that it ran on are the active ones."""
    path, model, spec = model_file("fcc128", num_channels=32, num_spline_points=32)
    s = st.fcc_box((8, 3, 3), 3.6, model["atomic_numbers"], seed=17, jitter=0.12)
    rng = np.random.default_rng(2)
    ids, weights = rng.integers(-1, 3, size=(s.num_atoms, 2)), rng.uniform(0.5, 1.5, size=(s.num_atoms, 2))
    one = MACE(path)
    sets = {name: adapters_of(one, name, 3, 4, q) for q, name in enumerate(("H1", "A1"))}

    def give(ev, rows):
        for name, (down, up) in sets.items():
            ev.set_adapters(name, down, up)
        ev.assign_adapters(ids[rows], weights[rows])

    give(one, np.arange(s.num_atoms))
    run(one, st.evaluator_inputs(s, st.neighbor_list(s, one.r_cut), one.atomic_numbers))
    f_ref, _, e_ref = one.reduce_forces()
    want = {name: one.adapter_gradients(name) for name in sets}
    ranks = []
    for r in range(2):
        ev = MACE(path, dtype=dtype)
        rk = SlabRank(make_slab_plan(s, spec.r_cut, r, 2, mode=mode), ev, spec.r_cut, ev.atomic_numbers)
        give(ev, np.concatenate([rk.plan.own_global, rk.plan.ghost_global]))
        rk.build_edges()
        ranks.append(rk)
    rel, fabs = (1e-10, 1e-9) if dtype == "float64" else (1e-4, 1e-3)
    for _ in range(2):
        energy, _, owned = evaluate_decomposed(ranks)
        forces = np.zeros_like(f_ref)
        for rk, f in zip(ranks, owned):
            forces[rk.plan.own_global] = f.cpu().numpy()
        assert abs(energy - e_ref) <= rel * abs(e_ref) and np.abs(forces - f_ref).max() <= fabs
        for name in ("H1", "A1"):
            total = [np.zeros(a.shape) for a in (*want[name][0], *want[name][1])]
            for rk in ranks:
                if mode == "recompute" and name == "A1":
                    with pytest.raises(SymmetrixError, match="no evaluation"):
                        rk.ev.adapter_gradients(name)
                    rk.ev.set_active_nodes(rk.plan.n_own)
                down, up, _ = rk.ev.adapter_gradients(name)
                total = [t + a for t, a in zip(total, (*down, *up))]
            for t, a in zip(total, (*want[name][0], *want[name][1])):
                assert np.abs(t - a).max() <= 10 * rel * np.abs(a).max()


@pytest.mark.parametrize("dtype", ["float64", "float32"])
def test_no_gradients_of_arrays_that_were_changed(model_file, dtype):
    """A linear's gradients are made of its input, the kept products of that input, and the adjoint of its output: other values in one of them
    (put there, received from another rank, added by a reverse stage) and they are refused until the stages have gone through again."""
    path, model, spec = model_file("fcc128", num_channels=24, num_spline_points=32)
    ev = MACE(path, dtype=dtype)
    inp = box(spec, model, 2, 7)
    n = int(inp["num_nodes"])
    ids, weights = np.arange(n)[:, None] % 3 - 1, np.linspace(0.5, 1.5, n)[:, None]
    sets = {name: adapters_of(ev, name, 2, 3, q) for q, name in enumerate(("H1", "A1"))}
    for name, (down, up) in sets.items():
        ev.set_adapters(name, down, up)
    ev.assign_adapters(ids, weights)

    def refused(*names):
        for name in sets:
            if name in names:
                with pytest.raises(SymmetrixError, match="no evaluation"):
                    ev.adapter_gradients(name)
            else:
                ev.adapter_gradients(name)

    run(ev, inp)
    refused()
    ev.set("M0", 2.0 * ev.get("M0"))
    refused("H1")
    ev.reverse_H1()
    refused("H1")                                     # the products kept are those of the old input
    ev.compute_H1()
    refused("H1", "A1")
    run(ev, inp)
    ev.set("H1_adj", 2.0 * ev.get("H1_adj"))
    refused("H1")
    ev.reverse_H1()
    refused()
    check_gradients(ev, "H1", *sets["H1"], ids, weights, dtype)
    ev.set("A1_adj", 2.0 * ev.get("A1_adj"))
    refused("A1")
    ev.reverse_A1()
    refused()
    check_gradients(ev, "A1", *sets["A1"], ids, weights, dtype)
    ev.reverse_Phi1(zero_dxyz=False, zero_H1_adj=False)            # adds to the adjoint of H1 once more
    refused("H1")
    run(ev, inp)
    rows = torch.arange(3, dtype=torch.int32, device="cuda")
    ev.halo_unpack("H1_adj", rows, ev.halo_pack("H1_adj", rows), add=True)
    refused("H1")
    run(ev, inp)
    ev.reverse_M1()
    refused("A1")
    run(ev, inp)
    ev.compute_Phi1()
    refused("H1", "A1")
    ev.reverse_A1()
    refused("H1", "A1")                               # no products of the new input have been kept
    run(ev, inp)
    refused()
