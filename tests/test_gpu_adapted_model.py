"""Evaluations in which every atom has its own variant of the model: adapters beside the channel-mixing linears of the evaluator.

An adapter with weight w turns the linear's matrix W into W + w down up, so a structure whose atoms all use one adapter is the model with
that matrix, which the numpy restatement evaluates. Tolerances are those of the evaluator's parity tests.
"""
import numpy as np
import pytest

from oracle.mace_numpy import MaceOracle
from oracle.mace_numpy_deep import DeepMaceOracle
from symmetrix_b200 import MACE, Symmetrix, SymmetrixError, structures as st
from tests import test_gpu_parity
from tests.test_gpu_parity import INPUT_KEYS, check_against

pytestmark = pytest.mark.gpu


def run(ev, inp):
    e, f = test_gpu_parity.run(ev, inp)
    return e, f.reshape(-1, 3)


def adapters_of(ev, linear, count, rank, seed):
    rng = np.random.default_rng(seed)
    shapes = ev._adapter_shapes(linear)
    down = [rng.standard_normal((count, i, rank)) / np.sqrt(i) for i, _ in shapes]
    up = [rng.standard_normal((count, rank, o)) * 0.4 / np.sqrt(rank) for _, o in shapes]
    return down, up


def variant(model, sets, mix):
    """The oracle of the model whose linears are W + sum_g mix[g] down[g] up[g]."""
    o = (DeepMaceOracle if model.get("num_interactions", 2) == 3 else MaceOracle)(model)
    for linear, (down, up) in sets.items():
        delta = [sum((m * a[g] @ b[g] for g, m in mix.items()), np.zeros((a.shape[1], b.shape[2]))) for a, b in zip(down, up)]
        if linear == "H1":
            o.H1_w = o.H1_w + np.array(delta)
        elif linear == "Hm":
            o.Hm_w = o.Hm_w + np.array(delta)
        else:
            w = getattr(o, linear + "_w")
            setattr(o, linear + "_w", [a + d for a, d in zip(w, delta)])
    return o


def joined(parts):
    """One edge set of several structures that do not see each other."""
    out, first = {k: [] for k in INPUT_KEYS}, 0
    for p in parts:
        for k in INPUT_KEYS[1:]:
            out[k].append(np.asarray(p[k]).reshape(-1) + (first if k == "neigh_indices" else 0))
        first += int(p["num_nodes"])
    return dict({k: np.concatenate(v) for k, v in out.items() if k != "num_nodes"}, num_nodes=first)


def box(spec, model, n, seed):
    s = st.fcc_box(n, 3.6, model["atomic_numbers"], seed=seed)
    return st.evaluator_inputs(s, st.neighbor_list(s, spec.r_cut), model["atomic_numbers"])


@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("L_max,channels", [(0, 24), (1, 33), (1, 64), (2, 16)])
def test_structures_with_variants_of_their_own(model_file, dtype, L_max, channels):
    path, model, spec = model_file("fcc128", num_channels=channels, num_spline_points=32, L_max=L_max)
    ev = MACE(path, dtype=dtype)
    sets = {"H1": adapters_of(ev, "H1", 3, 4, 1), "A1": adapters_of(ev, "A1", 3, 6, 2)}
    parts = [box(spec, model, 2, seed) for seed in (1, 2, 3, 4)]
    mixes = [{0: 0.7}, {2: 1.0, 0: -0.5}, {}, {1: 1.3}]
    ids, weights = [], []
    for p, mix in zip(parts, mixes):
        row = (list(mix.items()) + [(-1, np.nan)] * 2)[:2]
        ids += [[g for g, _ in row]] * int(p["num_nodes"])
        weights += [[w for _, w in row]] * int(p["num_nodes"])
    both = joined(parts)
    plain = run(ev, both)
    for name, (down, up) in sets.items():
        ev.set_adapters(name, down, up)
    unassigned = run(ev, both)
    assert np.array_equal(unassigned[0], plain[0])           # adapters that nobody uses
    ev.assign_adapters(np.array(ids), np.array(weights))
    before = ev.launch_count
    e, f = run(ev, both)
    assert ev.launch_count > before
    node = edge = 0
    for p, mix in zip(parts, mixes):
        e_ref, f_ref = variant(model, sets, mix).compute_node_energies_forces(p)
        n, m = int(p["num_nodes"]), len(p["r"])
        check_against(dtype, e[node:node + n], f[edge:edge + m], e_ref, np.asarray(f_ref).reshape(-1, 3))
        node, edge = node + n, edge + m
    again = run(ev, both)
    if dtype == "float64":
        assert np.array_equal(again[0], e) and np.array_equal(again[1], f)
    # stage by stage: the same sums
    ev.begin(*(both[k] for k in INPUT_KEYS))
    for name in ("A0", "M0", "H1", "Phi1", "A1", "M1", "H2", "readouts"):
        getattr(ev, "compute_" + name)()
    if dtype == "float64":
        assert np.array_equal(ev.node_energies, e)
    # one slot and no weights; then none at all
    ev.assign_adapters(np.repeat([1, -1, 5, 1], [int(p["num_nodes"]) for p in parts]))
    e1, f1 = run(ev, both)
    e_ref, _ = variant(model, sets, {1: 1.0}).compute_node_energies_forces(parts[0])
    n = int(parts[0]["num_nodes"])
    assert np.abs(e1[:n] - e_ref).max() <= (1e-9 if dtype == "float64" else 1e-3) * np.abs(e_ref).max()
    ev.assign_adapters(None)
    assert np.array_equal(run(ev, both)[0], plain[0])
    ev.set_adapters("H1", [], [])
    ev.set_adapters("A1", [], [])
    assert np.array_equal(run(ev, both)[0], plain[0])


@pytest.mark.parametrize("dtype", ["float64", "float32"])
def test_three_blocks(model_file, dtype):
    path, model, spec = model_file("deep256", num_channels=16, num_spline_points=32)
    ev = MACE(path, dtype=dtype)
    sets = {name: adapters_of(ev, name, 2, 3, q) for q, name in enumerate(("H1", "Am", "Hm", "A1"))}
    s = st.molecular_liquid(3, seed=3)
    inp = st.evaluator_inputs(s, st.neighbor_list(s, spec.r_cut), model["atomic_numbers"])
    for name, (down, up) in sets.items():
        ev.set_adapters(name, down, up)
    ev.assign_adapters(np.full(int(inp["num_nodes"]), 1), np.full(int(inp["num_nodes"]), 0.8))
    e, f = run(ev, inp)
    e_ref, f_ref = variant(model, sets, {1: 0.8}).compute_node_energies_forces(inp)
    check_against(dtype, e, f, e_ref, np.asarray(f_ref).reshape(-1, 3))


def test_gradients_against_differences(model_file):
    """float64: derivatives of the total energy by adapters and weights. The energy is a polynomial of low degree in them times smooth
    functions; a central difference of step h is off by about h^2 / 6 times the third derivative, of the size of the gradient itself for adapters of
    order one: with h = 1e-4, 1e-8 of it, and by the energy's rounding, 1e-16 |E| / h = 1e-12 |E|."""
    path, model, spec = model_file("fcc128", num_channels=12, num_spline_points=32)
    ev = MACE(path)
    sets = {name: adapters_of(ev, name, 2, 3, q) for q, name in enumerate(("H1", "A1"))}
    inp = box(spec, model, 2, 7)
    n = int(inp["num_nodes"])
    ids = np.array([[0, 1], [1, -1], [0, 0], [-1, -1]])[np.arange(n) % 4]
    weights = np.random.default_rng(3).uniform(0.5, 1.5, size=(n, 2))

    def energy():
        for name, (down, up) in sets.items():
            ev.set_adapters(name, down, up)
        ev.assign_adapters(ids, weights)
        return run(ev, inp)[0].sum()

    total = energy()
    grads = {name: ev.adapter_gradients(name) for name in sets}
    h, rng = 1e-4, np.random.default_rng(5)

    def check(array, grad, scale):
        for _ in range(4):
            at = tuple(int(rng.integers(0, m)) for m in array.shape)
            old = array[at]
            d = []
            for sign in (1, -1):
                array[at] = old + sign * h
                d.append(energy())
            array[at] = old
            assert abs((d[0] - d[1]) / (2 * h) - grad[at]) <= 1e-6 * scale + 1e-11 * abs(total)

    for name, (down, up) in sets.items():
        for q in range(len(down)):
            check(down[q], grads[name][0][q], np.abs(grads[name][0][q]).max())
            check(up[q], grads[name][1][q], np.abs(grads[name][1][q]).max())
    by_weight = sum(g[2] for g in grads.values())
    assert (by_weight[ids < 0] == 0).all()
    check(weights, by_weight, np.abs(by_weight).max())


def test_paths_in_any_order(model_file, tmp_path):
    """A file whose paths of a degree are in another order takes, and returns, the adapters' blocks in that order."""
    from symmetrix_b200.modelgen.generate import write_json
    from tests.test_gpu_parity import _permute_paths
    path, model, spec = model_file("fcc128", num_channels=8, num_spline_points=32)
    permuted = _permute_paths(model, np.random.default_rng(8))
    ppath = tmp_path / "permuted.json"
    write_json(permuted, ppath)
    inp = box(spec, model, 2, 11)
    ev = MACE(ppath)
    down, up = adapters_of(ev, "A1", 2, 3, 4)
    ev.set_adapters("A1", down, up)
    ev.assign_adapters(np.ones(int(inp["num_nodes"]), dtype=np.int32))
    e, f = run(ev, inp)
    e_ref, f_ref = variant(permuted, {"A1": (down, up)}, {1: 1.0}).compute_node_energies_forces(inp)
    check_against("float64", e, f, e_ref, np.asarray(f_ref).reshape(-1, 3))
    grad = ev.adapter_gradients("A1")[0]
    for q in range(4):
        at = (1, 3 + 8 * (grad[q].shape[1] // 8 - 1), 2)      # in the last block of the degree
        d = []
        for sign in (1, -1):
            moved = [a.copy() for a in down]
            moved[q][at] += sign * 1e-4
            ev.set_adapters("A1", moved, up)
            d.append(run(ev, inp)[0].sum())
        assert abs((d[0] - d[1]) / 2e-4 - grad[q][at]) <= 1e-6 * np.abs(grad[q]).max() + 1e-11 * abs(e.sum())


def test_calculator_and_fewer_active_nodes(model_file):
    path, model, spec = model_file("fcc128", num_channels=16, num_spline_points=32)
    s = st.fcc_box(2, 3.6, model["atomic_numbers"], seed=5)
    calc = Symmetrix(path)
    ev = calc.evaluator
    down, up = adapters_of(ev, "A1", 2, 3, 8)
    ev.set_adapters("A1", down, up)
    n = len(s.numbers)
    ev.assign_adapters(np.zeros(n + 5, dtype=np.int32))       # more nodes than the structure has: the first count
    types = np.array([list(model["atomic_numbers"]).index(z) for z in s.numbers])
    _, _, energy, _ = ev.evaluate(s.positions, types, s.cell, s.pbc)
    inp = st.evaluator_inputs(s, st.neighbor_list(s, spec.r_cut), model["atomic_numbers"])
    e_ref, _ = variant(model, {"A1": (down, up)}, {0: 1.0}).compute_node_energies_forces(inp)
    assert abs(energy - e_ref.sum()) <= 1e-10 * abs(e_ref.sum())
    ev.assign_adapters(np.zeros(n - 1, dtype=np.int32))
    with pytest.raises(SymmetrixError, match="assigned"):
        ev.evaluate(s.positions, types, s.cell, s.pbc)


def test_refusals(model_file):
    path, model, spec = model_file("fcc128", num_channels=8, num_spline_points=32)
    ev = MACE(path)
    down, up = adapters_of(ev, "H1", 2, 3, 1)
    inp = box(spec, model, 2, 1)
    n = int(inp["num_nodes"])
    with pytest.raises(SymmetrixError, match="no adapters"):
        ev.assign_adapters(np.zeros(n, dtype=np.int32))
    with pytest.raises(ValueError):
        ev.set_adapters("H2", down, up)
    with pytest.raises(ValueError):
        ev.set_adapters("H1", down[:1], up)
    with pytest.raises(ValueError):
        ev.set_adapters("H1", [d[:, :4] for d in down], up)
    with pytest.raises(SymmetrixError):
        ev.set_adapters("Hm", down, up)                       # two blocks
    with pytest.raises(SymmetrixError, match="rank"):
        ev.set_adapters("H1", [np.repeat(d, 30, axis=2) for d in down], [np.repeat(u, 30, axis=1) for u in up])
    ev.set_adapters("H1", down, up)
    with pytest.raises(SymmetrixError, match="same number"):
        ev.set_adapters("A1", *adapters_of(ev, "A1", 3, 2, 1))
    with pytest.raises(ValueError):
        ev.assign_adapters(np.zeros((n, 1, 1), dtype=np.int32))
    with pytest.raises(ValueError):
        ev.assign_adapters(np.zeros(n, dtype=np.int32), np.zeros((n, 2)))
    with pytest.raises(SymmetrixError, match="slots"):
        ev.assign_adapters(np.zeros((n, 65), dtype=np.int32))
    ev.assign_adapters(np.zeros(n, dtype=np.int32))
    with pytest.raises(SymmetrixError):
        ev.adapter_gradients("H1")                            # no evaluation yet
    run(ev, inp)
    ev.adapter_gradients("H1")
    with pytest.raises(SymmetrixError):
        ev.adapter_gradients("A1")                            # has none
    ev.set_adapters("H1", down, up)
    with pytest.raises(SymmetrixError):
        ev.adapter_gradients("H1")                            # other adapters than the evaluation's


def test_gradients_of_mixed_evaluations_are_refused(model_file):
    """Gradients need the linear's input and the adjoint of its output from one evaluation: not after new edges, not between stages."""
    path, model, spec = model_file("fcc128", num_channels=8, num_spline_points=32)
    ev = MACE(path)
    down, up = adapters_of(ev, "H1", 2, 3, 1)
    inp, other = box(spec, model, 2, 1), box(spec, model, 2, 2)
    n = int(inp["num_nodes"])
    ev.set_adapters("H1", down, up)
    ev.assign_adapters(np.arange(n, dtype=np.int32) % 2)
    run(ev, inp)
    first = ev.adapter_gradients("H1")
    args = [other[k] for k in INPUT_KEYS]
    ev.begin(int(other["num_nodes"]), *args[1:])
    with pytest.raises(SymmetrixError, match="no evaluation"):
        ev.adapter_gradients("H1")                            # the old arrays, the new edges
    for stage in ("compute_A0", "compute_M0", "compute_H1"):
        ev._stage(stage)
    with pytest.raises(SymmetrixError, match="no evaluation"):
        ev.adapter_gradients("H1")                            # the new input, the old adjoint
    run(ev, other)
    second = ev.adapter_gradients("H1")
    assert not np.array_equal(first[0][0], second[0][0])
    run(ev, inp)
    for a, b in zip(first[0] + first[1], sum(ev.adapter_gradients("H1")[:2], [])):
        np.testing.assert_array_equal(a, b)
