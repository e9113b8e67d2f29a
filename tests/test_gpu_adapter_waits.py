"""Bounded waits of the float32 linears with adapters that run out: reported by the next call that waits, and over with the next evaluation."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import MACE, SymmetrixError, _lib, structures as st
from tests.test_gpu_adapted_model import adapters_of
from tests.test_gpu_adapters import Case, everything

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cells", [2, 18])
@pytest.mark.parametrize("rank", [4, 40])
def test_an_evaluation_whose_waits_run_out_is_an_error(model_file, cells, rank):
    """The test switch takes the weights behind the first chunk from every CTA: one tile each (32 atoms) or five (23,328 atoms), two chunks a tile.
    What is lost is NaN, the call reports it, gradients of that evaluation are refused, and the next evaluation has the old results: the same
    bits up to the adjoint of A1. Behind that float32 evaluations add the senders' messages as they arrive, so forces agree to the evaluator's
    float32 bound."""
    path, model, spec = model_file("fcc128", num_channels=64, num_spline_points=32, r_cut=4.0)
    ev = MACE(path, dtype="float32")
    s = st.fcc_box(cells, 3.6, model["atomic_numbers"], seed=6)
    types = np.array([list(model["atomic_numbers"]).index(z) for z in s.numbers])
    for q, name in enumerate(("H1", "A1")):
        ev.set_adapters(name, *adapters_of(ev, name, 2, rank, q))
    ev.assign_adapters(np.arange(s.num_atoms, dtype=np.int32) % 2)
    args = (s.positions, types, s.cell, s.pbc)
    before, grads = ev.evaluate(*args), ev.adapter_gradients("A1")

    def same_results(out):
        np.testing.assert_array_equal(out[3], before[3])
        assert np.abs(out[0] - before[0]).max() <= min(1e-3, 1e-3 * np.abs(before[0]).max())

    ev.debug_expire_waits(2000)
    with pytest.raises(SymmetrixError, match="wait.*code 7") as err:
        ev.evaluate(*args)
    assert err.value.status == _lib.SMX_ERR_CUDA
    assert np.isnan(ev.get("H1")).all()
    for name in ("H1", "A1"):
        with pytest.raises(SymmetrixError, match="no evaluation"):
            ev.adapter_gradients(name)
    ev.debug_expire_waits(0)
    same_results(ev.evaluate(*args))
    # the pass of the gradients, which makes hidden rows only
    ev.debug_expire_waits(2000)
    with pytest.raises(SymmetrixError, match="wait.*code 7"):
        ev.adapter_gradients("A1")
    ev.debug_expire_waits(0)
    same_results(ev.evaluate(*args))
    again = ev.adapter_gradients("A1")
    for a, b in zip((*grads[0], *grads[1], grads[2]), (*again[0], *again[1], again[2])):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_check_of_a_linear(dtype):
    case = Case(dtype, [1, 3], [40, 40], [40, 40], 300, 2, 3, 5)
    layer, _, _, _ = everything(case)
    layer.check()
    layer._status.fill_(7)                      # what a kernel leaves there
    with pytest.raises(SymmetrixError, match="wait.*code 7") as err:
        layer.check()
    assert err.value.status == _lib.SMX_ERR_CUDA
    layer.check()
