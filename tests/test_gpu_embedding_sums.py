"""Long sums of the embeddings' gradients in float32, of values whose roundings all point the same way: the error counts the roundings of a chunk, not of the whole sum.

A product w g is rounded once. Inside a chunk of up to 512 pairs a run is added up by at most 8 roundings (a batch of eight), 64 (the batches) and 16 (pairs before the first and behind the
last whole batch); what crosses chunks is added in 64 bits and rounded once. With unit roundoff u that is at most (1 + 8 + 64 + 16 + 1) u sum |w g|, whatever the number of pairs:
BOUND. A dot product over a row: at most 4 + 5 + 4 roundings inside a CTA's share of the row, two factors, and one at the end."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import Embedding, EmbeddingPlan

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BOUND, DOT_BOUND = 90 * U, 16 * U


@pytest.mark.parametrize("width", [64, 63])
@pytest.mark.parametrize("pairs", [512, 1000000])
def test_a_frequent_token(width, pairs):
    # one value a column, a little above one: added to a sum of some hundreds it loses the same part of its last bits every time
    v = (1 + np.random.default_rng(5).integers(1, 2 ** 15, width) * 2.0 ** -23).astype(np.float32)
    gy = torch.as_tensor(v).cuda().expand(pairs, width)
    ids = torch.zeros(pairs, dtype=torch.int32, device="cuda")
    ids[pairs // 2] = 1
    table = torch.zeros(3, width, device="cuda")
    got = Embedding(table).backward(gy, EmbeddingPlan(ids, 3), want_weights=False).table.double().cpu().numpy()
    want = np.outer([pairs - 1, 1, 0], v.astype(np.float64))
    assert np.all(np.abs(got - want) <= BOUND * want), np.max(np.abs(got[0] - want[0]) / want[0]) / U


@pytest.mark.parametrize("width", [1, 130, 520, 200000, 200001])
def test_a_wide_row(width):
    v = np.float32(1 + 19661 * 2.0 ** -23)
    gy = torch.full((3, width), float(v), device="cuda")
    ids = torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda")
    got = Embedding(torch.ones(2, width, device="cuda")).backward(gy, EmbeddingPlan(ids, 2), want_table=False).weights.double().cpu().numpy()
    want = float(v) * width
    assert np.all(np.abs(got - want) <= DOT_BOUND * want), np.max(np.abs(got - want)) / want / U
