"""Embeddings: rows of a table named by tokens (elements, or pairs of a fine-tuned variant and an element), weighted, with their gradients.

``Embedding`` (``smx_embedding_*``) looks rows up, ``EmbeddingPlan`` sorts the tokens of a batch for the gradient of the table. Both work on CUDA tensors
(float32 or float64) and on torch's current stream of their device, wait for nothing, can be captured into CUDA graphs (after a first call
of a kind on a GPU) and are not recorded by autograd: the backward pass is a method.
"""
from __future__ import annotations

from collections import namedtuple

from . import _lib
from .adapters import _apart, _call, _not_of_plan, _out, _precision, _ptr, _rows, _stream, _values

EmbeddingGradients = namedtuple("EmbeddingGradients", ["table", "weights"])


def _tokens(ids, device=None):
    """(ids, rows, slots) of an int32 CUDA tensor ``[rows]`` or ``[rows, slots]``."""
    import torch
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
        raise ValueError("ids must be a CUDA tensor")
    if ids.dtype != torch.int32:
        raise ValueError(f"ids has dtype {ids.dtype}, expected torch.int32")
    if ids.dim() not in (1, 2):
        raise ValueError("ids must have shape [rows] or [rows, slots]")
    if device is not None and ids.device != device:
        raise ValueError(f"ids is on {ids.device}, expected {device}")
    return ids.contiguous(), ids.shape[0], ids.shape[1] if ids.dim() == 2 else 1


def _weights(weights, rows, slots, dtype, device):
    if weights is None:
        return None
    shape = (rows,) if slots == 1 and getattr(weights, "ndim", 2) == 1 else (rows, slots)
    return _values(weights, "weights", shape, dtype, device).contiguous()


class EmbeddingPlan:
    """The pairs (row, slot) of ``ids`` sorted by token: ``order`` holds the pair ``n * slots + s`` at every sorted position, ``tokens`` its token
    (``table_rows``: none; these come last), both int32. ``ids`` is an int32 CUDA tensor ``[rows]`` or ``[rows, slots]`` of rows of the table; any
    other value is an empty slot."""

    def __init__(self, ids, table_rows: int):
        ids, self.num_rows, self.slots = _tokens(ids)
        self.table_rows, self.device = int(table_rows), ids.device
        self._library = _lib.load()
        # (checked here too: a C int would hold what is left of a larger number)
        need = self._library.smx_embedding_plan_bytes(self.num_rows, self.slots, self.table_rows) if 1 <= self.table_rows <= _lib.EMBEDDING_MAX_ROWS else -1
        if need < 0:
            raise ValueError(f"{self.num_rows} rows with {self.slots} slots and a table of {self.table_rows} rows: the limits are {_lib.ROUTE_MAX_SLOTS} slots, "
                             f"{_lib.EMBEDDING_MAX_ROWS} table rows and 2^31 - 2^11 pairs, and one slot and table row at least")
        self._need, self._index, self._pairs = need, self.device.index, self.num_rows * self.slots
        self._plan = ids.new_empty(2 * self._pairs)
        self._order = self._plan.data_ptr()
        self._sorted = self._order + 4 * self._pairs
        self._home = _stream(self._index)
        self._make(ids)

    @property
    def order(self):
        return self._plan[:self._pairs]

    @property
    def tokens(self):
        return self._plan[self._pairs:]

    def update(self, ids) -> None:
        """The plan of other ids of the same shape, in the same tensors (of which `ids` must not be a part)."""
        ids, rows, slots = _tokens(ids, self.device)
        if (rows, slots) != (self.num_rows, self.slots):
            raise ValueError(f"ids must have {self.num_rows} rows with {self.slots} slots")
        self._make(_not_of_plan(ids, self._plan))

    def _make(self, ids):
        import torch
        ws = torch.empty(self._need, dtype=torch.uint8, device=self.device) if self._need else None
        _call(self._library.smx_embedding_plan, self._index, ids.data_ptr(), self.num_rows, self.slots, self.table_rows, self._order, self._sorted,
              _ptr(ws), self._need, self._use())

    def _use(self) -> int:
        """The current stream; the plan's memory stays until its work is done there, wherever the plan was made."""
        handle = _stream(self._index)
        if handle != self._home:
            import torch
            self._plan.record_stream(torch.cuda.current_stream(self._index))
        return handle


class Embedding:
    """Rows of ``table`` ``[table_rows, width]`` named by tokens: ``y[n] = scale * sum_s weights[n, s] * table[ids[n, s]]``.

    The tensor itself is kept and read in every call: values changed in place count from the next call on. Its rows may have any stride between
    them, inside a row it must be one."""

    def __init__(self, table, scale: float = 1.0):
        table = _values(table, "table", (None, None))
        if not 1 <= table.shape[0] <= _lib.EMBEDDING_MAX_ROWS:
            raise ValueError(f"table has shape {tuple(table.shape)}: 1 .. {_lib.EMBEDDING_MAX_ROWS} rows are supported")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("table must have rows of unit stride")
        self.table, self.scale = table, float(scale)
        self.table_rows, self.width = table.shape
        self.dtype, self.device = table.dtype, table.device
        self._shape, self._strides = tuple(table.shape), table.stride()
        self._stride = self._strides[0] if self.table_rows > 1 else self.width
        self._library, self._index, self._precision = _lib.load(), self.device.index, _precision(table.dtype)

    def _check(self):
        t = self.table
        if t.requires_grad or t.shape != self._shape or t.dtype is not self.dtype or t.get_device() != self._index:
            _values(t, "table", self._shape, self.dtype, self.device)
        if t.stride() != self._strides:
            raise ValueError("table has other strides than when the embedding was made")

    def forward(self, ids, weights=None, out=None):
        """``y`` ``[rows, width]``; ``ids`` as for ``EmbeddingPlan``, ``weights`` ``[rows, slots]`` (None: ones)."""
        self._check()
        ids, rows, slots = _tokens(ids, self.device)
        if not 1 <= slots <= _lib.ROUTE_MAX_SLOTS:
            raise ValueError(f"ids has {slots} slots: 1 .. {_lib.ROUTE_MAX_SLOTS} are supported")
        weights = _weights(weights, rows, slots, self.dtype, self.device)
        if out is None:
            y, stride = self.table.new_empty((rows, self.width)), self.width
        else:
            y, stride = _out(out, "out", (rows, self.width), self.dtype, self.device)
            _apart(y, self.table, ids, weights)
        _call(self._library.smx_embedding_forward, self._index, self._precision, self.table.data_ptr(), self._stride, self.table_rows, ids.data_ptr(), rows, slots,
              self.width, _ptr(weights), self.scale, y.data_ptr(), stride, _stream(self._index))
        return y

    def backward(self, grad_y, plan: EmbeddingPlan, weights=None, want_table: bool = True, want_weights: bool = True):
        """Gradients ``(table, weights)`` of a forward pass with the plan's ids and the same weights, None where not wanted: ``[table_rows, width]``,
        zero for rows without a token, and ``[rows, slots]``, zero in empty slots."""
        import torch
        self._check()
        if not isinstance(plan, EmbeddingPlan):
            raise ValueError("plan must be an EmbeddingPlan")
        if plan.device != self.device:
            raise ValueError(f"plan is on {plan.device}, expected {self.device}")
        if plan.table_rows != self.table_rows:
            raise ValueError(f"plan is of a table of {plan.table_rows} rows, the embedding's has {self.table_rows}")
        rows, slots = plan.num_rows, plan.slots
        grad_y, stride = _rows(grad_y, "grad_y", (rows, self.width), self.dtype, self.device)
        weights = _weights(weights, rows, slots, self.dtype, self.device)
        grad_table = self.table.new_empty((self.table_rows, self.width)) if want_table else None
        grad_weights = self.table.new_empty((rows, slots)) if want_weights else None
        need = self._library.smx_embedding_backward_bytes(self._precision, rows, slots, self.width)
        if need < 0:
            raise ValueError("the sizes exceed what smx_embedding_backward supports")
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _call(self._library.smx_embedding_backward, self._index, self._precision, grad_y.data_ptr(), stride, self.table.data_ptr(), self._stride, self.table_rows,
              plan._order, plan._sorted, rows, slots, self.width, _ptr(weights), self.scale, _ptr(grad_table), _ptr(grad_weights), _ptr(ws), need, plan._use())
        return EmbeddingGradients(grad_table, grad_weights)
