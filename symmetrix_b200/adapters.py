"""Fine-tuned variants of one model side by side: rows routed to groups and back, and linears with low-rank adapters.

``RowRouting`` sorts the rows of per-atom arrays by group (``smx_route_*``), ``AdapterLinear`` is a channel-mixing linear of all degrees with
every atom's own low-rank adapter, or weighted mixture of adapters, beside the shared weights (``smx_adapter_*``). Both work on CUDA tensors
(float32 or float64) and issue their work on torch's current stream of the tensors' device. Nothing waits for the GPU, so both can be captured
into CUDA graphs (the first call of a kind on a GPU comes before a capture). They are not recorded by autograd: the backward passes are
methods, and inputs that require gradients are refused while torch records.

Rows may have any stride between atoms; other strides than one inside a row are copied first.
"""
from __future__ import annotations

import ctypes
import threading
from collections import namedtuple

from . import _lib
from .mace import SymmetrixError

AdapterGradients = namedtuple("AdapterGradients", ["x", "down", "up", "weights"])


class _Errors(threading.local):
    def __init__(self):
        self.buffer = ctypes.create_string_buffer(256)


_errors = _Errors()


def _call(fn, index: int, *args) -> None:
    """A call of the library on device `index` (the message of a failure goes to a buffer of the thread)."""
    import torch
    if torch.cuda.current_device() == index:
        status = fn(*args, _errors.buffer, 256)
    else:
        with torch.cuda.device(index):
            status = fn(*args, _errors.buffer, 256)
    if status != _lib.SMX_OK:
        raise SymmetrixError(status, _errors.buffer.value.decode())


def _stream(index: int) -> int:
    """The handle of torch's current stream on device `index`."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)       # without making a Stream object, a tenth of the time
    return raw(index) if raw is not None else torch.cuda.current_stream(index).cuda_stream


def _precision(dtype) -> int:
    import torch
    return _lib.SMX_FP32 if dtype is torch.float32 else _lib.SMX_FP64


def _ptr(t):
    return None if t is None else t.data_ptr()


def _values(t, what: str, shape, dtype=None, device=None):
    """`t` checked: a float32 / float64 CUDA tensor of the given shape (None: any extent)."""
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype is not dtype if dtype is not None else t.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"{what} has dtype {t.dtype}, expected {'float32 or float64' if dtype is None else dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")
    if t.shape != shape and (t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape))):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple('any' if n is None else n for n in shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires gradients, but this operator is not recorded by autograd: use torch.no_grad() and its backward method")
    return t


def _rows(t, what: str, shape, dtype=None, device=None):
    """(tensor, row stride) of a two-dimensional array of rows."""
    t = _values(t, what, shape, dtype, device)
    rows, step = t.stride()
    if step != 1 and t.shape[1] > 1:
        t = t.contiguous()
        rows = t.stride(0)
    return t, (rows if t.shape[0] > 1 else t.shape[1])


def _out(t, what: str, shape, dtype, device):
    t = _values(t, what, shape, dtype, device)
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what} must have rows of unit stride that do not overlap")
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _apart(out, *inputs) -> None:
    """Refuses an output that shares memory with an input (the kernels read and write in no fixed order)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    if out.numel() == 0:
        return
    a0, a1 = span(out)
    for t in inputs:
        if t is not None and t.numel():
            b0, b1 = span(t)
            if a0 < b1 and b0 < a1:
                raise ValueError("out shares memory with an input")


class RowRouting:
    """Rows sorted by group, and back. ``ids`` is an int32 CUDA tensor ``[rows]`` or ``[rows, slots]`` of groups in ``0 .. num_groups - 1``;
    any other value is an empty slot.

    ``order``, ``position`` and ``offsets`` are the plan of ``smx_route_plan`` (int32): the pair ``n * slots + s`` at every sorted position
    with the empty slots last, the position of every pair (-1: empty), and the first position of every group."""

    def __init__(self, ids, num_groups: int):
        import torch
        if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
            raise ValueError("ids must be a CUDA tensor")
        if ids.dtype != torch.int32:
            raise ValueError(f"ids has dtype {ids.dtype}, expected torch.int32")
        if ids.dim() not in (1, 2):
            raise ValueError("ids must have shape [rows] or [rows, slots]")
        self.num_rows, self.slots = ids.shape[0], ids.shape[1] if ids.dim() == 2 else 1
        self.num_groups, self.device = int(num_groups), ids.device
        self._library = _lib.load()
        # (checked here too: a C int would hold what is left of a larger number)
        need = self._library.smx_route_plan_bytes(self.num_rows, self.slots, self.num_groups) if 1 <= self.num_groups <= _lib.ROUTE_MAX_GROUPS else -1
        if need < 0:
            raise ValueError(f"{self.num_rows} rows with {self.slots} slots and {self.num_groups} groups: the limits are {_lib.ROUTE_MAX_SLOTS} slots, "
                             f"{_lib.ROUTE_MAX_GROUPS} groups and 2^31 - 2^11 pairs, and one slot and group at least")
        self._need, self._index = need, self.device.index
        self._pairs = self.num_rows * self.slots
        self._plan = ids.new_empty(2 * self._pairs + self.num_groups + 1)
        base = self._plan.data_ptr()
        self._order, self._position, self._offsets = base, base + 4 * self._pairs, base + 8 * self._pairs
        self._home = _stream(self._index)
        self._make(ids)

    @property
    def order(self):
        return self._plan[:self._pairs]

    @property
    def position(self):
        return self._plan[self._pairs:2 * self._pairs].view(self.num_rows, self.slots)

    @property
    def offsets(self):
        return self._plan[2 * self._pairs:]

    def update(self, ids) -> None:
        """The plan of other ids of the same shape, in the same tensors."""
        import torch
        if not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.device != self.device or ids.numel() != self._pairs \
                or ids.dim() not in (1, 2) or ids.shape[0] != self.num_rows:
            raise ValueError(f"ids must be an int32 tensor of {self.num_rows} rows with {self.slots} slots on {self.device}")
        self._make(ids)

    def _make(self, ids):
        import torch
        ids = ids.contiguous()
        ws = torch.empty(self._need, dtype=torch.uint8, device=self.device) if self._need else None
        _call(self._library.smx_route_plan, self._index, ids.data_ptr(), self.num_rows, self.slots, self.num_groups, self._order, self._position,
              self._offsets, _ptr(ws), self._need, self._use())

    def _use(self) -> int:
        """The current stream; the plan's memory stays until its work is done there, wherever the plan was made."""
        handle = _stream(self._index)
        if handle != self._home:
            import torch
            self._plan.record_stream(torch.cuda.current_stream(self._index))
        return handle

    def _weights(self, weights, dtype):
        if weights is None:
            return None
        shape = (self.num_rows,) if self.slots == 1 and getattr(weights, "ndim", 2) == 1 else (self.num_rows, self.slots)
        return _values(weights, "weights", shape, dtype, self.device).contiguous()

    def dispatch(self, x, out=None):
        """``[rows * slots, width]``: every row of ``x`` once per group it goes to, in sorted order. Rows behind the last group are zero, or
        left as they were in ``out``."""
        x, stride = _rows(x, "x", (self.num_rows, None), None, self.device)
        shape = (self._pairs, x.shape[1])
        if out is None:
            rows = x.new_empty(shape)
        else:
            rows = _out(out, "out", shape, x.dtype, self.device)[0]
            if not rows.is_contiguous():
                raise ValueError("out must be contiguous")
            _apart(rows, x)
        _call(self._library.smx_route_dispatch, self._index, _precision(x.dtype), x.data_ptr(), stride, self.num_rows, self.slots, shape[1],
              self._position, self._offsets, self.num_groups, rows.data_ptr(), int(out is None), self._use())
        return rows

    def combine(self, rows, weights=None, base=None, out=None):
        """``base + sum_s weights[:, s] * rows[position[:, s]]`` (weights None: ones; base None: zero; ``out`` may be ``base``)."""
        rows = _values(rows, "rows", (self._pairs, None), None, self.device).contiguous()
        width, dtype = rows.shape[1], rows.dtype
        weights = self._weights(weights, dtype)
        base, base_stride = (None, 0) if base is None else _rows(base, "base", (self.num_rows, width), dtype, self.device)
        if out is None:
            y, y_stride = rows.new_empty((self.num_rows, width)), width
        else:
            y, y_stride = _out(out, "out", (self.num_rows, width), dtype, self.device)
            _apart(y, rows, weights, None if base is not None and base.data_ptr() == y.data_ptr() and base_stride == y_stride else base)
        _call(self._library.smx_route_combine, self._index, _precision(dtype), rows.data_ptr(), self._position, self.num_rows, self.slots, width,
              _ptr(weights), _ptr(base), base_stride, y.data_ptr(), y_stride, self._use())
        return y

    def dispatch_backward(self, grad_rows):
        """The gradient of ``dispatch``'s input: the sum of the gradients of its copies."""
        return self.combine(grad_rows)

    def combine_backward(self, grad_y, rows=None, weights=None):
        """(gradient of ``rows``, gradient of ``weights``) of ``combine``; the latter is None without ``rows``. The gradient of ``base`` is
        ``grad_y``."""
        grad_y, stride = _rows(grad_y, "grad_y", (self.num_rows, None), None, self.device)
        width, dtype = grad_y.shape[1], grad_y.dtype
        weights = self._weights(weights, dtype)
        if rows is not None:
            rows = _values(rows, "rows", (self._pairs, width), dtype, self.device).contiguous()
        grad_rows = grad_y.new_empty((self._pairs, width))
        grad_weights = None if rows is None else grad_y.new_empty((self.num_rows, self.slots))
        _call(self._library.smx_route_combine_backward, self._index, _precision(dtype), grad_y.data_ptr(), stride, _ptr(rows), self._position,
              self._offsets, self.num_groups, self.num_rows, self.slots, width, _ptr(weights), grad_rows.data_ptr(), _ptr(grad_weights), 1, self._use())
        return grad_rows, grad_weights


class AdapterLinear:
    """A linear of all degrees with low-rank adapters: ``y = x shared_l + sum_s w_s (x down_l[g_s]) up_l[g_s]`` for every component.

    ``shared``, ``down`` and ``up`` are lists with a tensor per degree: ``[in_l, out_l]``, ``[adapters, in_l, rank]`` and
    ``[adapters, rank, out_l]``; ``components`` the rows per atom of every degree (default 1, 3, 5, ...). An atom's row of ``x`` holds the
    components of degree 0, then those of degree 1, and so on, ``in_l`` channels each; ``y`` the same with ``out_l``. A factor in front of the
    adapters belongs into ``up``. ``shared`` may be None: adapters alone.

    The matrices are copied into the kernels' layout: after changing values in place, call ``set_adapters`` / ``set_shared`` again."""

    def __init__(self, shared, down, up, components=None):
        import torch
        down, up = list(down), list(up)
        if not down or len(down) > _lib.ADAPTER_MAX_DEGREES or len(up) != len(down) or (shared is not None and len(shared) != len(down)):
            raise ValueError(f"shared, down and up need one matrix for each of 1 .. {_lib.ADAPTER_MAX_DEGREES} degrees")
        first = _values(down[0], "down[0]", (None, None, None))
        self.dtype, self.device = first.dtype, first.device
        self.num_adapters, self.rank = first.shape[0], first.shape[2]
        if not 1 <= self.rank <= _lib.ADAPTER_MAX_RANK or not 1 <= self.num_adapters <= _lib.ROUTE_MAX_GROUPS:
            raise ValueError(f"down[0] has shape {tuple(first.shape)}: 1 .. {_lib.ROUTE_MAX_GROUPS} adapters of rank 1 .. {_lib.ADAPTER_MAX_RANK} are supported")
        self.components = [2 * l + 1 for l in range(len(down))] if components is None else [int(c) for c in components]
        if len(self.components) != len(down) or any(not 1 <= c <= 1024 for c in self.components):
            raise ValueError("components needs a number in 1 .. 1024 for each degree")
        self.in_channels, self.out_channels = [a.shape[1] for a in down], [b.shape[2] for b in up]
        if any(not 1 <= n <= 1 << 20 for n in self.in_channels + self.out_channels):
            raise ValueError("a degree needs 1 .. 1048576 channels")
        self.in_width = sum(c * i for c, i in zip(self.components, self.in_channels))
        self.out_width = sum(c * o for c, o in zip(self.components, self.out_channels))
        self._library = _lib.load()
        self._has_shared = shared is not None
        self._fixed = _lib.AdapterCall()
        f = self._fixed
        f.precision, f.num_degrees, f.num_groups, f.rank = _precision(self.dtype), len(down), self.num_adapters, self.rank
        f.slots = 1
        for d, c, i, o in zip(f.degrees, self.components, self.in_channels, self.out_channels):
            d.components, d.in_channels, d.out_channels = c, i, o
            d.shared = 1 if self._has_shared else None          # only whether there is one counts, except in smx_adapter_prepare
        need = self._library.smx_adapter_tiles_bytes(ctypes.byref(f))
        if need < 0:
            raise ValueError("the sizes exceed what smx_adapter_forward supports")
        self._index = self.device.index
        self._home = _stream(self._index)
        self._tiles = torch.empty(need + 16, dtype=torch.uint8, device=self.device)
        self._status = self._tiles[need:need + 4].view(torch.int32)
        self._status.zero_()
        f.tiles, f.status = self._tiles.data_ptr(), self._status.data_ptr()
        self.set_adapters(down, up)
        if self._has_shared:
            self.set_shared(shared)

    # ------------------------------------------------------------------ matrices
    def _prepare(self, parts, shared, down, up):
        call = self._copy()
        for q in range(call.num_degrees):
            d = call.degrees[q]
            d.shared, d.down, d.up = _ptr(shared[q]) if shared else d.shared, _ptr(down[q]) if down else None, _ptr(up[q]) if up else None
        call.stream = self._use()
        _call(self._library.smx_adapter_prepare, self._index, ctypes.byref(call), parts)

    def set_adapters(self, down, up) -> None:
        """Other values of the adapters, of the same shapes."""
        n = len(self.components)
        if len(down) != n or len(up) != n:
            raise ValueError(f"down and up need {n} matrices")
        down = [_values(a, f"down[{q}]", (self.num_adapters, self.in_channels[q], self.rank), self.dtype, self.device).contiguous() for q, a in enumerate(down)]
        up = [_values(b, f"up[{q}]", (self.num_adapters, self.rank, self.out_channels[q]), self.dtype, self.device).contiguous() for q, b in enumerate(up)]
        self._prepare(_lib.ADAPTER_MATRICES, None, down, up)

    def set_shared(self, shared) -> None:
        """Other values of the shared weights, of the same shapes."""
        if not self._has_shared:
            raise ValueError("the linear was made without shared weights")
        if len(shared) != len(self.components):
            raise ValueError(f"shared needs {len(self.components)} matrices")
        shared = [_values(w, f"shared[{q}]", (self.in_channels[q], self.out_channels[q]), self.dtype, self.device).contiguous() for q, w in enumerate(shared)]
        self._prepare(_lib.ADAPTER_SHARED, shared, None, None)

    # ------------------------------------------------------------------ calls
    def check(self) -> None:
        """Waits for the current stream and raises ``SymmetrixError`` if a bounded wait inside a kernel ran out in a call since the last check:
        what such a call lost holds NaN. (Calls themselves never wait, so they cannot tell.)"""
        code = int(self._status.item())
        if code:
            self._status.zero_()
            raise SymmetrixError(_lib.SMX_ERR_CUDA, f"a bounded wait ran out in a device kernel (code {code}); results are invalid")

    def _copy(self):
        call = _lib.AdapterCall()
        ctypes.memmove(ctypes.byref(call), ctypes.byref(self._fixed), ctypes.sizeof(call))
        return call

    def _use(self) -> int:
        handle = _stream(self._index)
        if handle != self._home:
            import torch
            self._tiles.record_stream(torch.cuda.current_stream(self._index))
        return handle

    def _begin(self, routing, weights):
        if not isinstance(routing, RowRouting):
            raise ValueError("routing must be a RowRouting")
        if routing.device != self.device:
            raise ValueError(f"routing is on {routing.device}, expected {self.device}")
        if routing.num_groups != self.num_adapters:
            raise ValueError(f"routing has {routing.num_groups} groups, the linear {self.num_adapters} adapters")
        weights = routing._weights(weights, self.dtype)
        call = self._copy()
        call.num_rows, call.slots = routing.num_rows, routing.slots
        call.order, call.position, call.offsets = routing._order, routing._position, routing._offsets
        call.weights = _ptr(weights)
        return call, weights

    def _run(self, fn, call, backward, routing):
        need = self._library.smx_adapter_workspace_bytes(ctypes.byref(call), backward)
        if need < 0:
            raise ValueError("the sizes exceed what smx_adapter_forward supports")
        ws = self._tiles.new_empty(need) if need else None
        call.workspace, call.workspace_bytes = _ptr(ws), need
        call.stream = self._use()
        if call.stream != routing._home:
            routing._use()
        _call(fn, self._index, ctypes.byref(call))

    def forward(self, x, routing: RowRouting, weights=None, out=None, keep_hidden: bool = False):
        """``y``, or ``(y, hidden)`` with ``keep_hidden``: the products ``x down`` of every pair, for ``backward``."""
        call, weights = self._begin(routing, weights)
        x, call.x_stride = _rows(x, "x", (routing.num_rows, self.in_width), self.dtype, self.device)
        if out is None:
            y, call.y_stride = x.new_empty((routing.num_rows, self.out_width)), self.out_width
        else:
            y, call.y_stride = _out(out, "out", (routing.num_rows, self.out_width), self.dtype, self.device)
            _apart(y, x, weights)
        call.x, call.y = _ptr(x), _ptr(y)
        hidden = None
        if keep_hidden:
            hidden = x.new_empty(self._library.smx_adapter_hidden_elements(ctypes.byref(call)))
            call.hidden = _ptr(hidden) if hidden.numel() else None
        self._run(self._library.smx_adapter_forward, call, 0, routing)
        return (y, hidden) if keep_hidden else y

    def backward(self, x, grad_y, routing: RowRouting, weights=None, hidden=None, want_x: bool = True, want_adapters: bool = True, want_weights: bool = True):
        """Gradients ``(x, down, up, weights)`` of a forward pass with the same ``x``, routing and weights, None where not wanted. ``hidden`` of
        that pass saves computing it again. The shared weights are frozen."""
        call, weights = self._begin(routing, weights)
        n, dev, dt = routing.num_rows, self.device, self.dtype
        x, call.x_stride = _rows(x, "x", (n, self.in_width), dt, dev)
        grad_y, call.grad_y_stride = _rows(grad_y, "grad_y", (n, self.out_width), dt, dev)
        call.x, call.grad_y = _ptr(x), _ptr(grad_y)
        if hidden is not None:
            hidden = _values(hidden, "hidden", (self._library.smx_adapter_hidden_elements(ctypes.byref(call)),), dt, dev).contiguous()
            if hidden.data_ptr() % 16:
                hidden = hidden.clone()
            call.hidden = _ptr(hidden) if hidden.numel() else None
        grad_x = grad_down = grad_up = grad_weights = None
        if want_x:
            grad_x = x.new_empty((n, self.in_width))
            call.grad_x, call.grad_x_stride = _ptr(grad_x), self.in_width
        if want_adapters:
            # one allocation for all degrees: half the time of one each
            g, r, at, grad_down, grad_up = self.num_adapters, self.rank, 0, [], []
            flat = x.new_empty(g * r * (sum(self.in_channels) + sum(self.out_channels)))
            base, size = flat.data_ptr(), flat.element_size()
            for d, i, o in zip(call.degrees, self.in_channels, self.out_channels):
                d.grad_down, d.grad_up = base + size * at, base + size * (at + g * i * r)
                grad_down.append(flat.as_strided((g, i, r), (i * r, r, 1), at))
                grad_up.append(flat.as_strided((g, r, o), (r * o, o, 1), at + g * i * r))
                at += g * r * (i + o)
        if want_weights:
            grad_weights = x.new_empty((n, routing.slots))
            call.grad_weights = _ptr(grad_weights) if grad_weights.numel() else None
        self._run(self._library.smx_adapter_backward, call, 1, routing)
        return AdapterGradients(grad_x, grad_down, grad_up, grad_weights)
