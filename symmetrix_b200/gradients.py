"""The common norm of many tensors, and their scaling to at most a given norm: what training does with all gradients before a step.

Works on CUDA tensors (float32 and float64, also mixed) of one device and on torch's current stream there (``smx_gradient_*``). Nothing waits:
the norm is a float64 tensor on the device, so the calls can be captured into CUDA graphs.
"""
from __future__ import annotations

from . import _lib
from .adapters import _call, _precision, _stream


def _dense(t, what: str, device):
    """`t` checked: a float32 / float64 CUDA tensor whose values lie next to one another."""
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype is not torch.float32 and t.dtype is not torch.float64:
        raise ValueError(f"{what} has dtype {t.dtype}, expected float32 or float64")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires gradients, but this operator is not recorded by autograd: use torch.no_grad()")
    return t


class GradientSet:
    """Tensors with a common norm. ``tensors`` is a list of contiguous CUDA tensors, float32 or float64 each; ``out`` (a list of the same shapes and types)
    receives the scaled values, the tensors themselves without it. Nothing in the lists may overlap, except an output with its own tensor
    where both are the same memory.

    The set holds on to the tensors' memory as it is when the set is made: a program whose gradients have buffers of their own makes it once. That memory must stay theirs: a
    tensor whose storage is resized afterwards needs another set."""

    def __init__(self, tensors, out=None):
        tensors = list(tensors)
        outs = None if out is None else list(out)
        if not tensors:
            raise ValueError("a set needs at least one tensor")
        if outs is not None and len(outs) != len(tensors):
            raise ValueError(f"out has {len(outs)} tensors, expected {len(tensors)}")
        self.device = None
        spans, entries = [], (_lib.Gradient * len(tensors))()
        for q, t in enumerate(tensors):
            # (another tensor of the same memory, which stays even if the program gives this one other memory)
            tensors[q] = t = _dense(t, f"tensors[{q}]", self.device).detach()
            self.device = t.device
            e, at, size = entries[q], t.data_ptr(), t.element_size() * t.numel()
            e.values, e.out, e.count, e.precision = at, at, t.numel(), _precision(t.dtype)
            spans.append((at, at + size))
            if outs is None:
                continue
            outs[q] = o = _dense(outs[q], f"out[{q}]", self.device).detach()
            if o.shape != t.shape or o.dtype is not t.dtype:
                raise ValueError(f"out[{q}] has shape {tuple(o.shape)} and dtype {o.dtype}, expected {tuple(t.shape)} and {t.dtype}")
            e.out = o.data_ptr()
            if o.data_ptr() != at:
                spans.append((o.data_ptr(), o.data_ptr() + size))
        spans = sorted(s for s in spans if s[0] < s[1])
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("tensors and out must not share memory")
        self.tensors, self.out = tuple(tensors), tuple(tensors if outs is None else outs)
        self._entries, self._library, self._index = entries, _lib.load(), self.device.index
        self._need = self._library.smx_gradient_workspace_bytes(entries, len(entries))
        if self._need < 0:
            raise ValueError("a tensor exceeds 2^40 values")

    def norm(self):
        """The square root of the sum of the squares of all values: a float64 tensor without dimensions."""
        import torch
        # the norm, and the partial sums behind it
        buffer = torch.empty(1 + self._need // 8, dtype=torch.float64, device=self.device)
        at = buffer.data_ptr()
        _call(self._library.smx_gradient_norm, self._index, self._entries, len(self._entries), at, at + 8, self._need, _stream(self._index))
        return buffer[0]

    def clip(self, max_norm: float):
        """Multiplies the tensors by ``max_norm / norm`` unless the norm is ``max_norm`` or less (into ``out``, which then receives copies) and returns the
        norm before that. A NaN among the values makes the norm and all results NaN; an infinite norm (infinities, float64 values from 1e154 on) makes finite values zero."""
        import torch
        max_norm = float(max_norm)
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm is {max_norm}: it must not be negative or NaN")
        buffer = torch.empty(1 + self._need // 8, dtype=torch.float64, device=self.device)
        at = buffer.data_ptr()
        _call(self._library.smx_gradient_clip, self._index, self._entries, len(self._entries), max_norm, at, at + 8, self._need, _stream(self._index))
        return buffer[0]


def gradient_norm(tensors):
    """The common norm of ``tensors``, see ``GradientSet.norm``."""
    return GradientSet(tensors).norm()


def clip_gradients(tensors, max_norm: float, out=None):
    """Scales ``tensors`` to a common norm of at most ``max_norm``, see ``GradientSet.clip``; returns the norm before that."""
    return GradientSet(tensors, out).clip(max_norm)
