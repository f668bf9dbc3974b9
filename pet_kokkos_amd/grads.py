"""A model's gradients as one: their norm, and clipping by it.

What a training step does between the backward (``layer.norm_rows_grads``,
``linear.linear_grads``, ``layer.attention_layer_grads``) and the update. The
reference evaluates and does not train, so it has no counterpart. Tensors are
float32, bfloat16 or float16, mixed as they come; the sums run in double on the
device in a fixed order, the factor stays there, and nothing synchronises. All
work runs in libpet_attn.so on the current torch stream.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .attention import DTYPES, _call_on, _scratch


class GradList:
    """The tensors of a step's gradients, checked and laid out for the library
    once: contiguous in any order of their axes, or a 2-D view of rows (or a column) in
    a wider matrix; all on one device, no two overlapping (different columns of one
    matrix do not). It keeps the memory that they have now, and every call reads what
    that then holds (a gradient set anew needs a new list: 3.3 us a tensor on the
    host)."""

    def __init__(self, tensors):
        self.tensors, self.device = [], None
        entries, spans = [], []
        for i, t in enumerate(tensors):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"gradient {i}: a torch tensor is needed")
            if t.device.type != "cuda" or (self.device is not None and t.device != self.device):
                raise ValueError(f"gradient {i}: on {t.device}, the first is on {self.device}")
            if t.dtype not in DTYPES:
                raise ValueError(f"gradient {i}: {t.dtype}, not float32, bfloat16 or float16")
            self.device = t.device
            t = t.detach()  # (its memory, whatever becomes of the caller's tensor)
            self.tensors.append(t)
            if t.numel() == 0:
                continue
            rows, cols, ld = _layout(t, i)
            entries.append((t.data_ptr(), rows, cols, ld, DTYPES[t.dtype]))
            spans.append((t.data_ptr(), t.data_ptr() + ((rows - 1) * ld + cols) * t.element_size(), i, t))
        spans.sort(key=lambda s: s[0])
        live = []  # the spans that reach past the next one's start
        for span in spans:
            live = [s for s in live if s[1] > span[0]]
            for _, _, i, t in live:
                if not _side_by_side(t, span[3]):
                    raise ValueError(f"gradients {min(i, span[2])} and {max(i, span[2])} overlap")
            live.append(span)
        self.array = (_lib.GradTensor * max(1, len(entries)))(*[_lib.GradTensor(*e) for e in entries])
        self.count = len(entries)
        self.scratch_bytes = _lib.load().pet_grad_workspace(self.count)


def _layout(t: torch.Tensor, i: int):
    """(rows, columns, leading dimension) of a tensor whose elements are
    consecutive in some order of its axes, or a 2-D view of rows."""
    axes = sorted((a for a in range(t.dim()) if t.shape[a] > 1), key=lambda a: t.stride(a))
    step = 1
    for a in axes:
        if t.stride(a) != step:
            break
        step *= t.shape[a]
    else:
        return 1, t.numel(), t.numel()
    if len(axes) == 1 and t.stride(axes[0]) > 0:
        return t.shape[axes[0]], 1, t.stride(axes[0])
    if len(axes) == 2 and t.stride(axes[0]) == 1 and t.stride(axes[1]) >= t.shape[axes[0]]:
        return t.shape[axes[1]], t.shape[axes[0]], t.stride(axes[1])
    raise ValueError(f"gradient {i}: strides {tuple(t.stride())} of shape {tuple(t.shape)}: contiguous elements, or "
                     "rows of a wider matrix, are needed")


def _side_by_side(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views whose spans overlap are different columns of one matrix: their
    rows lie whole multiples of the leading dimensions' common divisor apart, so
    columns that are apart modulo that never meet."""
    (rows_a, cols_a, ld_a), (rows_b, cols_b, ld_b) = _layout(a, 0), _layout(b, 1)
    wide_a, wide_b = cols_a * a.element_size(), cols_b * b.element_size()
    step = math.gcd(ld_a * a.element_size() if rows_a > 1 else 0, ld_b * b.element_size() if rows_b > 1 else 0)
    gap = (b.data_ptr() - a.data_ptr()) % step if step else 0
    return gap >= wide_a and gap + wide_b <= step


def _arguments(grads, norm_type, scale):
    if not isinstance(grads, GradList):
        grads = GradList(grads)
    p = {1.0: 1, 2.0: 2, math.inf: 0}.get(float(norm_type))
    if p is None:
        raise ValueError(f"norm_type {norm_type}: 1, 2 or infinity")
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}: a finite number is needed")
    return grads, p


def _out(out, device):
    if out is None:
        return torch.empty((), dtype=torch.float32, device=device)
    if not isinstance(out, torch.Tensor):
        raise TypeError("out: a torch tensor is needed")
    if out.device != device or out.dtype != torch.float32 or out.numel() != 1:
        raise ValueError(f"out must be one float32 on {device}")
    return out


def grad_norm(grads, norm_type: float = 2.0, scale: float = 1.0, out: torch.Tensor | None = None,
              scratch: torch.Tensor | None = None) -> torch.Tensor:
    """|scale| (sum over every element of |g|^p)^(1/p) as a device float32 (into
    ``out`` where given), p = norm_type 1, 2 or infinity. ``grads``: a GradList, or
    tensors to make one of. ``scratch``: GradList.scratch_bytes, else allocated."""
    grads, p = _arguments(grads, norm_type, scale)
    dev = grads.device or torch.device("cuda", torch.cuda.current_device())
    out, scratch = _out(out, dev), _scratch(scratch, grads.scratch_bytes, dev)
    _call_on(dev, "pet_grad_norm", _lib.load().pet_grad_norm, grads.array, grads.count, p, float(scale),
             out.data_ptr(), scratch.data_ptr(), scratch.numel() * scratch.element_size())
    return out


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, scale: float = 1.0, eps: float = 1e-6,
               out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """grad_norm, and every gradient times scale min(1, max_norm / (norm + eps))
    in place; returns the norm before clipping. ``scale`` undoes a loss's scale or
    averages over micro-batches. An infinite norm leaves 0 (NaN where a gradient is
    infinite), a NaN leaves NaN."""
    grads, p = _arguments(grads, norm_type, scale)
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise ValueError(f"max_norm {max_norm}, eps {eps}: at least 0 is needed")
    dev = grads.device or torch.device("cuda", torch.cuda.current_device())
    out, scratch = _out(out, dev), _scratch(scratch, grads.scratch_bytes, dev)
    _call_on(dev, "pet_grad_clip", _lib.load().pet_grad_clip, grads.array, grads.count, p, float(scale),
             float(max_norm), float(eps), out.data_ptr(), scratch.data_ptr(),
             scratch.numel() * scratch.element_size())
    return out
