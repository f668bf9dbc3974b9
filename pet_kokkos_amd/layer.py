"""The attention's input side over torch device tensors: the cf_seq bias
source, the token norm and the layer-level attention of a PET block.

``norm_rows`` / ``norm_rows_bwd`` mirror the reference's norm_rows /
norm_rows_bwd (src/ops.hpp:376-436): RMSNorm, or LayerNorm when a bias is
given; ``cf_seq`` its pet_cfseq pass (src/device_neighbors.cpp:318-323);
``attention_layer`` / ``attention_layer_bwd`` the attention block of
PetModel::ff_layer / ff_layer_bwd (src/feedforward.cpp:96-123, :292-329):
tokens -> norm -> qkv = linear(., W_in, b_in) -> attention, and back to the
tokens' adjoint (atom rows set, live edge rows accumulated).

For training, which the reference does not do: the norms take rows in bfloat16
and float16 and up to 16384 columns, ``norm_rows_grads`` makes the norm's
parameters' gradients with its input's adjoint, and ``attention_layer_grads``
the gradients of every parameter of an attention block with its backward. All
work runs in libpet_attn.so on the current torch stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import (DTYPES, Tokens, Workspace, _call_on, _live, _mat, _ptr, _scratch, _stream, _typed, _vector,
                        _weight, shape)

MAX_WIDTH = 16384  # PET_NORM_MAX_WIDTH


def cf_seq(off: torch.Tensor, cut: torch.Tensor, N: int, S: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """cf_seq [N, S]: 1 for the atom's own slot, its kept edges' cutoff factors
    (``cut``, packed order), 0 past its count."""
    lib = _lib.load()
    out = torch.empty((N, S), dtype=torch.float32, device=off.device) if out is None else out
    T = N + (int(cut.numel()) if cut is not None else 0)
    sh = _lib.Shape(N, T, S, 1, 16, 0, 1.0)
    _lib.check(lib.pet_attn_cf_seq(sh, off.data_ptr(), _ptr(cut), out.data_ptr(), _mat(out, "cf_seq", S), _stream()),
               "pet_attn_cf_seq")
    return out


def _width(D: int) -> None:
    if D < 1 or D > MAX_WIDTH:
        raise ValueError(f"rows of {D} columns: the norms take 1 to {MAX_WIDTH}")


def _reach(t: torch.Tensor | None, name: str, n: int, what: str) -> None:
    """Rows and vectors beside inp are as long as it needs them."""
    if t is not None and (t.shape[0] if what == "rows" else t.numel()) < n:
        raise ValueError(f"{name} has {tuple(t.shape)} {what}, expected {n}")


def norm_rows(out: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None) -> None:
    """out = norm(inp) row by row (out may be inp): RMSNorm, or LayerNorm with a
    bias. Rows in float32, bfloat16 or float16, up to 16384 columns; the
    weight and bias float32."""
    lib = _lib.load()
    rows, D = inp.shape
    if inp.dtype != torch.float32 or D > 2048:
        dev = inp.device
        ldi, ldo = _typed(inp, "in", rows, D, inp.dtype, dev), _typed(out, "out", rows, D, inp.dtype, dev)
        _width(D)
        _call_on(dev, "pet_norm_rows_typed", lib.pet_norm_rows_typed, DTYPES[inp.dtype], rows, D, out.data_ptr(), ldo,
                 inp.data_ptr(), ldi, _vector(weight, "weight", D, dev),
                 None if bias is None else _vector(bias, "bias", D, dev))
        return
    _reach(out, "out", rows, "rows")
    _reach(weight, "weight", D, "elements")
    _reach(bias, "bias", D, "elements")
    _lib.check(lib.pet_norm_rows(rows, D, out.data_ptr(), _mat(out, "out", D), inp.data_ptr(), _mat(inp, "in", D),
                                 _weight(weight, "weight"), None if bias is None else _weight(bias, "bias"),
                                 _stream()), "pet_norm_rows")


def norm_rows_bwd(in_adj: torch.Tensor, out_adj: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor, ln: bool,
                  beta: float = 0.0) -> None:
    """in_adj = beta * in_adj + the norm's input adjoint for out_adj (rows as
    norm_rows takes them)."""
    lib = _lib.load()
    rows, D = inp.shape
    if inp.dtype != torch.float32 or D > 2048:
        norm_rows_grads(in_adj, None, None, out_adj, inp, weight, ln, beta)
        return
    _reach(in_adj, "in_adj", rows, "rows")
    _reach(out_adj, "out_adj", rows, "rows")
    _reach(weight, "weight", D, "elements")
    _lib.check(lib.pet_norm_rows_bwd(rows, D, in_adj.data_ptr(), _mat(in_adj, "in_adj", D), float(beta),
                                     out_adj.data_ptr(), _mat(out_adj, "out_adj", D), inp.data_ptr(),
                                     _mat(inp, "in", D), _weight(weight, "weight"), int(bool(ln)), _stream()),
               "pet_norm_rows_bwd")


def norm_rows_grads(in_adj: torch.Tensor | None, weight_adj: torch.Tensor | None, bias_adj: torch.Tensor | None,
                    out_adj: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor, ln: bool, beta: float = 0.0,
                    beta_w: float = 0.0, live: torch.Tensor | None = None,
                    scratch: torch.Tensor | None = None) -> None:
    """The norm's backward with its parameters' gradients: in_adj = beta *
    in_adj + the input adjoint, weight_adj = beta_w * weight_adj + sum over rows
    of out_adj * xhat, bias_adj the same of out_adj (LayerNorm). Each of the
    three may be None (not all); in_adj may be out_adj or inp. Rows as norm_rows
    takes them, the gradients float32. ``live`` (one int32 on the device): only
    rows before it count, the rows after are neither read nor written.
    ``scratch``: pet_norm_rows_grads_workspace(rows, D) bytes, else allocated."""
    lib = _lib.load()
    if not isinstance(inp, torch.Tensor) or inp.dim() != 2:
        raise ValueError("in must be a row-major 2-D view")
    (rows, D), dev, dt = inp.shape, inp.device, inp.dtype
    ldi, ldg = _typed(inp, "in", rows, D, dt, dev), _typed(out_adj, "out_adj", rows, D, dt, dev)
    lda = 0 if in_adj is None else _typed(in_adj, "in_adj", rows, D, dt, dev)
    _width(D)
    if bias_adj is not None and not ln:
        raise ValueError("bias_adj: an RMSNorm has no bias")
    if in_adj is None and weight_adj is None and bias_adj is None:
        raise ValueError("in_adj, weight_adj and bias_adj are all None: nothing to make")
    w_adj = None if weight_adj is None else _vector(weight_adj, "weight_adj", D, dev)
    b_adj = None if bias_adj is None else _vector(bias_adj, "bias_adj", D, dev)
    if w_adj is not None or b_adj is not None:
        scratch = _scratch(scratch, lib.pet_norm_rows_grads_workspace(rows, D), dev)
        ws, nbytes = scratch.data_ptr(), scratch.numel() * scratch.element_size()
    else:
        ws, nbytes = None, 0
    _call_on(dev, "pet_norm_rows_grads", lib.pet_norm_rows_grads, DTYPES[dt], rows, D, _ptr(in_adj), lda, float(beta),
             out_adj.data_ptr(), ldg, inp.data_ptr(), ldi, _vector(weight, "weight", D, dev), int(bool(ln)), w_adj,
             b_adj, float(beta_w), _live(live, dev), ws, nbytes)


def attention_layer(ws: Workspace, key: str, out: torch.Tensor, tokens: torch.Tensor, norm_w: torch.Tensor,
                    norm_b: torch.Tensor | None, w_in: torch.Tensor, b_in: torch.Tensor | None, cf_seq: torch.Tensor,
                    w_out: torch.Tensor, b_out: torch.Tensor | None, tk: Tokens, S: int, heads: int, head_dim: int,
                    temperature: float) -> None:
    """The attention of one PET block from its tokens; the backward's saves
    (merged, ml) stay in ``ws`` under ``key``."""
    lib = _lib.load()
    D = heads * head_dim
    T = tokens.shape[0]
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    merged = ws.n2(key + ":merged", T, D)
    ml = ws.n2(key + ":ml", tk.N * heads * S, 2)
    scratch = ws.bytes("attention_layer:scratch", lib.pet_attention_layer_workspace(sh))
    _lib.check(lib.pet_attention_layer(sh, out.data_ptr(), _mat(out, "out", D), tokens.data_ptr(),
                                       _mat(tokens, "tokens", D), _weight(norm_w, "norm_w"),
                                       None if norm_b is None else _weight(norm_b, "norm_b"), _weight(w_in, "w_in"),
                                       None if b_in is None else _weight(b_in, "b_in"), cf_seq.data_ptr(),
                                       _mat(cf_seq, "cf_seq"), _weight(w_out, "w_out"),
                                       None if b_out is None else _weight(b_out, "b_out"), tk.off.data_ptr(),
                                       merged.data_ptr(), ml.data_ptr(), scratch.data_ptr(), scratch.numel(),
                                       _stream()), "pet_attention_layer")


def attention_layer_bwd(ws: Workspace, key: str, tokens_adj: torch.Tensor, cf_seq_adj: torch.Tensor,
                        out_adj: torch.Tensor, tokens: torch.Tensor, norm_w: torch.Tensor,
                        norm_b: torch.Tensor | None, w_in: torch.Tensor, b_in: torch.Tensor | None,
                        cf_seq: torch.Tensor, w_out: torch.Tensor, tk: Tokens, S: int, heads: int, head_dim: int,
                        temperature: float) -> None:
    """Its backward: tokens_adj's atom rows set, live edge rows accumulated
    (dead rows untouched); cf_seq_adj accumulates."""
    lib = _lib.load()
    D = heads * head_dim
    T = tokens.shape[0]
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    merged, ml = ws.peek2(key + ":merged"), ws.peek2(key + ":ml")
    scratch = ws.bytes("attention_layer:scratch", lib.pet_attention_layer_workspace(sh))
    _lib.check(lib.pet_attention_layer_bwd(sh, tokens_adj.data_ptr(), _mat(tokens_adj, "tokens_adj", D),
                                           cf_seq_adj.data_ptr(), _mat(cf_seq_adj, "cf_seq_adj"),
                                           out_adj.data_ptr(), _mat(out_adj, "out_adj", D), tokens.data_ptr(),
                                           _mat(tokens, "tokens", D), _weight(norm_w, "norm_w"),
                                           None if norm_b is None else _weight(norm_b, "norm_b"),
                                           _weight(w_in, "w_in"), None if b_in is None else _weight(b_in, "b_in"),
                                           cf_seq.data_ptr(), _mat(cf_seq, "cf_seq"), _weight(w_out, "w_out"),
                                           tk.off.data_ptr(), merged.data_ptr(), ml.data_ptr(), scratch.data_ptr(),
                                           scratch.numel(), _stream()), "pet_attention_layer_bwd")


_LAYER_GRADS = ("norm_w", "norm_b", "w_in", "b_in", "w_out", "b_out")


def attention_layer_grads(ws: Workspace, key: str, grads: dict, tokens_adj: torch.Tensor, cf_seq_adj: torch.Tensor,
                          out_adj: torch.Tensor, tokens: torch.Tensor, norm_w: torch.Tensor,
                          norm_b: torch.Tensor | None, w_in: torch.Tensor, b_in: torch.Tensor | None,
                          cf_seq: torch.Tensor, w_out: torch.Tensor, tk: Tokens, S: int, heads: int, head_dim: int,
                          temperature: float, beta: float = 0.0) -> None:
    """attention_layer_bwd with the gradients of the layer's parameters:
    ``grads`` holds the tensors they go to by name (norm_w, norm_b, w_in, b_in,
    w_out, b_out, each of its parameter's shape; those not there are not made, a
    bias's not without its weight's), each onto beta times itself. Dead rows
    count for none, whatever they hold. ``ws`` serves one stream at a time; a call
    that is captured into a graph finds its scratch there from an eager call before
    it, and a call of a larger shape replaces that scratch: a graph has a ``ws`` of its
    own."""
    lib = _lib.load()
    D, dev = heads * head_dim, tokens.device
    T = tokens.shape[0]
    for t, name in ((tokens, "tokens"), (tokens_adj, "tokens_adj"), (out_adj, "out_adj")):
        _typed(t, name, T, D, torch.float32, dev)
    for t, name in ((cf_seq, "cf_seq"), (cf_seq_adj, "cf_seq_adj")):
        _typed(t, name, tk.N, t.shape[-1], torch.float32, dev)
        if t.shape[1] < S:
            raise ValueError(f"{name} narrower than S")
    for t, name, size in ((w_in, "w_in", (3 * D, D)), (w_out, "w_out", (D, D)), (norm_w, "norm_w", (D,)),
                          (norm_b, "norm_b", (D,)), (b_in, "b_in", (3 * D,))):
        if t is not None and (t.device != dev or t.dtype != torch.float32 or tuple(t.shape) != size
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 {list(size)} on {dev}")
    if tk.off.device != dev or tk.off.dtype != torch.int32 or tk.off.numel() != tk.N + 1 \
            or not tk.off.is_contiguous():
        raise ValueError(f"tk.off must be {tk.N + 1} contiguous int32 on {dev}")
    unknown = sorted(set(grads) - set(_LAYER_GRADS))
    if unknown:
        raise ValueError(f"grads: no parameter named {', '.join(unknown)}")
    for b, w in (("b_in", "w_in"), ("b_out", "w_out")):
        if b in grads and w not in grads:
            raise ValueError(f"grads: {b} without {w}")
    if "norm_b" in grads and norm_b is None:
        raise ValueError("grads: norm_b, but an RMSNorm has no bias")
    pg = _lib.LayerGrads(beta=float(beta))
    for name, g in grads.items():
        size = {"w_in": (3 * D, D), "w_out": (D, D), "b_in": (3 * D,)}.get(name, (D,))
        if not isinstance(g, torch.Tensor) or g.device != dev or g.dtype != torch.float32 or tuple(g.shape) != size \
                or not g.is_contiguous():
            raise ValueError(f"grads: {name} must be a contiguous float32 {list(size)} on {dev}")
        setattr(pg, name, g.data_ptr())
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    merged, ml = ws.peek2(key + ":merged"), ws.peek2(key + ":ml")
    if merged.shape != (T, D) or ml.shape != (tk.N * heads * S, 2) or merged.device != dev:
        raise ValueError(f"the saves under {key} are of another shape or on another device")
    scratch = ws.bytes("attention_layer_grads:scratch", lib.pet_attention_layer_grads_workspace(sh))
    _call_on(dev, "pet_attention_layer_grads", lib.pet_attention_layer_grads, sh, ctypes.byref(pg),
             tokens_adj.data_ptr(), _mat(tokens_adj, "tokens_adj", D), cf_seq_adj.data_ptr(),
             _mat(cf_seq_adj, "cf_seq_adj"), out_adj.data_ptr(), _mat(out_adj, "out_adj", D), tokens.data_ptr(),
             _mat(tokens, "tokens", D), _weight(norm_w, "norm_w"), None if norm_b is None else _weight(norm_b, "norm_b"),
             _weight(w_in, "w_in"), None if b_in is None else _weight(b_in, "b_in"), cf_seq.data_ptr(),
             _mat(cf_seq, "cf_seq"), _weight(w_out, "w_out"), tk.off.data_ptr(), merged.data_ptr(), ml.data_ptr(),
             scratch.data_ptr(), scratch.numel())
