"""The reference's attention interface over torch device tensors.

``attention`` and ``attention_bwd`` mirror pet::attention / pet::attention_bwd
(reference src/ops.hpp:121-148, src/attention.cpp:2189-2206): same arguments,
same meaning, same conventions -- row-major fp32 views with their own leading
dimension, ``out`` overwritten, ``in_adj`` computed onto ``beta * in_adj``,
``cf_seq_adj`` accumulated, the forward's saves kept in a Workspace under
``key + ":merged"`` and ``key + ":ml"`` for the backward to find. Errors raise
(PetAttnError, a RuntimeError, as the reference's std::runtime_error).

``attention_chunked`` / ``attention_bwd_chunked`` mirror the reference's
chunked forms (src/ops.hpp:133-146): runs of atoms of about ``chunk`` tokens,
qkv made per run by a ``make_qkv(qkv_rows, r0, r1)`` callable.

``attn_fwd`` / ``attn_bwd`` expose the core kernels alone (no linears),
``attn_fwd_run`` / ``attn_bwd_run`` their per-run forms.

For training, which the reference does not do: ``attn_fwd_typed`` /
``attn_bwd_typed`` are the core of bfloat16 and float16 rows, with key and value
heads shared by groups of query heads, a learned bias by relative position
(``RelativeBias``, ``relative_buckets``) and dropout of the probabilities
(``Dropout``), whose mask the backward makes again. All
work runs in libpet_attn.so on the current torch stream; torch only provides
device memory and the stream.
"""
from __future__ import annotations

import dataclasses
import math

import torch

from . import _lib


@dataclasses.dataclass
class Tokens:
    """CSR token layout (reference src/ops.hpp:31-37): atom n's tokens are row
    n and rows N + off[n] .. N + off[n+1] - 1; ``dead`` when rows past
    N + off[N] exist (an edge capacity)."""
    off: torch.Tensor  # int32 [N+1], device
    N: int
    dead: bool = False


class Workspace:
    """Named device buffers that outlive a call (the reference's Workspace
    n2/peek2, include/pet/kokkos.hpp:65-235): the forward's saves and the
    backward's scratch."""

    def __init__(self, device=None):
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self._named: dict[str, torch.Tensor] = {}

    def n2(self, key: str, rows: int, cols: int) -> torch.Tensor:
        t = self._named.get(key)
        if t is None or t.shape != (rows, cols):
            t = torch.empty((rows, cols), dtype=torch.float32, device=self.device)
            self._named[key] = t
        return t

    def bytes(self, key: str, nbytes: int) -> torch.Tensor:
        t = self._named.get(key)
        if t is None or t.numel() < nbytes:
            t = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=self.device)
            self._named[key] = t
        return t

    def peek2(self, key: str) -> torch.Tensor:
        if key not in self._named:
            raise RuntimeError(f"pet: workspace has no buffer named '{key}' (was the forward run with save=True?)")
        return self._named[key]


MOST = (1 << 31) - 1  # rows or columns: the library counts them in int, and ctypes wraps what passes it


def _mat(t: torch.Tensor, name: str, width: int | None = None) -> int:
    if t.dim() == 2 and max(t.shape) > MOST:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: at most {MOST} rows and columns")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a row-major 2-D view")
    if width is not None and t.shape[1] != width:
        raise ValueError(f"{name} has {t.shape[1]} columns, expected {width}")
    return t.stride(0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weight(t: torch.Tensor, name: str) -> int:
    # The kernels run after this returns: a temporary contiguous copy would be
    # freed under them, so the weight itself must be contiguous.
    if t.device.type != "cuda" or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 device tensor")
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PET_DTYPE_*


def _typed(t: torch.Tensor, name: str, rows: int, width: int, dtype: torch.dtype, device) -> int:
    """The leading dimension of a row-major [rows, width] view of the dtype on the device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is needed")
    if rows > MOST or width > MOST:
        raise ValueError(f"{name}: {rows} x {width}, at most {MOST} rows and columns")
    if t.dtype is dtype and t.shape == (rows, width) and t.device == device and rows > 1 and width > 1:
        ld, step = t.stride()  # (what a small call's host side waits for: the checks below again, in one go)
        if step == 1 and ld >= width and device.type == "cuda" and dtype in DTYPES:
            return ld
    if t.device != device or t.device.type != "cuda":
        raise ValueError(f"{name}: on {t.device}, the operands' device is {device}")
    if t.dtype != dtype or t.dtype not in DTYPES:
        raise ValueError(f"{name}: {t.dtype}, the rows' type is {dtype} (float32, bfloat16 or float16)")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != width:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(rows, width)}")
    if width > 1 and rows > 0 and t.stride(1) != 1:
        raise ValueError(f"{name} must be a row-major 2-D view")
    if rows <= 1:
        return width
    if t.stride(0) < width:
        raise ValueError(f"{name}: rows overlap (stride {t.stride(0)} < width {width})")
    return t.stride(0)


def _vector(t: torch.Tensor, name: str, n: int, device) -> int:
    """The address of a contiguous float32 [n] on the device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is needed")
    if t.device != device or t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{n}] on {device}")
    return t.data_ptr()


def _live(t, device):
    """The address of the device's count of live rows (one int32), None for all."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError("live: a torch tensor is needed")
    if t.device != device or t.dtype != torch.int32 or t.numel() != 1:
        raise ValueError(f"live must be one int32 on {device}")
    return t.data_ptr()


def _scratch(t, nbytes: int, device) -> torch.Tensor:
    """A caller's scratch of at least nbytes, or one of this call's own."""
    if t is None:
        return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    if not isinstance(t, torch.Tensor):
        raise TypeError("scratch: a torch tensor is needed")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"scratch: a contiguous tensor on {device}")
    return t


def _call_on(device, what: str, fn, *args) -> None:
    """fn(*args, stream) with the device's current stream, the device current."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)  # torch.cuda.current_stream(device).cuda_stream, 2 us less
    if index == torch.cuda.current_device():
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code != _lib.OK:
        raise _lib.PetAttnError(code, what)


def shape(N: int, T: int, S: int, heads: int, head_dim: int, temperature: float = 1.0,
          dead: bool = False) -> _lib.Shape:
    # pet_attn_scale's own arithmetic, rounded to float by the struct: a call of the
    # library less in a forward and in a backward, whose host side is what a small
    # cell's attention waits for
    if type(head_dim) is int and type(temperature) is float and head_dim > 0 and temperature > 0.0:
        scale = 1.0 / (math.sqrt(head_dim) * temperature)
    else:
        scale = _lib.load().pet_attn_scale(head_dim, temperature)
    return _lib.Shape(N, T, S, heads, head_dim, int(dead), scale)


def attn_fwd(qkv: torch.Tensor, off: torch.Tensor, cf_seq: torch.Tensor, heads: int, head_dim: int,
             temperature: float = 1.0, N: int | None = None, dead: bool = False, merged: torch.Tensor | None = None,
             ml: torch.Tensor | None = None, save: bool = True):
    """The core forward: (merged [T, D], ml [N*H*S, 2] or None)."""
    lib = _lib.load()
    D = heads * head_dim
    T = qkv.shape[0]
    N = off.shape[0] - 1 if N is None else N
    S = cf_seq.shape[1]
    if merged is None:
        merged = torch.empty((T, D), dtype=torch.float32, device=qkv.device)
    if ml is None and save:
        ml = torch.empty((N * heads * S, 2), dtype=torch.float32, device=qkv.device)
    sh = shape(N, T, S, heads, head_dim, temperature, dead)
    _lib.check(lib.pet_attn_fwd(sh, qkv.data_ptr(), _mat(qkv, "qkv", 3 * D), off.data_ptr(), cf_seq.data_ptr(),
                                _mat(cf_seq, "cf_seq"), merged.data_ptr(), _mat(merged, "merged", D), _ptr(ml),
                                _stream()), "pet_attn_fwd")
    return merged, ml


def attn_bwd(qkv: torch.Tensor, off: torch.Tensor, dmerged: torch.Tensor, merged: torch.Tensor, ml: torch.Tensor,
             cf_seq: torch.Tensor, heads: int, head_dim: int, temperature: float = 1.0,
             cf_seq_adj: torch.Tensor | None = None, N: int | None = None, dead: bool = False,
             qkv_adj: torch.Tensor | None = None, cfh: torch.Tensor | None = None):
    """The core backward: (qkv_adj [T, 3D], cf_seq_adj [N, S] accumulated onto,
    cfh [N, H, S], each key slot's sum over queries of dS per head)."""
    lib = _lib.load()
    D = heads * head_dim
    T = qkv.shape[0]
    N = off.shape[0] - 1 if N is None else N
    S = cf_seq.shape[1]
    if qkv_adj is None:
        qkv_adj = torch.empty((T, 3 * D), dtype=torch.float32, device=qkv.device)
    if cfh is None:
        cfh = torch.empty((N, heads, S), dtype=torch.float32, device=qkv.device)
    if cf_seq_adj is None:
        cf_seq_adj = torch.zeros((N, S), dtype=torch.float32, device=qkv.device)
    sh = shape(N, T, S, heads, head_dim, temperature, dead)
    _lib.check(lib.pet_attn_bwd(sh, qkv.data_ptr(), _mat(qkv, "qkv", 3 * D), off.data_ptr(), dmerged.data_ptr(),
                                _mat(dmerged, "dmerged", D), merged.data_ptr(), _mat(merged, "merged", D),
                                ml.data_ptr(), cf_seq.data_ptr(), _mat(cf_seq, "cf_seq"), qkv_adj.data_ptr(),
                                _mat(qkv_adj, "qkv_adj", 3 * D), cfh.data_ptr(), cf_seq_adj.data_ptr(),
                                _mat(cf_seq_adj, "cf_seq_adj"), _stream()), "pet_attn_bwd")
    return qkv_adj, cf_seq_adj, cfh


@dataclasses.dataclass
class Dropout:
    """Elements left out with probability ``p`` (in steps of 2^-16, at most 65534 /
    65536), the rest scaled by 1 / (1 - p). ``state``: two int64 on the device, a seed
    and a step (its low 32 bits count), read as the kernels run: a program that adds to
    the step there draws anew in each replay of a graph. ``call`` (0 .. 2^32 - 1) tells
    the calls of one step apart; a backward is given its forward's."""
    p: float
    state: torch.Tensor
    call: int = 0


def _dropout(d, device):
    """The library's argument of a Dropout, None for none."""
    if d is None:
        return None
    if not isinstance(d, Dropout):
        raise TypeError("dropout: a Dropout is needed")
    t = d.state
    if not isinstance(t, torch.Tensor):
        raise TypeError("dropout: state: a torch tensor is needed")
    if t.device != device or t.dtype != torch.int64 or tuple(t.shape) != (2,) or not t.is_contiguous():
        raise ValueError(f"dropout: state must be two contiguous int64 on {device}")
    if not 0.0 <= d.p <= 65534 / 65536:
        raise ValueError(f"dropout: p {d.p}: 0 to 65534/65536")
    if not 0 <= d.call < 1 << 32:
        raise ValueError(f"dropout: call {d.call}: 0 to 2^32 - 1")
    return _lib.DropoutArgs(t.data_ptr(), float(d.p), int(d.call))


MAX_BUCKETS, MAX_REACH = 64, 1024  # PET_BIAS_MAX_BUCKETS, PET_BIAS_MAX_REACH


@dataclasses.dataclass
class RelativeBias:
    """A learned bias of the logits: key j adds table[buckets[clamp(positions[j] -
    positions[i], -reach, reach) + reach]][h] for query i of head h, the positions of
    their rows. ``table`` float32 [n_buckets, heads] (at most 64 buckets), ``buckets``
    int32 [2 reach + 1] (``relative_buckets`` makes one; values past the table's ends count
    as its ends), ``positions`` int32, one a row of qkv: any whole numbers, an order's
    or an edge's radial shell's."""
    table: torch.Tensor
    buckets: torch.Tensor
    positions: torch.Tensor


def relative_buckets(n_buckets: int, reach: int, two_sided: bool = True, device=None) -> torch.Tensor:
    """The bucket of each offset -reach .. reach (key's position less the query's) as
    int32 [2 reach + 1]: half of the buckets to each sign (an odd one is left over), of a
    half the first half one to an offset, the rest at equal ratios up to ``reach``, the
    last taking what lies past it. Not ``two_sided``: all of them to keys at or before
    the query, a key after it in bucket 0. Borders are found in whole numbers."""
    if not 1 <= n_buckets <= MAX_BUCKETS or not 0 <= reach <= MAX_REACH:
        raise ValueError(f"{n_buckets} buckets, reach {reach}: 1 to {MAX_BUCKETS} buckets, reach 0 to {MAX_REACH}")
    half = max(1, n_buckets // 2 if two_sided else n_buckets)
    single = max(1, half // 2)
    wide = half - single
    side = []
    for d in range(reach + 1):
        # b is the last bucket with d >= single (reach / single)^((b - single) / wide)
        b = min(d, half - 1)
        if d >= single:
            b = min(single, half - 1)
            while b < half - 1 and d ** wide * single ** (b + 1 - single) >= reach ** (b + 1 - single) * single ** wide:
                b += 1
        side.append(b)
    after = [b + (half if n_buckets > 1 else 0) for b in side[1:]] if two_sided else [0] * reach
    return torch.tensor(side[:0:-1] + side[:1] + after, dtype=torch.int32, device=device)


def _bias(b, heads: int, rows: int, device):
    """The library's argument of a RelativeBias, None for none."""
    if b is None:
        return None
    if not isinstance(b, RelativeBias):
        raise TypeError("bias: a RelativeBias is needed")
    for t, name in ((b.table, "table"), (b.buckets, "buckets"), (b.positions, "positions")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"bias: {name}: a torch tensor is needed")
        kind = torch.float32 if name == "table" else torch.int32
        if t.device != device or t.dtype != kind or not t.is_contiguous():
            raise ValueError(f"bias: {name} must be contiguous {kind} on {device}")
    if b.table.dim() != 2 or b.table.shape[1] != heads or not 1 <= b.table.shape[0] <= MAX_BUCKETS:
        raise ValueError(f"bias: table has shape {tuple(b.table.shape)}, expected 1 to {MAX_BUCKETS} rows of {heads}")
    if b.buckets.dim() != 1 or b.buckets.numel() % 2 != 1 or b.buckets.numel() > 2 * MAX_REACH + 1:
        raise ValueError(f"bias: buckets has shape {tuple(b.buckets.shape)}: 2 reach + 1, reach at most {MAX_REACH}")
    if tuple(b.positions.shape) != (rows,):
        raise ValueError(f"bias: positions has shape {tuple(b.positions.shape)}, expected {(rows,)}")
    return _lib.BiasArgs(b.table.data_ptr(), b.buckets.data_ptr(), b.positions.data_ptr(), b.table.shape[0],
                         b.buckets.numel() // 2)


def _typed_call(qkv, off, cf_seq, heads, head_dim, kv_heads, temperature, dead, N):
    """What attn_fwd_typed and attn_bwd_typed check alike: (shape, kv_heads, ldq, ldc)."""
    if not isinstance(qkv, torch.Tensor) or not isinstance(off, torch.Tensor) or not isinstance(cf_seq, torch.Tensor):
        raise TypeError("qkv, off and cf_seq: torch tensors are needed")
    dev = qkv.device
    kv_heads = heads if kv_heads is None else kv_heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads or not 1 <= head_dim <= 128:
        raise ValueError(f"{heads} heads, {kv_heads} key heads of {head_dim}: whole groups of heads of 1 to 128")
    if qkv.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"qkv: {qkv.dtype}, not bfloat16 or float16 (float32 rows: attn_fwd, attn_bwd)")
    if qkv.dim() != 2:
        raise ValueError("qkv must be a row-major 2-D view")
    T = qkv.shape[0]
    ldq = _typed(qkv, "qkv", T, (heads + 2 * kv_heads) * head_dim, qkv.dtype, dev)
    if off.device != dev or off.dtype != torch.int32 or off.dim() != 1 or not off.is_contiguous() or off.numel() < 1:
        raise ValueError(f"off must be contiguous int32 [N + 1] on {dev}")
    N = off.numel() - 1 if N is None else N
    if not 0 <= N < off.numel() or T < N:
        raise ValueError(f"{N} atoms: off has {off.numel()} entries, qkv {T} rows")
    if cf_seq.dim() != 2 or cf_seq.shape[1] < 1:
        raise ValueError("cf_seq must be a row-major 2-D view")
    ldc = _typed(cf_seq, "cf_seq", N, cf_seq.shape[1], torch.float32, dev)
    if not temperature > 0.0:
        raise ValueError(f"temperature {temperature}: more than 0 is needed")
    return shape(N, T, cf_seq.shape[1], heads, head_dim, temperature, dead), kv_heads, ldq, ldc


def _saves(ml, count: int, device) -> int:
    if not isinstance(ml, torch.Tensor):
        raise TypeError("ml: a torch tensor is needed")
    if ml.device != device or ml.dtype != torch.float32 or tuple(ml.shape) != (count, 2) or not ml.is_contiguous():
        raise ValueError(f"ml must be a contiguous float32 {[count, 2]} on {device}")
    return ml.data_ptr()


def attn_fwd_typed(qkv: torch.Tensor, off: torch.Tensor, cf_seq: torch.Tensor, heads: int, head_dim: int,
                   temperature: float = 1.0, kv_heads: int | None = None, bias: RelativeBias | None = None,
                   dropout: Dropout | None = None, N: int | None = None, dead: bool = False,
                   merged: torch.Tensor | None = None, ml: torch.Tensor | None = None, save: bool = True):
    """attn_fwd of bfloat16 or float16 rows: (merged [T, heads * head_dim], ml
    [N*heads*S, 2] or None). qkv [T, (heads + 2 kv_heads) * head_dim] = [Q | K | V];
    key head k serves the query heads k G .. k G + G - 1, G = heads / kv_heads. ml holds
    (max, 1/sum), (0, 0) where no token or no key is."""
    sh, kv_heads, ldq, ldc = _typed_call(qkv, off, cf_seq, heads, head_dim, kv_heads, temperature, dead, N)
    dev, T, D, S = qkv.device, qkv.shape[0], heads * head_dim, cf_seq.shape[1]
    b, d = _bias(bias, heads, T, dev), _dropout(dropout, dev)
    if merged is None:
        merged = torch.empty((T, D), dtype=qkv.dtype, device=dev)
    ldm = _typed(merged, "merged", T, D, qkv.dtype, dev)
    if ml is None and save:
        ml = torch.empty((sh.n_atoms * heads * S, 2), dtype=torch.float32, device=dev)
    _call_on(dev, "pet_attn_fwd_typed", _lib.load().pet_attn_fwd_typed, DTYPES[qkv.dtype], sh, kv_heads, qkv.data_ptr(),
             ldq, off.data_ptr(), cf_seq.data_ptr(), ldc, b, d, merged.data_ptr(), ldm,
             None if ml is None else _saves(ml, sh.n_atoms * heads * S, dev))
    return merged, ml


def attn_bwd_typed(qkv: torch.Tensor, off: torch.Tensor, dmerged: torch.Tensor, merged: torch.Tensor, ml: torch.Tensor,
                   cf_seq: torch.Tensor, heads: int, head_dim: int, temperature: float = 1.0,
                   kv_heads: int | None = None, bias: RelativeBias | None = None, dropout: Dropout | None = None,
                   qkv_adj: torch.Tensor | None = None, cf_seq_adj: torch.Tensor | None = None,
                   bias_adj: torch.Tensor | None = None, beta: float = 0.0, N: int | None = None, dead: bool = False,
                   scratch: torch.Tensor | None = None):
    """attn_fwd_typed's backward from the adjoint of merged, merged and ml as it left
    them and its bias and dropout: qkv_adj [T, (heads + 2 kv_heads) * head_dim], and
    where given, each onto beta times itself (0: overwritten, where attn_bwd accumulates),
    cf_seq_adj [N, S] and bias_adj (the bias table's shape, float32). ``scratch``: pet_attn_bwd_typed_workspace bytes, else
    allocated. Returns (qkv_adj, cf_seq_adj, bias_adj)."""
    sh, kv_heads, ldq, ldc = _typed_call(qkv, off, cf_seq, heads, head_dim, kv_heads, temperature, dead, N)
    dev, dt, T, D, S = qkv.device, qkv.dtype, qkv.shape[0], heads * head_dim, cf_seq.shape[1]
    W = D + 2 * kv_heads * head_dim
    b, d = _bias(bias, heads, T, dev), _dropout(dropout, dev)
    ldg, ldm = _typed(dmerged, "dmerged", T, D, dt, dev), _typed(merged, "merged", T, D, dt, dev)
    if qkv_adj is None:
        qkv_adj = torch.empty((T, W), dtype=dt, device=dev)
    lda = _typed(qkv_adj, "qkv_adj", T, W, dt, dev)
    ldca = 0 if cf_seq_adj is None else _typed(cf_seq_adj, "cf_seq_adj", sh.n_atoms, S, torch.float32, dev)
    if bias_adj is not None:
        if bias is None:
            raise ValueError("bias_adj without a bias")
        if not isinstance(bias_adj, torch.Tensor):
            raise TypeError("bias_adj: a torch tensor is needed")
        if bias_adj.device != dev or bias_adj.dtype != torch.float32 or bias_adj.shape != bias.table.shape \
                or not bias_adj.is_contiguous():
            raise ValueError(f"bias_adj must be a contiguous float32 {list(bias.table.shape)} on {dev}")
    lib = _lib.load()
    scratch = _scratch(scratch, lib.pet_attn_bwd_typed_workspace(DTYPES[dt], sh, kv_heads, 0 if b is None else b.n_buckets),
                       dev)
    _call_on(dev, "pet_attn_bwd_typed", lib.pet_attn_bwd_typed, DTYPES[dt], sh, kv_heads, qkv.data_ptr(), ldq,
             off.data_ptr(), dmerged.data_ptr(), ldg, merged.data_ptr(), ldm,
             _saves(ml, sh.n_atoms * heads * S, dev), cf_seq.data_ptr(), ldc, b, d, qkv_adj.data_ptr(), lda,
             _ptr(cf_seq_adj), ldca, _ptr(bias_adj), float(beta), scratch.data_ptr(),
             scratch.numel() * scratch.element_size())
    return qkv_adj, cf_seq_adj, bias_adj


def attention(ws: Workspace, key: str, out: torch.Tensor, qkv: torch.Tensor, cf_seq: torch.Tensor,
              w_out: torch.Tensor, b_out: torch.Tensor | None, tk: Tokens, S: int, heads: int, head_dim: int,
              temperature: float, save: bool) -> None:
    """pet::attention: multi-head attention over each atom's tokens with log cf
    as a per-key bias, then out = merged W_out^T + b_out. With ``save`` the
    backward's inputs stay in ``ws`` under ``key``."""
    lib = _lib.load()
    D = heads * head_dim
    T = qkv.shape[0]
    if cf_seq.shape[1] < S:
        raise ValueError("cf_seq narrower than S")
    merged = ws.n2(key + ":merged", T, D) if save else torch.empty((T, D), dtype=torch.float32, device=qkv.device)
    ml = ws.n2(key + ":ml", tk.N * heads * S, 2) if save else None
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    _lib.check(lib.pet_attention(sh, out.data_ptr(), _mat(out, "out", D), qkv.data_ptr(), _mat(qkv, "qkv", 3 * D),
                                 cf_seq.data_ptr(), _mat(cf_seq, "cf_seq"), _weight(w_out, "w_out"),
                                 None if b_out is None else _weight(b_out, "b_out"), tk.off.data_ptr(), merged.data_ptr(), _ptr(ml), _stream()),
               "pet_attention")


def attention_bwd(ws: Workspace, key: str, in_adj: torch.Tensor, cf_seq_adj: torch.Tensor, out_adj: torch.Tensor,
                  qkv: torch.Tensor, cf_seq: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, tk: Tokens,
                  S: int, heads: int, head_dim: int, temperature: float, beta: float) -> None:
    """pet::attention_bwd: in_adj (onto beta * in_adj) is the adjoint of the
    input linear's input; cf_seq_adj accumulates; ``key`` names the forward's
    saves."""
    lib = _lib.load()
    D = heads * head_dim
    T = qkv.shape[0]
    merged, ml = ws.peek2(key + ":merged"), ws.peek2(key + ":ml")
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    nbytes = lib.pet_attention_bwd_workspace(sh)
    scratch = ws.bytes("attention_bwd:scratch", nbytes)
    d_in = w_in.shape[1]
    _lib.check(lib.pet_attention_bwd(sh, in_adj.data_ptr(), _mat(in_adj, "in_adj", d_in), d_in,
                                     cf_seq_adj.data_ptr(), _mat(cf_seq_adj, "cf_seq_adj"), out_adj.data_ptr(),
                                     _mat(out_adj, "out_adj", D), qkv.data_ptr(), _mat(qkv, "qkv", 3 * D),
                                     cf_seq.data_ptr(), _mat(cf_seq, "cf_seq"), _weight(w_in, "w_in"),
                                     _weight(w_out, "w_out"), tk.off.data_ptr(), merged.data_ptr(),
                                     ml.data_ptr(), float(beta), scratch.data_ptr(), scratch.numel(), _stream()),
               "pet_attention_bwd")


def attn_fwd_run(n0: int, n1: int, e0: int, qkv_chunk: torch.Tensor, off: torch.Tensor, cf_seq: torch.Tensor,
                 merged: torch.Tensor, ml: torch.Tensor | None, heads: int, head_dim: int, T: int,
                 temperature: float = 1.0) -> None:
    """The core forward of atoms [n0, n1) from their chunk of qkv rows (own
    rows, then edges' rows from edge e0); merged [T, D] and ml at the whole's
    rows and slots."""
    lib = _lib.load()
    D = heads * head_dim
    N = off.shape[0] - 1
    sh = shape(N, T, cf_seq.shape[1], heads, head_dim, temperature)
    _lib.check(lib.pet_attn_fwd_run(sh, n0, n1, e0, qkv_chunk.data_ptr(), _mat(qkv_chunk, "qkv_chunk", 3 * D),
                                    off.data_ptr(), cf_seq.data_ptr(), _mat(cf_seq, "cf_seq"), merged.data_ptr(),
                                    _mat(merged, "merged", D), _ptr(ml), _stream()), "pet_attn_fwd_run")


def attn_bwd_run(n0: int, n1: int, e0: int, qkv_chunk: torch.Tensor, off: torch.Tensor, dmerged_chunk: torch.Tensor,
                 merged: torch.Tensor, ml: torch.Tensor, cf_seq: torch.Tensor, qkv_adj_chunk: torch.Tensor,
                 cfh: torch.Tensor, heads: int, head_dim: int, T: int, temperature: float = 1.0) -> None:
    """The core backward of atoms [n0, n1) in their chunk rows; cfh [N, H, S]
    at the whole's slots (no cf adjoint, no dead rows)."""
    lib = _lib.load()
    D = heads * head_dim
    N = off.shape[0] - 1
    sh = shape(N, T, cf_seq.shape[1], heads, head_dim, temperature)
    _lib.check(lib.pet_attn_bwd_run(sh, n0, n1, e0, qkv_chunk.data_ptr(), _mat(qkv_chunk, "qkv_chunk", 3 * D),
                                    off.data_ptr(), dmerged_chunk.data_ptr(),
                                    _mat(dmerged_chunk, "dmerged_chunk", D), merged.data_ptr(),
                                    _mat(merged, "merged", D), ml.data_ptr(), cf_seq.data_ptr(),
                                    _mat(cf_seq, "cf_seq"), qkv_adj_chunk.data_ptr(),
                                    _mat(qkv_adj_chunk, "qkv_adj_chunk", 3 * D), cfh.data_ptr(), _stream()),
               "pet_attn_bwd_run")


def atom_runs(off_host, chunk: int):
    """Runs [n0, n1) of consecutive atoms of at most about ``chunk`` tokens (at
    least one atom), with their first and end edges: the reference's atom_runs
    (src/attention.cpp:2060-2070)."""
    N = len(off_host) - 1
    runs, n0 = [], 0
    while n0 < N:
        n1 = n0 + 1
        while n1 < N and (n1 + 1 - n0) + (int(off_host[n1 + 1]) - int(off_host[n0])) <= chunk:
            n1 += 1
        runs.append((n0, n1, int(off_host[n0]), int(off_host[n1])))
        n0 = n1
    return runs


class _RunRows:
    """The make_qkv callback the library calls: the pointer it passes is inside
    the workspace tensor, so the Python callable gets a torch view of it."""

    def __init__(self, make_qkv, ws: torch.Tensor, width: int):
        self.make_qkv = make_qkv
        self.ws = ws.view(torch.float32) if ws.dtype == torch.uint8 else ws
        self.base = ws.data_ptr()
        self.width = width
        self.error = None
        self.cfunc = _lib.MAKE_QKV(self)

    def __call__(self, ctx, ptr, ld, r0, r1, stream):
        try:
            start = (ptr - self.base) // 4
            rows = self.ws[start:start + (r1 - r0) * ld].view(r1 - r0, ld)[:, :self.width]
            self.make_qkv(rows, r0, r1)
        except BaseException as e:  # an exception cannot cross the C frame
            self.error = e


def _chunk_workspace(ws: Workspace, tk: Tokens, off_host, sh, chunk: int):
    lib = _lib.load()
    import numpy as np
    oh = np.ascontiguousarray(off_host, dtype=np.int32)
    nbytes = lib.pet_attention_chunked_workspace(sh, oh.ctypes.data, chunk)
    return oh, ws.bytes("attention_chunked:scratch", nbytes), nbytes


def attention_chunked(ws: Workspace, key: str, out: torch.Tensor, make_qkv, cf_seq: torch.Tensor, w_out: torch.Tensor,
                      b_out: torch.Tensor | None, tk: Tokens, off_host, S: int, heads: int, head_dim: int,
                      temperature: float, save: bool, chunk: int) -> None:
    """pet::attention_chunked: attention() over runs of atoms of about
    ``chunk`` tokens; ``make_qkv(qkv_rows, r0, r1)`` writes the qkv rows of
    tokens [r0, r1) into ``qkv_rows``. ``off_host`` is off on the host."""
    lib = _lib.load()
    D = heads * head_dim
    T = out.shape[0]
    merged = ws.n2(key + ":merged", T, D) if save else torch.empty((T, D), dtype=torch.float32, device=out.device)
    ml = ws.n2(key + ":ml", tk.N * heads * S, 2) if save else None
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    oh, scratch, nbytes = _chunk_workspace(ws, tk, off_host, sh, chunk)
    cb = _RunRows(make_qkv, scratch, 3 * D)
    code = lib.pet_attention_chunked(sh, out.data_ptr(), _mat(out, "out", D), cb.cfunc, None, cf_seq.data_ptr(),
                                     _mat(cf_seq, "cf_seq"), _weight(w_out, "w_out"),
                                     None if b_out is None else _weight(b_out, "b_out"), tk.off.data_ptr(),
                                     oh.ctypes.data, merged.data_ptr(), _ptr(ml), chunk, scratch.data_ptr(), nbytes,
                                     _stream())
    if cb.error is not None:
        raise cb.error
    _lib.check(code, "pet_attention_chunked")


def attention_bwd_chunked(ws: Workspace, key: str, in_adj: torch.Tensor, cf_seq_adj: torch.Tensor,
                          out_adj: torch.Tensor, make_qkv, cf_seq: torch.Tensor, w_in: torch.Tensor,
                          w_out: torch.Tensor, tk: Tokens, off_host, S: int, heads: int, head_dim: int,
                          temperature: float, beta: float, chunk: int) -> None:
    """pet::attention_bwd_chunked over the same runs."""
    lib = _lib.load()
    D = heads * head_dim
    T = in_adj.shape[0]
    merged, ml = ws.peek2(key + ":merged"), ws.peek2(key + ":ml")
    sh = shape(tk.N, T, S, heads, head_dim, temperature, tk.dead)
    oh, scratch, nbytes = _chunk_workspace(ws, tk, off_host, sh, chunk)
    cb = _RunRows(make_qkv, scratch, 3 * D)
    d_in = w_in.shape[1]
    code = lib.pet_attention_bwd_chunked(sh, in_adj.data_ptr(), _mat(in_adj, "in_adj", d_in), d_in,
                                         cf_seq_adj.data_ptr(), _mat(cf_seq_adj, "cf_seq_adj"), out_adj.data_ptr(),
                                         _mat(out_adj, "out_adj", D), cb.cfunc, None, cf_seq.data_ptr(),
                                         _mat(cf_seq, "cf_seq"), _weight(w_in, "w_in"), _weight(w_out, "w_out"),
                                         tk.off.data_ptr(), oh.ctypes.data, merged.data_ptr(), ml.data_ptr(),
                                         float(beta), chunk, scratch.data_ptr(), nbytes, _stream())
    if cb.error is not None:
        raise cb.error
    _lib.check(code, "pet_attention_bwd_chunked")
