"""The training operators' refusals, without a GPU: every bad argument is
turned away before any device work (the addresses here are stand-ins)."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest
import torch

from pet_kokkos_amd import _lib, grads, layer, linear

A, B, C, W, WS = (4096 * (i + 1) for i in range(5))
F32, BF16, F16 = 0, 1, 2


def norm(dtype=BF16, rows=4, width=8, out=A, ldo=8, inp=B, ldi=8, w=W, b=None):
    return _lib.load().pet_norm_rows_typed(dtype, rows, width, out, ldo, inp, ldi, w, b, None)


def test_norm_refusals():
    assert norm(dtype=3) == norm(dtype=-1) == _lib.EINVAL
    assert norm(rows=-1) == norm(width=0) == norm(width=16385, ldo=16385, ldi=16385) == _lib.EINVAL
    assert norm(out=None) == norm(inp=None) == norm(w=None) == _lib.EINVAL
    assert norm(ldo=7) == norm(ldi=7) == _lib.EINVAL
    assert norm(out=A + 1) == norm(inp=B + 1) == _lib.EALIGN  # half an element off
    assert norm(dtype=F32, out=A + 2) == norm(dtype=F32, inp=B + 1) == _lib.EALIGN


def norm_grads(dtype=F32, rows=4, width=8, in_adj=A, lda=8, g=B, ldg=8, x=C, ldx=8, w=W, ln=1, wa=WS, ba=WS, ws=WS,
               nbytes=1 << 30):
    return _lib.load().pet_norm_rows_grads(dtype, rows, width, in_adj, lda, 0.0, g, ldg, x, ldx, w, ln, wa, ba, 0.0,
                                           None, ws, nbytes, None)


def test_norm_grads_refusals():
    lib = _lib.load()
    assert norm_grads(dtype=7) == norm_grads(rows=-1) == norm_grads(width=0) == _lib.EINVAL
    assert norm_grads(width=16385, lda=16385, ldg=16385, ldx=16385) == _lib.EINVAL
    assert norm_grads(g=None) == norm_grads(x=None) == norm_grads(w=None) == _lib.EINVAL
    assert norm_grads(lda=7) == norm_grads(ldg=7) == norm_grads(ldx=7) == _lib.EINVAL
    assert norm_grads(in_adj=None, wa=None, ba=None) == _lib.EINVAL  # nothing to make
    assert norm_grads(ln=0) == _lib.EINVAL  # an RMSNorm's bias
    assert norm_grads(in_adj=A + 2) == norm_grads(g=B + 1) == norm_grads(x=C + 2) == norm_grads(ws=WS + 4) == _lib.EALIGN
    assert norm_grads(wa=WS + 2) == norm_grads(w=W + 1) == _lib.EALIGN
    need = lib.pet_norm_rows_grads_workspace(4, 8)
    assert need > 0 and norm_grads(ws=None) == norm_grads(nbytes=need - 1) == _lib.EWORKSPACE
    assert lib.pet_norm_rows_grads_workspace(-1, 8) == lib.pet_norm_rows_grads_workspace(4, 0) == 0


def linear_grads(dtype=F32, M=4, N=8, K=16, g=A, ldg=8, x=B, ldx=16, wa=C, ldw=16, ba=W, ws=WS, nbytes=1 << 40):
    return _lib.load().pet_linear_grads(dtype, M, N, K, g, ldg, x, ldx, None, wa, ldw, ba, 0.0, ws, nbytes, None)


def test_linear_grads_refusals():
    lib = _lib.load()
    assert linear_grads(dtype=3) == linear_grads(M=-1) == linear_grads(N=0) == linear_grads(K=0) == _lib.EINVAL
    assert linear_grads(g=None) == linear_grads(x=None) == linear_grads(wa=None) == _lib.EINVAL
    assert linear_grads(ldg=7) == linear_grads(ldx=15) == linear_grads(ldw=15) == _lib.EINVAL
    big = 1 << 16
    assert linear_grads(N=big, K=big, ldg=big, ldx=big, ldw=big) == _lib.EINDEX
    assert linear_grads(g=A + 2) == linear_grads(x=B + 1) == linear_grads(wa=C + 2) == linear_grads(ba=W + 1) == _lib.EALIGN
    assert linear_grads(dtype=F16, g=A + 1) == linear_grads(ws=WS + 8) == _lib.EALIGN
    need = lib.pet_linear_grads_workspace(F32, 4, 8, 16)
    assert need > 0 and linear_grads(ws=None) == linear_grads(nbytes=need - 1) == _lib.EWORKSPACE
    assert lib.pet_linear_grads_workspace(3, 4, 8, 16) == lib.pet_linear_grads_workspace(F32, -1, 8, 16) == 0


def clip(entries=((A, 2, 3, 3, F32),), p=2, scale=1.0, max_norm=1.0, eps=1e-6, out=B, ws=WS, nbytes=1 << 30, n=None,
         norm_only=False):
    lib = _lib.load()
    array = (_lib.GradTensor * max(1, len(entries)))(*[_lib.GradTensor(*e) for e in entries])
    n = len(entries) if n is None else n
    if norm_only:
        return lib.pet_grad_norm(array, n, p, scale, out, ws, nbytes, None)
    return lib.pet_grad_clip(array, n, p, scale, max_norm, eps, out, ws, nbytes, None)


@pytest.mark.parametrize("norm_only", [True, False])
def test_gradient_list_refusals(norm_only):
    def call(**a):
        return clip(norm_only=norm_only, **a)
    assert call(p=3) == call(p=-1) == call(n=-1) == call(out=None) == _lib.EINVAL
    assert call(scale=math.nan) == call(scale=math.inf) == _lib.EINVAL
    assert call(entries=((A, -1, 3, 3, F32),)) == call(entries=((A, 2, -3, 3, F32),)) == _lib.EINVAL
    assert call(entries=((A, 2, 3, 2, F32),)) == call(entries=((None, 2, 3, 3, F32),)) == _lib.EINVAL
    assert call(entries=((A, 2, 3, 3, 3),)) == _lib.EINVAL
    assert call(entries=((A, 1 << 20, 1 << 17, 1 << 17, BF16),)) == _lib.EINDEX
    assert call(entries=((A + 2, 2, 3, 3, F32),)) == call(entries=((A + 1, 2, 3, 3, F16),)) == _lib.EALIGN
    assert call(ws=None) == call(nbytes=_lib.load().pet_grad_workspace(1) - 1) == _lib.EWORKSPACE
    assert call(ws=WS + 4) == call(out=B + 2) == _lib.EALIGN
    assert _lib.load().pet_grad_workspace(-1) == 0 < _lib.load().pet_grad_workspace(0)


def test_clip_refusals():
    for bad in (-1.0, math.nan):
        assert clip(max_norm=bad) == clip(eps=bad) == _lib.EINVAL
    assert clip(eps=math.inf) == _lib.EINVAL


def test_layer_grads_refusals():
    lib = _lib.load()
    sh = _lib.Shape(2, 6, 4, 1, 16, 0, 0.25)
    need = lib.pet_attention_layer_grads_workspace(ctypes.byref(sh))
    assert need > lib.pet_attention_layer_workspace(ctypes.byref(sh))
    assert lib.pet_attention_layer_grads_workspace(None) == 0

    def call(pg, norm_b=None, nbytes=need, tokens=A, out_adj=A, ldo=16, merged=A, ws=1 << 20):
        return lib.pet_attention_layer_grads(ctypes.byref(sh), None if pg is None else ctypes.byref(pg), A, 16, A, 4,
                                             out_adj, ldo, tokens, 16, A, norm_b, A, None, A, 4, A, A, merged, A, ws,
                                             nbytes, None)
    assert call(None) == _lib.EINVAL
    assert call(_lib.LayerGrads(norm_b=A)) == _lib.EINVAL  # an RMSNorm's bias
    assert call(_lib.LayerGrads(b_in=A)) == call(_lib.LayerGrads(b_out=A)) == _lib.EINVAL
    assert call(_lib.LayerGrads(), tokens=None) == call(_lib.LayerGrads(), out_adj=None) == _lib.EINVAL
    assert call(_lib.LayerGrads(), merged=None) == call(_lib.LayerGrads(), ldo=15) == _lib.EINVAL
    assert call(_lib.LayerGrads(), nbytes=need - 1) == call(_lib.LayerGrads(), ws=None) == _lib.EWORKSPACE
    assert call(_lib.LayerGrads(), ws=(1 << 20) + 16) == _lib.EALIGN


def test_host_tensors_are_refused():
    """There is no CPU path: tensors in host memory raise before the library is called."""
    x, w = torch.zeros(4, 8), torch.zeros(8)
    with pytest.raises(ValueError):
        layer.norm_rows(x.bfloat16(), x.bfloat16(), w, None)
    with pytest.raises(ValueError):
        layer.norm_rows_bwd(x.half(), x.half(), x.half(), w, False)
    with pytest.raises(ValueError):
        layer.norm_rows_grads(x, w, None, x, x, w, False)
    with pytest.raises(ValueError):
        linear.linear_grads(x, x, torch.zeros(8, 8))
    with pytest.raises(TypeError):
        linear.linear_grads(x, None, torch.zeros(8, 8))
    with pytest.raises(ValueError):
        grads.GradList([x])
    with pytest.raises(TypeError):
        grads.GradList([3.0])


def test_layouts_of_gradients():
    """Which strides count as consecutive, as rows of a wider matrix, or as neither."""
    t = torch.zeros(4, 6, 8)
    assert grads._layout(t, 0) == (1, 192, 192)
    assert grads._layout(t.permute(2, 0, 1), 0) == (1, 192, 192)
    assert grads._layout(t[:, :, :5][0], 0) == (6, 5, 8)
    assert grads._layout(t[0].t()[:5], 0) == (6, 5, 8)
    assert grads._layout(t[0, :, 3:4], 0) == (6, 1, 8) == grads._layout(t[0, :, 3], 0)
    assert grads._layout(torch.zeros(()), 0) == (1, 1, 1)
    for bad in (t[:, ::2, :5], t[0, :, ::2], torch.zeros(3, 1).expand(3, 4), t[:, :5, :]):
        with pytest.raises(ValueError):
            grads._layout(bad, 0)
    a, b = t[0][:, :5], t[0][:, 5:]
    assert grads._side_by_side(a, b) and not grads._side_by_side(a, t[0][:, 4:])


def test_a_gradient_twice():
    """One tensor for two gradients would be written by both."""
    assert norm_grads(wa=A, ba=A) == _lib.EINVAL
    assert linear_grads(wa=C, ba=C) == _lib.EINVAL
    sh = _lib.Shape(2, 6, 4, 1, 16, 0, 0.25)
    need = _lib.load().pet_attention_layer_grads_workspace(ctypes.byref(sh))
    for pg in (_lib.LayerGrads(norm_w=B, norm_b=B), _lib.LayerGrads(w_in=B, w_out=B), _lib.LayerGrads(norm_w=B, w_out=C, b_out=B)):
        assert _lib.load().pet_attention_layer_grads(ctypes.byref(sh), ctypes.byref(pg), A, 16, A, 4, A, 16, A, 16, A, A, A,
                                                     None, A, 4, A, A, A, A, 1 << 20, need, None) == _lib.EINVAL


def test_views_of_one_row():
    """A row expanded to a matrix of one has a leading dimension of 0."""
    t = torch.zeros(10)
    a, b = t[:6].as_strided((1, 6), (0, 1)), t[4:].as_strided((1, 6), (0, 1))
    assert not grads._side_by_side(a, b)


def test_workspaces_follow_the_sizes():
    """The norm gradients' workspace holds a row of sums a workgroup: no more than
    there are rows, nor than the chip takes of that width at once."""
    need = _lib.load().pet_norm_rows_grads_workspace
    for width in (1, 100, 512, 513, 4096, 4097, 16384):
        row = 2 * 4 * width
        assert need(0, width) == need(1, width) == row and need(3, width) == 3 * row
        most = need((1 << 31) - 1, width)
        assert most % row == 0 and 256 * row <= most <= 2048 * row
    assert need((1 << 31) - 1, 16384) == 256 * 2 * 4 * 16384
    assert _lib.load().pet_grad_workspace((1 << 31) - 1) > 0


def test_no_training_kernel_spills(tmp_path):
    """The weight gradients' accumulators, and the norms' rows of a multiple of the
    vector, stay in registers: each spill is read and written every step or row."""
    from test_kernel_resources import kernels
    sizes = kernels(tmp_path)
    wgrad = {n: s for n, s in sizes.items() if "wgrad_kernel" in n}
    norms = {n: s for n, s in sizes.items() if "norm_grads_kernel" in n and "ELb1EL" in n or "norm_typed_fwd" in n}
    assert len(wgrad) == 9 and len(norms) > 40
    assert {n: s for n, s in {**wgrad, **norms}.items() if s > 0} == {}


def test_layer_grads_refuse_a_shape():
    """A shape without heads, columns or rows enough comes back as an error (no size is
    computed of it), and so do products of nothing."""
    lib = _lib.load()

    def call(sh, w_out=A, out_adj=A, pg=_lib.LayerGrads(), ldo=16):
        return lib.pet_attention_layer_grads(ctypes.byref(sh), ctypes.byref(pg), A, 16, A, 4, out_adj, ldo, A, 16, A, A, A,
                                             None, A, 4, w_out, A, A, A, 1 << 20, 1 << 40, None)
    for bad, code in (((2, 6, 4, 0, 16), _lib.EINVAL), ((2, 6, 4, 1, 0), _lib.EHEADDIM), ((2, 6, 4, -1, 16), _lib.EINVAL),
                      ((2, 6, 4, 1, -16), _lib.EHEADDIM), ((2, 6, 4, 1, 129), _lib.EHEADDIM), ((2, -6, 4, 1, 16), _lib.EINVAL),
                      ((2, 1, 4, 1, 16), _lib.EINVAL), ((-1, 6, 4, 1, 16), _lib.EINVAL), ((2, 6, 0, 1, 16), _lib.EINVAL),
                      ((0, 0, 0, 0, 16), _lib.EINVAL), ((2, (1 << 31) - 1, 4, 64, 128), _lib.EINDEX)):
        sh = _lib.Shape(*bad, 0, 0.25)
        assert lib.pet_attention_layer_grads_workspace(ctypes.byref(sh)) == 0, bad
        assert call(sh) == code, bad
    sh = _lib.Shape(2, 6, 4, 1, 16, 0, 0.25)
    assert call(sh, w_out=None) == call(sh, out_adj=None) == call(sh, ldo=15) == _lib.EINVAL
    assert lib.pet_attention_layer_grads_workspace(ctypes.byref(_lib.Shape(0, 0, 0, 1, 16, 0, 0.25))) > 0  # no tokens: no slots


def test_layer_bwd_refuses_no_operands():
    """The backward without parameters' gradients: a null operand of its first product."""
    lib = _lib.load()
    sh = _lib.Shape(2, 6, 4, 1, 16, 0, 0.25)

    def call(w_out=A, out_adj=A, ldo=16):
        return lib.pet_attention_layer_bwd(ctypes.byref(sh), A, 16, A, 4, out_adj, ldo, A, 16, A, A, A, None, A, 4, w_out, A,
                                           A, A, 1 << 20, 1 << 40, None)
    assert call(w_out=None) == call(out_adj=None) == call(ldo=15) == _lib.EINVAL


def test_columns_side_by_side():
    """Views whose elements lie between each other's are apart where their columns are."""
    m, h = torch.zeros(12, 10), torch.zeros(12, 20, dtype=torch.float16)
    for a, b in ((m[:, 0], m[:, 1]), (m[:, 1], m[:, 0]), (m.t()[:3], m.t()[3:]), (m.t()[:3], m[:, 3:]), (m[:, 0], m[:, 1:]),
                 (m[::2, :4], m[:, 4:]), (m[::3, :4], m[::2, 4:]), (m[::2], m[1::2]), (m[2, 3:5], m[:, :3]),
                 (m[:, :3], m[2, 3:5]), (h[:, :6], h.view(torch.float32)[:, 3:])):
        assert grads._side_by_side(a, b) and grads._side_by_side(b, a)
    for a, b in ((m[:, 0], m[:, 0]), (m[:, :2], m[:, 1]), (m.t()[:4], m[:, 3:]), (m[::2, :5], m[:, 4:]), (m[::2], m[::3]),
                 (m[2], m[:, :3]), (m[2, 2:5], m[:, :3]), (m, m[:, 3]), (h[:, :7], h.view(torch.float32)[:, 3:])):
        assert not grads._side_by_side(a, b) and not grads._side_by_side(b, a)


def test_linear_grads_past_a_launch():
    """A weight of 2^24 tiles: 2^32 threads of one launch, which would come out as none."""
    one, edge = 1 << 30, (1 << 30) - 64
    assert linear_grads(N=one, K=1, ldg=one, ldx=1, ldw=1) == linear_grads(N=1, K=one, ldg=1, ldx=one, ldw=one) == _lib.EINDEX
    assert linear_grads(N=edge + 1, K=1, ldg=one, ldx=1, ldw=1) == _lib.EINDEX
    assert linear_grads(N=edge, K=1, ldg=one, ldx=1, ldw=1, ws=None) == _lib.EWORKSPACE  # fits


def test_in_place_needs_the_same_rows():
    """In place with another leading dimension a row would be written over one not yet read."""
    assert norm(out=A, inp=A, ldo=8, ldi=9) == norm(dtype=F32, out=A, inp=A, ldo=9, ldi=8) == _lib.EINVAL
    assert norm_grads(in_adj=A, lda=9, g=A, ldg=8) == norm_grads(in_adj=A, lda=8, x=A, ldx=9) == _lib.EINVAL
    # one row has no next one: past that check, to the workspace's
    assert norm_grads(rows=1, in_adj=A, lda=9, g=A, ldg=8, ws=None) == _lib.EWORKSPACE
    assert norm_grads(in_adj=A, lda=9, g=A, ldg=9, ws=None) == norm_grads(in_adj=None, lda=0, g=A, ws=None) == _lib.EWORKSPACE


def test_a_launch_takes_what_its_arguments_hold():
    """4096 bytes of arguments: 56 of a launch's own, then 16 a slot, two a tensor whose
    rows are apart; the workspace is of that many tensors a launch."""
    need = _lib.load().pet_grad_workspace
    most = (4096 - 56) // 16 // 2
    assert need(most) == need(1) and need(most + 1) == 2 * need(1) and need(10 * most) == 10 * need(1)


def test_cpp_calls_refuse_shapes():
    """The C++ training calls throw for views that do not fit together."""
    from pet_kokkos_amd import build
    if not os.path.exists(build.CPP_TEST5):
        pytest.fail(f"{build.CPP_TEST5} is not built (python -m pet_kokkos_amd.build)")
    res = subprocess.run([build.CPP_TEST5], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout == "", res.stdout + res.stderr


def test_rows_past_an_int():
    """2^32 rows and more would come to the library as what is left of them modulo 2^32."""
    w = torch.ones(1)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(1, dtype=dtype).expand((1 << 32) + 5, 1)
        for call in (lambda: layer.norm_rows(x, x, w, None), lambda: layer.norm_rows_bwd(x, x, x, w, False),
                     lambda: layer.norm_rows_grads(x, w, None, x, x, w, False), lambda: linear.linear_grads(x, x, w[:, None]),
                     lambda: linear.linear_grads(x.t(), x.t(), w[:, None])):
            with pytest.raises(ValueError, match=str((1 << 31) - 1)):
                call()


def test_no_fp32_rows():
    """No rows have no addresses: the fp32 norms take them as the typed ones do."""
    lib = _lib.load()
    assert lib.pet_norm_rows(0, 8, None, 8, None, 8, W, None, None) == _lib.OK == norm(rows=0, out=None, inp=None)
    assert lib.pet_norm_rows_bwd(0, 8, None, 8, 0.0, None, 8, None, 8, W, 0, None) == _lib.OK
    assert lib.pet_norm_rows(0, 8, None, 8, None, 8, None, None, None) == lib.pet_norm_rows(1, 8, None, 8, A, 8, W, None, None) == _lib.EINVAL
    assert lib.pet_norm_rows_bwd(1, 8, A, 8, 0.0, None, 8, B, 8, W, 0, None) == _lib.EINVAL


def test_fp32_norms_reach_no_further():
    """Fewer rows or a shorter vector than the input's would be read or written past their end."""
    x, w = torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: layer.norm_rows(x[:3], x, w, None), lambda: layer.norm_rows(x, x, w[:7], None),
                 lambda: layer.norm_rows(x, x, w, w[:7]), lambda: layer.norm_rows_bwd(x[:3], x, x, w, True),
                 lambda: layer.norm_rows_bwd(x, x[:3], x, w, True), lambda: layer.norm_rows_bwd(x, x, x, w[:7], False)):
        with pytest.raises(ValueError, match="(rows|elements), expected"):
            call()
