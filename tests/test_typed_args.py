"""The typed attention's and the dropout's refusals and formulas, without a GPU: bad
arguments are turned away before any device work (the addresses here are stand-ins), and
the formulas that the GPU tests compare with agree with differences and published
numbers."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest
import torch

from pet_kokkos_amd import _lib, build, layer
from pet_kokkos_amd import attention as A
from typed_attention import Case, attention_mask, rows_mask, threefry

P = [4096 * (i + 1) for i in range(12)]
F32, BF16, F16 = 0, 1, 2


def drop(state=P[10], p=0.1, call=0):
    return _lib.DropoutArgs(state, p, call)


def bias(table=P[7], buckets=P[8], positions=P[9], n=8, reach=4):
    return _lib.BiasArgs(table, buckets, positions, n, reach)


def shape(N=2, T=6, S=4, H=4, hd=16, dead=0, scale=0.25):
    return _lib.Shape(N, T, S, H, hd, dead, scale)


def rows(dtype=BF16, n=4, width=8, out=P[0], ldo=8, x=P[1], ldx=8, r=P[2], ldr=8, d=None, live=None):
    return _lib.load().pet_dropout_rows(dtype, n, width, out, ldo, x, ldx, r, ldr, drop() if d is None else d, live, None)


def test_dropout_rows_refusals():
    assert rows(dtype=3) == rows(n=-1) == rows(width=0) == _lib.EINVAL
    assert rows(out=None) == rows(x=None) == rows(ldo=7) == rows(ldx=7) == rows(ldr=7) == _lib.EINVAL
    assert rows(out=P[1], ldo=9) == rows(out=P[2], ldo=9) == _lib.EINVAL  # in place, but of other rows
    assert rows(out=P[0] + 1) == rows(x=P[1] + 1) == rows(r=P[2] + 1) == rows(live=P[3] + 2) == _lib.EALIGN
    assert rows(dtype=F32, x=P[1] + 2) == rows(d=drop(state=P[3] + 4)) == _lib.EALIGN
    assert rows(d=drop(state=None)) == rows(d=drop(p=-0.1)) == rows(d=drop(p=math.nan)) == _lib.EINVAL
    assert rows(d=drop(p=1.0)) == rows(d=drop(p=65535 / 65536)) == rows(d=drop(p=2.0)) == _lib.EINVAL
    assert _lib.load().pet_dropout_rows(BF16, 4, 8, P[0], 8, P[1], 8, None, 0, None, None, None) == _lib.EINVAL
    assert rows(n=0, out=None, x=None) == _lib.OK


def fwd(dtype=BF16, sh=None, kv=2, qkv=P[0], ldq=128, off=P[1], cf=P[2], ldc=4, b=None, d=None, merged=P[3], ldm=64, ml=P[4]):
    sh = shape() if sh is None else sh
    return _lib.load().pet_attn_fwd_typed(dtype, sh, kv, qkv, ldq, off, cf, ldc, b, d, merged, ldm, ml, None)


def bwd(dtype=BF16, sh=None, kv=2, qkv=P[0], ldq=128, off=P[1], g=P[5], ldg=64, merged=P[3], ldm=64, ml=P[4], cf=P[2], ldc=4,
        b=None, d=None, adj=P[6], lda=128, cfa=None, ldca=0, ta=None, ws=1 << 20, nbytes=1 << 40):
    sh = shape() if sh is None else sh
    return _lib.load().pet_attn_bwd_typed(dtype, sh, kv, qkv, ldq, off, g, ldg, merged, ldm, ml, cf, ldc, b, d, adj, lda, cfa,
                                          ldca, ta, 0.0, ws, nbytes, None)


def test_more_heads_than_a_launch_holds():
    """The tables' sums are a workgroup of 1024 threads a head."""
    wide = dict(sh=shape(H=(1 << 20) + 1, hd=1), kv=1, ldq=1 << 40, ldg=1 << 40, ldm=1 << 40, lda=1 << 40, b=bias())
    assert bwd(ta=P[11], **wide) == _lib.EINDEX
    assert bwd(ta=P[11], ws=None, **{**wide, "sh": shape(H=1 << 20, hd=1)}) == _lib.EWORKSPACE


@pytest.mark.parametrize("call", [fwd, bwd])
def test_attention_refusals(call):
    assert call(dtype=F32) == call(dtype=3) == call(kv=0) == call(kv=3) == _lib.EINVAL
    assert call(sh=shape(N=-1)) == call(sh=shape(T=1)) == call(sh=shape(S=0)) == call(sh=shape(H=0)) == _lib.EINVAL
    assert call(sh=shape(hd=0)) == call(sh=shape(hd=129)) == _lib.EHEADDIM
    assert call(qkv=None) == call(off=None) == call(cf=None) == call(merged=None) == _lib.EINVAL
    assert call(ldq=127) == call(ldm=63) == call(ldc=3) == _lib.EINVAL
    for scale in (0.0, -1.0, math.nan, math.inf, 1e-45):
        assert call(sh=shape(scale=scale)) == _lib.EINVAL
    big = shape(H=1 << 24, hd=128)
    assert call(sh=big, kv=1 << 24, ldq=1 << 40, ldm=1 << 40) == _lib.EINDEX
    assert call(sh=shape(S=(1 << 31) - 1, H=1 << 10, hd=1), kv=1, ldq=1 << 40, ldc=1 << 40, ldm=1 << 40) == _lib.EINDEX
    assert call(sh=shape(N=1 << 28, T=1 << 28, S=100), ldc=100) == _lib.EINDEX
    assert call(qkv=P[0] + 1) == call(merged=P[3] + 1) == call(off=P[1] + 2) == call(cf=P[2] + 2) == _lib.EALIGN
    assert call(ml=P[4] + 4) == _lib.EALIGN
    assert call(b=bias(table=None)) == call(b=bias(buckets=None)) == call(b=bias(positions=None)) == _lib.EINVAL
    assert call(b=bias(n=0)) == call(b=bias(n=65)) == call(b=bias(reach=-1)) == call(b=bias(reach=1025)) == _lib.EINVAL
    assert call(b=bias(table=P[7] + 2)) == call(b=bias(buckets=P[8] + 1)) == call(b=bias(positions=P[9] + 2)) == _lib.EALIGN
    assert call(d=drop(state=None)) == call(d=drop(p=1.0)) == _lib.EINVAL
    assert call(d=drop(state=P[3] + 4)) == _lib.EALIGN


def test_backward_refusals():
    lib = _lib.load()
    assert bwd(g=None) == bwd(ml=None) == bwd(adj=None) == bwd(ldg=63) == bwd(lda=127) == _lib.EINVAL
    assert bwd(cfa=P[7], ldca=3) == bwd(ta=P[7]) == _lib.EINVAL  # a table's adjoint without a table
    assert bwd(g=P[5] + 1) == bwd(adj=P[6] + 1) == bwd(cfa=P[7] + 2, ldca=4) == bwd(b=bias(), ta=P[7] + 2) == _lib.EALIGN
    for nb in (0, 8):
        need = lib.pet_attn_bwd_typed_workspace(BF16, shape(), 2, nb)
        b = bias() if nb else None
        assert need > 0 and bwd(ws=None, b=b) == bwd(nbytes=need - 1, b=b) == _lib.EWORKSPACE
    assert bwd(ws=(1 << 20) + 8) == _lib.EALIGN
    assert lib.pet_attn_bwd_typed_workspace(BF16, None, 2, 0) == lib.pet_attn_bwd_typed_workspace(F32, shape(), 2, 0) == 0
    assert lib.pet_attn_bwd_typed_workspace(BF16, shape(), 3, 0) == lib.pet_attn_bwd_typed_workspace(BF16, shape(), 2, 65) == 0
    assert lib.pet_attn_bwd_typed_workspace(BF16, shape(N=-1), 2, 0) == lib.pet_attn_bwd_typed_workspace(BF16, shape(T=-1), 2, 0) == 0


def test_host_tensors_and_wrong_shapes_are_refused():
    x, off, cf = torch.zeros(6, 96).bfloat16(), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 4)
    state = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError):
        A.attn_fwd_typed(x, off, cf, 2, 16)  # no CPU path
    with pytest.raises(ValueError):
        A.attn_fwd_typed(x.float(), off, cf, 2, 16)
    with pytest.raises(ValueError):
        A.attn_fwd_typed(x, off, cf, 3, 16, kv_heads=2)
    with pytest.raises(ValueError):
        A.attn_fwd_typed(x, off, cf, 2, 129)
    with pytest.raises(TypeError):
        A.attn_fwd_typed(x, None, cf, 2, 16)
    with pytest.raises(ValueError):
        layer.dropout_rows(x, x, A.Dropout(0.1, state))
    with pytest.raises(TypeError):
        layer.dropout_rows(x, x, None)


def test_plans_are_checked():
    dev, state = torch.device("cpu"), torch.zeros(2, dtype=torch.int64)
    assert A._dropout(None, dev) is None and A._bias(None, 2, 6, dev) is None
    assert A._dropout(A.Dropout(0.25, state, 5), dev).call == 5
    for d in (A.Dropout(-0.1, state), A.Dropout(1.0, state), A.Dropout(math.nan, state), A.Dropout(0.1, state, -1),
              A.Dropout(0.1, state, 1 << 32), A.Dropout(0.1, state.int()), A.Dropout(0.1, torch.zeros(4, dtype=torch.int64)[::2]),
              A.Dropout(0.1, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            A._dropout(d, dev)
    with pytest.raises(TypeError):
        A._dropout(0.1, dev)
    good = dict(table=torch.zeros(8, 2), buckets=torch.zeros(9, dtype=torch.int32), positions=torch.zeros(6, dtype=torch.int32))
    assert A._bias(A.RelativeBias(**good), 2, 6, dev).reach == 4
    for name, t in (("table", torch.zeros(8, 3)), ("table", torch.zeros(65, 2)), ("table", torch.zeros(0, 2)),
                    ("table", torch.zeros(8, 2).double()), ("table", torch.zeros(8, 4)[:, ::2]), ("buckets", good["buckets"][:8]),
                    ("buckets", torch.zeros(2051, dtype=torch.int32)), ("buckets", good["buckets"].long()),
                    ("positions", torch.zeros(5, dtype=torch.int32)), ("positions", torch.zeros(6))):
        with pytest.raises(ValueError):
            A._bias(A.RelativeBias(**{**good, name: t}), 2, 6, dev)
    with pytest.raises(TypeError):
        A._bias(A.RelativeBias(**{**good, "table": None}), 2, 6, dev)
    with pytest.raises(TypeError):
        A._bias("table", 2, 6, dev)


@pytest.mark.parametrize("n,reach", [(32, 128), (17, 50), (64, 1024), (2, 1), (1, 0), (1, 5), (3, 7), (32, 5), (4, 0)])
@pytest.mark.parametrize("two_sided", [True, False])
def test_relative_buckets(n, reach, two_sided):
    """Every offset's bucket lies in the table, grows with the distance, is one to an offset near 0, and, past that, its
    border is the formula's: single (reach / single)^(i / wide), the offsets next to a border apart."""
    t = A.relative_buckets(n, reach, two_sided).tolist()
    assert len(t) == 2 * reach + 1 and all(0 <= b < n for b in t)
    back, ahead = t[reach::-1], t[reach:]
    assert back == sorted(back) and t[reach] == 0
    half = max(1, n // 2 if two_sided else n)
    single = max(1, half // 2)
    for side in ([back, [0] + [b - (half if n > 1 else 0) for b in ahead[1:]]] if two_sided else [back]):
        for d, b in enumerate(side):
            if d < single:
                assert b == min(d, half - 1)
            else:
                place = single + math.log(d / single) / math.log(reach / single) * (half - single) if reach > single else half
                if abs(place - round(place)) > 1e-9:
                    assert b == min(half - 1, math.floor(place))
    if not two_sided:
        assert all(b == 0 for b in ahead)
    with pytest.raises(ValueError):
        A.relative_buckets(65, 10)
    with pytest.raises(ValueError):
        A.relative_buckets(8, 1025)


def test_threefry_known_answers():
    """The generator's published answers (20 rounds), and the masks' shape and scale from it."""
    m = 0xFFFFFFFF
    for key, counter, want in (((0, 0), (0, 0), (0x6B200159, 0x99BA4EFE)), ((m, m), (m, m), (0x1CB996FC, 0xBB002BE7)),
                               ((0x13198A2E, 0x03707344), (0x243F6A88, 0x85A308D3), (0xC4923A9C, 0x483DF7A0))):
        assert tuple(int(v) for v in threefry(key, counter, 20)) == want
    mask = rows_mask(3, 4, 5, 0.25, 50, 203)
    assert mask.shape == (50, 203) and set(mask.unique().tolist()) == {0.0, 65536 / 49152}
    assert attention_mask(3, 4, 5, 0.25, [0, 9, 10], 2).shape == (2, 3, 3)


def test_the_formulas_against_differences():
    """The backward's formula is the forward's derivative: central differences in 64 bits, error of the order of the step
    squared (2^-20) and of rounding over the step (2^-52 / 2^-10)."""
    case = Case([5, 9], 2, 1, 4, torch.float16, buckets=4, reach=3, p=0.2, zeros=0.2)
    case.buckets = A.relative_buckets(4, 3)
    case.qkv, case.cf, case.table = case.qkv.double(), case.cf.double(), case.table.double()
    w = case.dmerged = case.dmerged.double()
    got = case.backward(case.forward()[0])
    gen = torch.Generator().manual_seed(0)
    for x, name in ((case.qkv, "qkv_adj"), (case.cf, "cf_seq_adj"), (case.table, "bias_adj")):
        delta = torch.randn(x.shape, generator=gen, dtype=torch.float64) * (x != 0)
        keep, ends = x.clone(), []
        for sign in (1, -1):
            x.copy_(keep + sign * 2.0 ** -10 * delta)
            ends.append(float((w * case.forward()[0]).sum()))
        x.copy_(keep)
        quotient, along = (ends[0] - ends[1]) * 2.0 ** 9, float((got[name][0] * delta).sum())
        assert abs(quotient - along) <= 2.0 ** -14 * float((got[name][0] * delta).abs().sum()), name


def test_cpp_calls_refuse_shapes():
    """The C++ calls throw for views that do not fit together, before they reach the GPU."""
    if not os.path.exists(build.CPP_TEST6):
        pytest.fail(f"{build.CPP_TEST6} is not built (python -m pet_kokkos_amd.build)")
    res = subprocess.run([build.CPP_TEST6], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout == "", res.stdout + res.stderr
