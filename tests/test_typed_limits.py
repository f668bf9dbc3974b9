"""Sizes of the typed attention past an int's and results over operands, without a GPU."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from pet_kokkos_amd import _lib, build
from test_kernel_resources import kernels
from test_typed_args import P, bias, bwd, fwd, shape


def test_cpp_calls_refuse_products_past_an_int():
    if not os.path.exists(build.CPP_TEST7):
        pytest.fail(f"{build.CPP_TEST7} is not built (python -m pet_kokkos_amd.build)")
    res = subprocess.run([build.CPP_TEST7], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout == "", res.stdout + res.stderr


def test_results_in_an_operands_place_are_refused():
    """The kernels read rows again after others' results are written."""
    assert fwd(merged=P[0]) == fwd(ml=P[2]) == _lib.EINVAL
    assert bwd(adj=P[0]) == bwd(adj=P[5]) == bwd(adj=P[3]) == bwd(cfa=P[2], ldca=4) == bwd(cfa=P[4], ldca=4) == _lib.EINVAL
    assert bwd(b=bias(), ta=P[7]) == bwd(b=bias(), ta=P[2]) == bwd(b=bias(), ta=P[4]) == _lib.EINVAL
    assert bwd(ws=None) == bwd(ws=None, cfa=P[8], ldca=4, b=bias(), ta=P[10]) == _lib.EWORKSPACE
    none = dict(sh=shape(N=0, T=0), qkv=None, cf=None, merged=None, ml=None)  # no rows, no places
    assert fwd(**none) == _lib.OK and bwd(**none, g=None, adj=None, ws=None) == _lib.EWORKSPACE


def most_scratch(kernel, dims, tiles, group, whole, bias, drop, half):
    """Bytes of scratch a lane that a typed attention kernel may take: none but in the families here."""
    parts = 0 if whole else 1
    if kernel == "fwd_short":
        return 24 if dims == 64 and drop and not bias else 0
    if kernel == "fwd_long":
        return 0 if dims < 128 or not (drop or bias and parts) else (164, 296)[parts] if drop else (0, 20)[parts]
    if kernel == "bwd_short":
        if dims == 128:
            return (276, 228)[parts] if tiles == 1 else (1516, 776)[parts] if group else (356, 288)[parts]
        if tiles == 1:
            return 0
        if dims == 64:
            return 204 if group else 0 if bias else 108 if drop else 8 * half
        return 0 if not group or bias else 104 if drop else 40 * half
    if kernel == "bwd_kv":
        return (0 if dims == 32 else 172 if bias or drop else 0) if dims < 128 else (288, 292)[parts]
    return 0 if dims < 128 else (340, 540)[parts]


def test_typed_kernels_take_no_more_scratch(tmp_path):
    """Reloads in a pairs' loop cost its time; what the kernels of 64 and 128 dims take is known and does not grow."""
    sizes, seen = kernels(tmp_path), 0
    for name, size in sizes.items():
        m = re.search(r"typed_(fwd_short|fwd_long|bwd_short|bwd_kv|bwd_q)_kernelIDF16(b|_)Li(\d+)E(?:Li(\d)E)?((?:Lb[01]E)+)", name)
        if not m:
            continue
        flags = [f == "1" for f in re.findall(r"Lb([01])E", m[5])]
        group = flags.pop(0) if m[1] == "bwd_short" else False
        seen += 1
        assert size <= most_scratch(m[1], int(m[3]), int(m[4] or 0), group, *flags, m[2] == "_"), (name, size)
    assert seen == 224
