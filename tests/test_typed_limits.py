"""Sizes of the typed attention past an int's and results over operands, without a GPU."""
from __future__ import annotations

import os
import subprocess

import pytest

from pet_kokkos_amd import _lib, build
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
