"""Sizes of the typed attention past an int's, without a GPU."""
from __future__ import annotations

import os
import subprocess

import pytest

from pet_kokkos_amd import build


def test_cpp_calls_refuse_products_past_an_int():
    if not os.path.exists(build.CPP_TEST7):
        pytest.fail(f"{build.CPP_TEST7} is not built (python -m pet_kokkos_amd.build)")
    res = subprocess.run([build.CPP_TEST7], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout == "", res.stdout + res.stderr
