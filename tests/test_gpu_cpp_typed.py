"""The typed attention, its backward and the dropout through the C++ interface
(include/pet/train.hpp, compiled into tests/cpp/typed_attention_test) give the bits of
the Python calls on the same data."""
from __future__ import annotations

import os
import subprocess

import numpy as np
import pytest
import torch

from pet_kokkos_amd import attention as A
from pet_kokkos_amd import build as B
from pet_kokkos_amd import layer as L
from pet_kokkos_amd import systems

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[7, 1, 0, 30, 12], [150, 3]])
def test_cpp_typed_attention(device, tmp_path, counts):
    if not os.path.exists(B.CPP_TEST6):
        pytest.fail(f"{B.CPP_TEST6} is not built (python -m pet_kokkos_amd.build)")
    rng = np.random.default_rng(43)
    H, Hk, hd, nb, R = 4, 2, 24, 6, 9
    D, W = H * hd, (H + 2 * Hk) * hd
    tk = systems.tokens_from_counts(counts, seed=3)
    N, T, S = tk.n_atoms, tk.n_rows, tk.slots
    bf = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(torch.bfloat16)
    qkv, g = bf(T, W), bf(T, D)
    f32 = {"cf": np.ascontiguousarray(tk.cf_seq, dtype=np.float32), "table": rng.standard_normal((nb, H)).astype(np.float32)}
    i32 = {"off": np.ascontiguousarray(tk.off, dtype=np.int32), "buckets": rng.integers(0, nb, 2 * R + 1).astype(np.int32),
           "pos": rng.integers(-20, 20, T).astype(np.int32)}
    state = np.array([12345678901, 7], dtype=np.int64)
    for k, v in {"qkv": qkv, "g": g}.items():
        v.view(torch.int16).numpy().tofile(tmp_path / f"{k}.b16")
    for k, v in f32.items():
        v.tofile(tmp_path / f"{k}.f32")
    for k, v in i32.items():
        v.tofile(tmp_path / f"{k}.i32")
    state.tofile(tmp_path / "state.i64")
    print("[gpu] C++ typed attention", counts, flush=True)
    res = subprocess.run([B.CPP_TEST6, str(tmp_path), *(str(x) for x in (N, T, S, H, Hk, hd, nb, R))], capture_output=True,
                         text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    t = {k: torch.from_numpy(v).to(device) for k, v in {**f32, **i32}.items()}
    st = torch.from_numpy(state).to(device)
    qkv, g = qkv.to(device), g.to(device)
    bias = A.RelativeBias(t["table"], t["buckets"], t["pos"])
    first, second = A.Dropout(0.25, st, 1), A.Dropout(0.25, st, 2)
    args = dict(kv_heads=Hk, bias=bias, dropout=first)
    merged, ml = torch.zeros((T, D), dtype=torch.bfloat16, device=device), torch.zeros((N * H * S, 2), device=device)
    A.attn_fwd_typed(qkv, t["off"], t["cf"], H, hd, merged=merged, ml=ml, **args)
    rows = torch.zeros_like(merged)
    L.dropout_rows(rows, merged, second, residual=g)
    adj = torch.zeros((T, W), dtype=torch.bfloat16, device=device)
    csa, ta = torch.zeros((N, S), device=device), torch.zeros((nb, H), device=device)
    A.attn_bwd_typed(qkv, t["off"], rows, merged, ml, t["cf"], H, hd, qkv_adj=adj, cf_seq_adj=csa, bias_adj=ta, **args)
    for name, x in {"merged": merged, "rows": rows, "qkv_adj": adj}.items():
        got = np.fromfile(tmp_path / f"{name}.b16", dtype=np.int16)
        assert np.array_equal(got, x.view(torch.int16).cpu().numpy().ravel()), name
    for name, x in {"ml": ml, "cf_adj": csa, "table_adj": ta}.items():
        assert np.array_equal(np.fromfile(tmp_path / f"{name}.f32", dtype=np.float32), x.cpu().numpy().ravel()), name
