"""A training step through the C++ interface (include/pet/train.hpp, compiled
into tests/cpp/train_test) gives the bits of the Python calls on the same data."""
from __future__ import annotations

import os
import subprocess

import numpy as np
import pytest
import torch

from pet_kokkos_amd import attention as A
from pet_kokkos_amd import build as B
from pet_kokkos_amd import grads as G
from pet_kokkos_amd import layer as L
from pet_kokkos_amd import linear as D
from pet_kokkos_amd import systems

pytestmark = pytest.mark.gpu


def test_cpp_training_step(device, tmp_path):
    if not os.path.exists(B.CPP_TEST4):
        pytest.fail(f"{B.CPP_TEST4} is not built (python -m pet_kokkos_amd.build)")
    rng = np.random.default_rng(41)
    H, hd = 2, 32
    d = H * hd
    tk = systems.tokens_from_counts([7, 1, 30, 12], seed=3)
    N, T, S = tk.n_atoms, tk.n_rows, tk.slots
    a = {"tokens": rng.standard_normal((T, d)), "g": rng.standard_normal((T, d)), "nw": 1 + 0.1 * rng.standard_normal(d),
         "nb": 0.1 * rng.standard_normal(d), "w_in": rng.standard_normal((3 * d, d)) / 8, "b_in": rng.standard_normal(3 * d),
         "w_out": rng.standard_normal((d, d)) / 8, "b_out": rng.standard_normal(d), "cf": tk.cf_seq}
    a = {k: np.ascontiguousarray(v, dtype=np.float32) for k, v in a.items()}
    for k, v in a.items():
        v.tofile(tmp_path / f"{k}.f32")
    np.ascontiguousarray(tk.off, dtype=np.int32).tofile(tmp_path / "off.i32")
    print("[gpu] C++ training step", flush=True)
    res = subprocess.run([B.CPP_TEST4, str(tmp_path), str(N), str(T), str(S), str(H), str(hd)], capture_output=True,
                         text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    t = {k: torch.from_numpy(v).to(device) for k, v in a.items()}
    tok, ws = A.Tokens(torch.from_numpy(tk.off).to(device), N), A.Workspace(device)
    out, tadj, csa = torch.empty((T, d), device=device), torch.zeros((T, d), device=device), torch.zeros((N, S), device=device)
    L.attention_layer(ws, "l", out, t["tokens"], t["nw"], t["nb"], t["w_in"], t["b_in"], t["cf"], t["w_out"], t["b_out"], tok,
                      S, H, hd, 1.0)
    new = lambda *s: torch.zeros(s, device=device)
    g = {"norm_w": new(d), "norm_b": new(d), "w_in": new(3 * d, d), "b_in": new(3 * d), "w_out": new(d, d), "b_out": new(d)}
    L.attention_layer_grads(ws, "l", g, tadj, csa, t["g"], t["tokens"], t["nw"], t["nb"], t["w_in"], t["b_in"], t["cf"],
                            t["w_out"], tok, S, H, hd, 1.0)
    more = [new(d, d), new(d), new(d), new(d)]
    D.linear_grads(t["g"], t["tokens"], more[0], more[1])
    L.norm_rows_grads(None, more[2], more[3], t["g"], t["tokens"], t["nw"], True)
    grads = [*g.values(), *more]
    norm = G.clip_grads(grads, 1.0)
    flat = torch.cat([x.flatten() for x in grads]).cpu().numpy()
    assert np.array_equal(np.fromfile(tmp_path / "grads.f32", dtype=np.float32), flat)
    assert np.array_equal(np.fromfile(tmp_path / "tokens_adj.f32", dtype=np.float32), tadj.cpu().numpy().ravel())
    assert np.fromfile(tmp_path / "norm.f32", dtype=np.float32)[0] == norm.item() > 1.0
