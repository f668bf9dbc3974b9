"""The typed attention's backward where its numbers span a wide range: probabilities far
under 1 in fp16. Bounds as in tests/typed_attention.py, without what it allows fp16's
smallest probabilities."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_typed_attention import BF16, F16, OnDevice, within
from typed_attention import U, Case, half

pytestmark = pytest.mark.gpu


def values_adjoint(case, merged):
    """dV and its bound: P M is rounded to the type at a scale that brings 1 / (1 - p) to
    2^13 .. 2^14, so by h of itself or, under 2^-14 there, by 2^-25 2^-13 of 1 / (1 - p)."""
    H, Hk, hd, h = case.H, case.Hk, case.hd, half(case.dtype)
    G = H // Hk
    adj, tol = (torch.zeros((case.T, Hk * hd), dtype=torch.float64) for _ in range(2))
    for n in range(case.N):
        rows, q, k, v, cf, keys, queries, index, mask, prob, top, total, some, e_p = case.attend(n)
        c = len(rows)
        do = torch.where(queries[:, None], case.dmerged[rows].double(), 0.0).view(c, H, hd).transpose(0, 1)
        pm = prob * (1.0 if mask is None else mask)
        few = 2.0 ** -38 * (1.0 if mask is None else float(mask.max())) if case.dtype == F16 else 0.0
        dv, dv_t = pm.transpose(1, 2) @ do, ((h + e_p + (G * c + 4) * U) * pm + few).transpose(1, 2) @ do.abs()

        def grouped(x):
            return (x * keys[None, :, None]).reshape(Hk, G, c, hd).sum(1).transpose(0, 1).reshape(c, -1)
        adj[rows], tol[rows] = grouped(dv), grouped(dv_t)
    return adj, tol + h * adj.abs() + 4 * torch.finfo(case.dtype).smallest_normal * h


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("p", [0.0, 0.25, 0.9])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", [([2500], 2, 1, 32), ([2000, 3], 1, 1, 128), ([300, 40], 4, 4, 20),
                                                            ([100, 60], 2, 2, 64), ([90, 127], 4, 2, 32), ([30, 9], 2, 1, 16)])
def test_keys_of_small_probability(device, dtype, p, counts, heads, kv_heads, head_dim):
    """Half of the keys near the cutoff, at factors of 1e-6 to 1e-3: their probabilities lie under fp16's 2^-14, most
    under its 2^-25, and their values' adjoints are sums of them times adjoints of one sign."""
    case = Case(counts, heads, kv_heads, head_dim, dtype, seed=head_dim, p=p)
    rng = np.random.default_rng(0)
    for n, c in enumerate(counts):
        near = torch.from_numpy(rng.random(c) < 0.5)
        far = torch.from_numpy(10.0 ** rng.uniform(-6, -3, c)).float()
        case.cf[n, 1:c + 1] = torch.where(near, case.cf[n, 1:c + 1], far)
    case.dmerged = (case.dmerged.double() * 40 + 32).to(dtype)
    d = OnDevice(case, device)
    d.forward(), d.backward()
    ref, tol = values_adjoint(case, d.merged.cpu())
    within(d.adj[:, (heads + kv_heads) * head_dim:], ref, tol, "dV")
