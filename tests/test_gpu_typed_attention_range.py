"""The typed attention's backward where its numbers span a wide range: probabilities far
under 1 in fp16, adjoints of other sizes from head to head and atom to atom, infinities
and NaN in some of them. Bounds as in tests/typed_attention.py, without what it allows
fp16's smallest probabilities and the table's sums."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from pet_kokkos_amd import attention as A
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


def table_adjoint(case, merged):
    """The table's adjoint and its bound: each dS is off as in typed_attention.py and rounded to a whole number of a
    unit, of which a bound of the dS of its atom and head holds 2^27 or more (past 128 slots 2^30); where that bound
    passes fp32's range they are added in float64. Sums of whole numbers are exact, the result is rounded to fp32.
    A bucket with a dS that is not finite is not finite either."""
    H, hd = case.H, case.hd
    nb = case.table.shape[0]
    tab, err = torch.zeros((nb, H), dtype=torch.float64), torch.zeros((nb, H), dtype=torch.float64)
    long = case.S > 128
    for n in range(case.N):
        rows, q, k, v, cf, keys, queries, index, mask, prob, top, total, some, e_p = case.attend(n)
        c = len(rows)
        do, o = (torch.where(queries[:, None], x[rows].double(), 0.0).view(c, H, hd).transpose(0, 1)
                 for x in (case.dmerged, merged))
        m = 1.0 if mask is None else mask
        most = 1.0 if mask is None else float(mask.max())
        dp, dp_mag = m * (do @ v.transpose(1, 2)), m * (do.abs() @ v.abs().transpose(1, 2))
        d, d_mag = (do * o).sum(-1, keepdim=True), (do * o).abs().sum(-1, keepdim=True)
        ds = prob * (dp - d)
        e_ds = e_p * prob * (dp.abs() + d.abs()) + (hd + 8) * U * prob * (dp_mag + d_mag)
        if long:
            bound = do.norm(dim=-1).amax(1) * v.norm(dim=-1).amax(1) * most + d.abs().amax((1, 2))
        else:
            bound = hd * do.abs().amax((1, 2)) * v.abs().amax((1, 2)) * most + d.abs().amax((1, 2))
        bound = torch.where(bound < 2.0 ** 128, bound, 0.0)  # (a NaN is not less)
        step = bound * 2.0 ** (-31 if long else -28) * (1 + 2.0 ** -10) + 2.0 ** -126
        for b in range(nb):
            at = index == b
            tab[b] += torch.where(at, ds, 0.0).sum((1, 2))
            err[b] += torch.where(at, e_ds + step[:, None, None], 0.0).sum((1, 2))
    return tab, err + 2 * U * tab.abs() + 2.0 ** -149


def check_table(d, where=""):
    """Runs the case; the table's adjoint against its bound, buckets that are not finite by their formula apart."""
    d.forward(), d.backward()
    ref, tol = table_adjoint(d.case, d.merged.cpu())
    some = torch.isfinite(ref)
    got = d.table_adj.double().cpu()
    assert torch.equal(torch.isfinite(got), some), where
    within(torch.where(some, got, 0.0), torch.where(some, ref, 0.0), torch.where(some, tol, 0.0), f"{where} bias_adj")
    return some


LAYOUTS = [([700], 4, 4, 32), ([300, 140, 20], 4, 2, 32), ([60, 127], 4, 4, 32), ([60, 100], 4, 2, 64), ([30, 9], 4, 1, 16)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", LAYOUTS)
def test_the_tables_sums_are_as_good_as_their_pairs(device, dtype, p, counts, heads, kv_heads, head_dim):
    check_table(OnDevice(Case(counts, heads, kv_heads, head_dim, dtype, seed=1, buckets=12, reach=30, p=p, zeros=0.1), device))


@pytest.mark.parametrize("dtype,step", [(BF16, -20), (BF16, 20), (F16, -5), (F16, 5)])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", LAYOUTS)
def test_heads_with_adjoints_of_other_sizes(device, dtype, step, counts, heads, kv_heads, head_dim):
    case = Case(counts, heads, kv_heads, head_dim, dtype, seed=1, buckets=12, reach=30)
    for h in range(heads):
        at = slice(h * head_dim, (h + 1) * head_dim)
        case.dmerged[:, at] = (case.dmerged[:, at].double() * 2.0 ** (step * h)).to(dtype)
    check_table(OnDevice(case, device))


def tiers(counts, heads, kv_heads, head_dim, dtype, size):
    """Atoms in thirds: those of third t have adjoints times size(t) and positions 0 and t + 1, a bucket an offset."""
    case = Case(counts, heads, kv_heads, head_dim, dtype, seed=2, buckets=9, reach=4)
    case.buckets = torch.arange(9, dtype=torch.int32)
    rng = np.random.default_rng(1)
    for n in range(case.N):
        t, rows = 3 * n // case.N, case.rows(n)
        case.pos[rows] = torch.from_numpy(rng.integers(0, 2, len(rows)) * (t + 1)).int()
        case.dmerged[rows] = (case.dmerged[rows].double() * size(t)).to(dtype)
    return case


MANY = [([5] * 420, 32, 32, 8), ([9] * 420, 64, 32, 8), ([130] * 24, 32, 32, 8), ([140] * 18, 32, 16, 8)]


@pytest.mark.parametrize("dtype,step", [(BF16, 24), (BF16, -24), (F16, 5), (F16, -5)])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", MANY)
def test_atoms_with_adjoints_of_other_sizes(device, dtype, step, counts, heads, kv_heads, head_dim):
    """More atoms than workgroups, adjoints growing or shrinking from one of a workgroup's atoms to its next."""
    check_table(OnDevice(tiers(counts, heads, kv_heads, head_dim, dtype, lambda t: 2.0 ** (step * (t - 1))), device))


@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", LAYOUTS)
def test_adjoints_at_the_end_of_the_range(device, counts, heads, kv_heads, head_dim):
    case = Case(counts, heads, kv_heads, head_dim, BF16, seed=1, buckets=12, reach=30)
    case.dmerged = (case.dmerged.double() * 2.0 ** -100).to(BF16)
    check_table(OnDevice(case, device))


@pytest.mark.parametrize("size", [-100, 100])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", [([699], 4, 4, 32), ([299, 141], 4, 2, 20), ([59, 127], 4, 2, 32)])
def test_adjoints_at_the_ends_of_the_range_and_none_of_the_result(device, size, counts, heads, kv_heads, head_dim):
    """The values' mean is 0, so dO.O is 0 and the bound is of dO and the values alone."""
    case = Case(counts, heads, kv_heads, head_dim, BF16, seed=1, buckets=12, reach=30)
    case.table[:] = 0.0
    case.cf[:] = (case.cf > 0).float()
    case.qkv[:, heads * head_dim:(heads + kv_heads) * head_dim] = 0.0
    for n in range(case.N):
        rows = case.rows(n)
        case.qkv[rows[1::2], (heads + kv_heads) * head_dim:] = -case.qkv[rows[::2], (heads + kv_heads) * head_dim:]
    case.dmerged = (case.dmerged.double() * 2.0 ** size).to(BF16)
    check_table(OnDevice(case, device))


@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", LAYOUTS + MANY)
def test_a_bound_past_the_range(device, counts, heads, kv_heads, head_dim):
    """Adjoints and values whose largest have no dim in common: their products' bound overflows, no product does."""
    case = tiers(counts, heads, kv_heads, head_dim, BF16, lambda t: 1.0)
    rows, width = case.rows(0), heads * head_dim
    for h in range(heads):
        case.dmerged[rows, h * head_dim] *= 2.0 ** 70
        case.dmerged[rows, h * head_dim + 1] = 0.0
    for k in range(kv_heads):
        at = width + (kv_heads + k) * head_dim
        case.qkv[rows, at] = 0.0
        case.qkv[rows, at + 1] *= 2.0 ** 70
    d = OnDevice(case, device)
    check_table(d)
    for _ in range(3):
        first = d.table_adj.clone()
        d.backward()
        assert torch.equal(first, d.table_adj)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("what", ["adjoint", "value"])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", [([60, 127], 4, 2, 32), ([300, 140, 20], 4, 2, 32), *MANY])
def test_what_is_not_finite_stays_in_its_head_and_buckets(device, dtype, bad, what, counts, heads, kv_heads, head_dim):
    case = tiers(counts, heads, kv_heads, head_dim, dtype, lambda t: 1.0)
    case.pos[case.rows(0)] = 0  # (all pairs of the atom in one bucket)
    row, head = case.rows(0)[3], 2
    if what == "adjoint":
        case.dmerged[row, head * head_dim + 1] = bad
    else:
        case.qkv[row, (heads + kv_heads + head * kv_heads // heads) * head_dim + 1] = bad
    some = check_table(OnDevice(case, device), what)
    gone = heads // kv_heads if what == "value" else 1
    assert int((~some).sum()) == gone and not some[4, head]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("atoms,tokens", [(10000, 128), (600, 512)])
def test_the_products_roundings_do_not_add_up(device, dtype, atoms, tokens):
    """1.6e8 pairs of one bucket. Logits are 0, so P is 1 / tokens, a power of two, and exact. Of hd products each dP
    has at most hd roundings of at most U of its magnitudes' sum; with none of them favoured, their square is a third
    of that on the mean, and so is that of dO.O's, of dS's own (U of itself) and a unit's half: 6 of their deviations. (The
    atoms' bounds are within 2 of each other, so a unit is at most twice the fitting one.)"""
    hd = 32
    gen = torch.Generator(device).manual_seed(0)
    T, edges = atoms * tokens, tokens - 1
    qkv = torch.zeros(T, 3 * hd, dtype=dtype, device=device)
    qkv[:, 2 * hd:] = (torch.randn(T, hd, generator=gen, device=device).clamp(-3, 3) * 0.7).to(dtype)
    g = (torch.randn(T, hd, generator=gen, device=device).clamp(-3, 3) * 0.05).to(dtype)
    off = torch.arange(atoms + 1, dtype=torch.int32, device=device) * edges
    cf = torch.ones(atoms, tokens, device=device)
    bias = A.RelativeBias(torch.zeros(1, 1, device=device), torch.zeros(1, dtype=torch.int32, device=device),
                          torch.zeros(T, dtype=torch.int32, device=device))
    merged, ml = A.attn_fwd_typed(qkv, off, cf, 1, hd, bias=bias)
    assert (ml[:, 1] == 1 / tokens).all() and (ml[:, 0] == 0).all()
    table = torch.zeros(1, 1, device=device)
    A.attn_bwd_typed(qkv, off, g, merged, ml, cf, 1, hd, bias=bias, bias_adj=table)

    def by_atom(x):  # [atoms, tokens, hd]
        return torch.cat([x[:atoms, None], x[atoms:].view(atoms, edges, hd)], 1).double()
    v, do, o = (by_atom(x) for x in (qkv[:, 2 * hd:], g, merged))
    d, d_mag = (do * o).sum(-1), (do * o).abs().sum(-1)
    ref = ((do * v.sum(1, keepdim=True)).sum(-1) / tokens - d).sum()

    def squares(x, y):  # of x_i.y_j over all pairs of an atom
        return (torch.bmm(x.transpose(1, 2).contiguous(), x) * torch.bmm(y.transpose(1, 2).contiguous(), y)).sum()
    bound = (hd * do.abs().amax((1, 2)) * v.abs().amax((1, 2)) + d.abs().amax(1))
    assert float(bound.max()) <= 2 * float(bound.min())
    unit = bound.max() * 2.0 ** (-32 if tokens <= 128 else -35)
    variance = ((hd / 3) * U ** 2 * squares(do.abs(), v.abs()) + 2 * U ** 2 * (squares(do, v) + tokens * (d ** 2).sum())) / tokens ** 2 \
        + (hd / 3) * U ** 2 * (d_mag ** 2).sum() + atoms * tokens ** 2 * unit ** 2 / 12
    error = float(table.double()[0, 0] - ref)
    assert abs(error) <= 6 * math.sqrt(float(variance)) + U * abs(float(ref)), (error, math.sqrt(float(variance)), float(ref))
