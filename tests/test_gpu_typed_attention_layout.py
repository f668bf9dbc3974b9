"""What the typed attention writes and what it leaves alone, where offsets promise more
than there is; heads and layouts that no other test of it has."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from pet_kokkos_amd import _lib
from pet_kokkos_amd import attention as A
from test_gpu_typed_attention import BF16, F16, OnDevice, within
from typed_attention import Case

pytestmark = pytest.mark.gpu


class Cut(Case):
    """A case whose offsets are replaced: an atom's tokens are cut to the slots and the rows."""

    def __init__(self, off, slots, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.off, self.S = np.array(off, dtype=np.int32), slots
        self.cf = torch.ones((self.N, self.S))

    def rows(self, n):
        first, last = int(self.off[n]), int(self.off[n + 1])
        edges = min(last - first, self.S - 1, self.T - self.N - first)
        return [n] + ([self.N + first + i for i in range(edges)] if first >= 0 else [])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("off,counts,slots,heads,kv_heads", [
    ([0, 9, 24, 4000], [9, 11, 5], 12, 2, 2), ([-4, 2 ** 30, 7, 7], [9, 11, 5], 12, 2, 2), ([3, 9, 9, 20], [9, 11, 5], 30, 4, 2),
    ([0, 200, 411, 616], [200, 211, 205], 150, 2, 1), ([0, 200, 411, 4000], [200, 211, 205], 190, 2, 2),
    ([5, 200, 380, 500], [200, 211, 205], 300, 4, 1), ([-4, 2 ** 30, 7, 7], [200, 211, 205], 212, 2, 2)])
def test_rows_of_no_atom_are_left_as_they_were(device, dtype, off, counts, slots, heads, kv_heads):
    """Offsets past the slots or the rows are cut, ones that are no range give an atom its own token; the rows that are
    then no atom's, the columns beside the rows and what lies around them keep what they held, whatever the scratch holds."""
    case = Cut(off, slots, counts, heads, kv_heads, 32, dtype, buckets=8, reach=9, p=0.1)
    d = OnDevice(case, device, pad=5, shift=3)
    mine = sorted(r for n in range(case.N) for r in case.rows(n))
    assert len(set(mine)) == len(mine) < case.T
    others = torch.ones(case.T, dtype=torch.bool)
    others[mine] = False
    nbytes = _lib.load().pet_attn_bwd_typed_workspace(A.DTYPES[dtype], A.shape(case.N, case.T, case.S, heads, 32), kv_heads, 8)
    scratch = torch.full((nbytes + 512,), 255, dtype=torch.uint8, device=device)
    d.forward(), d.backward(scratch=scratch[:nbytes])
    assert (scratch[nbytes:] == 255).all()
    for view in (d.merged, d.adj):
        assert (view[others.to(device)] == 3).all()
        whole = torch.as_strided(view, (view.shape[0], view.shape[1] + 5), (view.stride(0), 1))
        assert torch.isnan(whole[:, view.shape[1]:]).all()
        before = torch.as_strided(view, (3,), (1,), 0)
        assert torch.isnan(before).all()
    out, tol, ml, ml_tol = case.forward()
    within(d.merged[mine], out[mine], tol[mine], "merged")
    within(d.ml, ml, ml_tol, "ml")
    got = {"qkv_adj": d.adj[mine], "cf_seq_adj": d.cf_adj, "bias_adj": d.table_adj}
    for name, (ref, bound) in case.backward(d.merged.cpu()).items():
        if name == "qkv_adj":
            ref, bound = ref[mine], bound[mine]
        within(got[name], ref, bound, name)


@pytest.mark.parametrize("kv_heads", [1, 4100])
@pytest.mark.parametrize("buckets", [0, 2])
def test_more_heads_and_atoms_than_a_grid_holds(device, kv_heads, buckets):
    """A workgroup goes through as many atoms more as the grid has fewer of them."""
    OnDevice(Case([0] * 2100, 4100, kv_heads, 1, BF16, buckets=buckets, reach=buckets // 2), device).check()


def test_more_heads_and_atoms_than_a_grid_holds_past_128_slots(device):
    """The bits of a call are those of the calls on its halves, whose grids are whole."""
    H, N, S = 4100, 1100, 130
    gen = torch.Generator().manual_seed(0)
    qkv = torch.randn(N, H + 2, generator=gen).to(BF16).to(device)
    g = torch.randn(N, H, generator=gen).to(BF16).to(device)
    cf = torch.zeros(N, S, device=device)
    cf[:, 0] = 1.0

    def call(at):
        n = len(range(N)[at])
        off = torch.zeros(n + 1, dtype=torch.int32, device=device)
        merged, ml = A.attn_fwd_typed(qkv[at], off, cf[at], H, 1, kv_heads=1)
        adj, cf_adj, _ = A.attn_bwd_typed(qkv[at], off, g[at], merged, ml, cf[at], H, 1, kv_heads=1,
                                          cf_seq_adj=torch.empty(n, S, device=device))
        return merged, adj, cf_adj
    whole, halves = call(slice(0, N)), [call(slice(0, N // 2)), call(slice(N // 2, N))]
    for x, *parts in zip(whole, *halves):
        assert torch.equal(x, torch.cat(parts))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias,p", [(False, 0.0), (True, 0.0), (False, 0.3), (True, 0.3)])
@pytest.mark.parametrize("kv_heads", [1, 2])
@pytest.mark.parametrize("head_dim", [72, 80, 96, 100, 128])
def test_wide_heads_of_65_to_128_slots(device, dtype, bias, p, kv_heads, head_dim):
    """Two tiles of keys a wave at 128 dims, with what an atom is staged from in more than one round."""
    OnDevice(Case([64, 70, 100, 127, 3], 2, kv_heads, head_dim, dtype, seed=head_dim, buckets=20 if bias else 0,
                  reach=40 if bias else 0, p=p, zeros=0.1, dead=2), device).check()


@pytest.mark.parametrize("kv_heads", [1, 2])
def test_the_most_of_a_workgroups_memory(device, kv_heads):
    """128 slots of heads of 128, 64 buckets and a reach of 1024."""
    case = Case([127, 20, 90], 2, kv_heads, 128, BF16, seed=4, buckets=64, reach=1024, p=0.1)
    OnDevice(case, device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [20, 33, 50, 16, 48, 80, 96])
@pytest.mark.parametrize("counts", [[70, 127, 2], [140, 300]])
def test_heads_between_the_instances(device, dtype, head_dim, counts):
    OnDevice(Case(counts, 4, 2, head_dim, dtype, seed=head_dim, buckets=9, reach=12, p=0.2, zeros=0.1), device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 4, 32), (8, 2, 128), (6, 3, 20)])
def test_many_small_molecules(device, dtype, heads, kv_heads, head_dim):
    """More atoms of up to 16 tokens than workgroups: one wave each, grouped heads and a table in turn."""
    rng = np.random.default_rng(5)
    OnDevice(Case(rng.integers(3, 16, 1500), heads, kv_heads, head_dim, dtype, seed=6, buckets=9, reach=7, p=0.1, zeros=0.1,
                  slots=16), device).check()
