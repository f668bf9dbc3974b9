"""Attention of 16-bit rows, its backward and dropout on the GPU, each against its
formula in 64 bits at bounds counted from the roundings (tests/typed_attention.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from pet_kokkos_amd import _lib
from pet_kokkos_amd import attention as A
from pet_kokkos_amd import layer as L
from typed_attention import U, Case, half, rows_mask

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def within(got, ref, tol, what):
    got = got.double().cpu()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), what
    excess = (got - ref).abs() - tol
    i = int(excess.argmax())
    assert excess.flatten()[i] <= 0, f"{what}[{i}]: {got.flatten()[i]} against {ref.flatten()[i]}, allowed {tol.flatten()[i]}"


class OnDevice:
    """A Case's tensors on the device and the calls on them; pad: columns past each row's end."""

    def __init__(self, case, device, pad=0, shift=0):
        self.case, self.dev = case, device

        def rows(x):
            buf = torch.full((x.shape[0] * (x.shape[1] + pad) + shift + 8,), math.nan, dtype=x.dtype, device=device)
            v = buf[shift:shift + x.shape[0] * (x.shape[1] + pad)].view(x.shape[0], -1)[:, :x.shape[1]]
            v.copy_(x)
            return v
        self.rows = rows
        self.qkv, self.dmerged = rows(case.qkv), rows(case.dmerged)
        self.off, self.cf = torch.from_numpy(case.off).to(device), case.cf.to(device)
        self.bias = None
        if case.table is not None:
            if case.buckets is None:
                case.buckets = A.relative_buckets(case.table.shape[0], case.reach)
            self.bias = A.RelativeBias(case.table.to(device), case.buckets.to(device), case.pos.to(device))
        self.drop = A.Dropout(case.p, torch.tensor(case.state, dtype=torch.int64, device=device), case.call) if case.p else None
        self.merged = rows(torch.full((case.T, case.H * case.hd), 3.0, dtype=case.dtype))
        self.ml = torch.full((case.N * case.H * case.S, 2), math.nan, device=device)
        self.adj = rows(torch.full(case.qkv.shape, 3.0, dtype=case.dtype))
        self.cf_adj = torch.full((case.N, case.S), math.nan, device=device)
        self.table_adj = None if case.table is None else torch.full(case.table.shape, math.nan, device=device)

    def forward(self):
        c = self.case
        return A.attn_fwd_typed(self.qkv, self.off, self.cf, c.H, c.hd, c.temperature, c.Hk, self.bias, self.drop,
                                dead=c.dead > 0, merged=self.merged, ml=self.ml)

    def backward(self, beta=0.0, scratch=None):
        c = self.case
        return A.attn_bwd_typed(self.qkv, self.off, self.dmerged, self.merged, self.ml, self.cf, c.H, c.hd,
                                c.temperature, c.Hk, self.bias, self.drop, self.adj, self.cf_adj, self.table_adj, beta,
                                dead=c.dead > 0, scratch=scratch)

    def check(self, what=""):
        out, tol, ml, ml_tol = self.case.forward()
        self.forward()
        within(self.merged, out, tol, f"{what} merged")
        within(self.ml, ml, ml_tol, f"{what} ml")
        self.backward()
        got = {"qkv_adj": self.adj, "cf_seq_adj": self.cf_adj, "bias_adj": self.table_adj}
        for name, (ref, bound) in self.case.backward(self.merged.cpu()).items():
            within(got[name], ref, bound, f"{what} {name}")


SMALL = [4, 0, 8, 1, 33, 15, 16]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [1, 8, 16, 24, 32, 33, 64, 80, 100, 128])
def test_head_dims(device, dtype, head_dim):
    OnDevice(Case(SMALL, 2, 2, head_dim, dtype, seed=head_dim), device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts", [[0], [0, 0, 0], [14], [15], [16], [31], [32], [62], [63], [64], [65], [127], [128], [129],
                                    [255, 3], [300, 0, 129, 128, 127], [700]])
def test_lengths(device, dtype, counts):
    OnDevice(Case(counts, 2, 1, 32, dtype, seed=len(counts) + counts[0], buckets=8, reach=20, p=0.2, zeros=0.1), device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.75])
@pytest.mark.parametrize("heads,kv_heads,head_dim,counts", [(4, 4, 32, SMALL), (6, 2, 40, [70, 3, 150]), (4, 1, 128, [20, 90, 200]),
                                                            (8, 8, 64, [40, 70, 55, 10])])
def test_variants(device, dtype, bias, p, heads, kv_heads, head_dim, counts):
    OnDevice(Case(counts, heads, kv_heads, head_dim, dtype, seed=heads, buckets=32 if bias else 0, reach=50 if bias else 0,
                  p=p, zeros=0.15, dead=5, temperature=1.3), device).check()


@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (3, 3), (8, 8)])
@pytest.mark.parametrize("head_dim", [24, 32, 50])
def test_strides_and_alignments(device, pad, shift, head_dim):
    OnDevice(Case(SMALL + [140], 3, 1, head_dim, BF16, seed=pad, dead=2, slots=200), device, pad, shift).check()


@pytest.mark.parametrize("buckets,reach", [(1, 0), (2, 1), (17, 50), (64, 1024), (32, 5)])
@pytest.mark.parametrize("group", [1, 2])
def test_tables(device, buckets, reach, group):
    OnDevice(Case([60, 3, 140], 4, 4 // group, 32, BF16, seed=buckets, buckets=buckets, reach=reach), device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim,counts,slots", [
    (1, 1, 32, [700], None), (1, 1, 128, [1100], None), (2, 1, 64, [520, 3], None), (3, 3, 48, [600, 0, 129], None),
    (4, 2, 33, [150, 300], None), (2, 2, 100, [200, 1], None), (2, 1, 116, [530], None), (2, 1, 32, [3, 0, 40], 1500)])
def test_long_passes_in_parts(device, dtype, heads, kv_heads, head_dim, counts, slots):
    """Heads and queries shared out among workgroups, heads in odd pieces, a few tokens in many slots."""
    OnDevice(Case(counts, heads, kv_heads, head_dim, dtype, seed=head_dim, buckets=9, reach=30, p=0.2, zeros=0.1, dead=4,
                  slots=slots), device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,heads,kv_heads,head_dim", [(SMALL, 4, 4, 32), ([50, 127, 3], 4, 2, 64), ([200, 17], 4, 1, 128)])
def test_a_block_forward_and_backward(device, dtype, counts, heads, kv_heads, head_dim):
    """out = x + M2 attention(qkv) and its adjoints from out's. M2 of p = 1/2 is 0 or 2: the adjoint of merged is
    exact, and out is off by twice merged's bound and the rounding of itself."""
    case = Case(counts, heads, kv_heads, head_dim, dtype, seed=3, buckets=12, reach=9, p=0.125, zeros=0.1)
    out_adj = case.dmerged
    m2 = rows_mask(*case.state, 8, 0.5, case.T, heads * head_dim)
    case.dmerged = (m2 * out_adj.double()).to(dtype)
    d = OnDevice(case, device)
    x = torch.randn(case.T, heads * head_dim, generator=torch.Generator().manual_seed(1)).to(dtype)
    after = A.Dropout(0.5, d.drop.state, 8)
    d.forward()
    out = x.to(device)
    L.dropout_rows(out, d.merged, after, out)
    merged, tol, *_ = case.forward()
    ref = x.double() + m2 * merged
    within(out, ref, m2 * tol + half(dtype) * (ref.abs() + m2 * tol) + 2.0 ** -24 * (x.double().abs() + 2 * merged.abs()), "out")
    d.dmerged.fill_(math.nan)
    L.dropout_rows(d.dmerged, out_adj.to(device), after)
    assert torch.equal(d.dmerged.cpu(), case.dmerged)
    d.backward()
    for name, (want, bound) in case.backward(d.merged.cpu()).items():
        within({"qkv_adj": d.adj, "cf_seq_adj": d.cf_adj, "bias_adj": d.table_adj}[name], want, bound, name)


@pytest.mark.parametrize("edges,fine,unit", [(63, 26, 2.0 ** -30), (255, 30, 2.0 ** -36)])
def test_the_tables_sums_do_not_drift(device, edges, fine, unit):
    """Logits all 0, so P = 1 / tokens, and the values' sum 0, so dO.O = 0 but at the rows that set the sums' unit: every
    dS is exact, in quarters of a unit. Rounded to whole units each is off by 1/2 at most and by nothing on the mean,
    so n pairs by 6 * 0.36 sqrt(n) units (0.36: the root of a mean square of 1/8, of quarters as likely as each other)."""
    rng = np.random.default_rng(0)
    tokens, N, hd = edges + 1, 8, 8
    case = Case([edges] * N, 1, 1, hd, BF16, buckets=2, reach=1)
    qkv, g = torch.zeros(case.T, 3 * hd, dtype=torch.float64), torch.zeros(case.T, hd, dtype=torch.float64)
    case.table, case.buckets, case.cf = torch.zeros(2, 1), torch.tensor([0, 1, 1]).int(), torch.ones(N, tokens)
    exact = torch.zeros(2, dtype=torch.float64)
    for n in range(N):
        rows = case.rows(n)
        v = rng.integers(1, 128, tokens // 2)
        v = np.concatenate([v, -v])
        w = rng.integers(-127, 128, tokens)
        w[0] = 0
        qkv[rows, 2 * hd + 1] = torch.from_numpy(v * 2.0 ** -(fine // 2))
        qkv[rows[0], 2 * hd] = 1.0
        g[rows, 1] = torch.from_numpy(w * 2.0 ** -(fine // 2))
        g[rows[0], 0] = 1.0
        case.pos[rows] = torch.from_numpy(np.where(v > 0, 10, 0)).int()
    case.qkv, case.dmerged = qkv.to(BF16), g.to(BF16)
    d = OnDevice(case, device)
    d.forward(), d.backward()
    ref, _ = case.backward(d.merged.cpu())["bias_adj"]
    pairs = N * tokens ** 2
    within(d.table_adj, ref, 6 * 0.36 * math.sqrt(pairs) * unit + U * ref.abs(), "bias_adj")


def test_many_atoms_share_the_workgroups(device):
    """More items than workgroups: the table's sums run over several atoms in each."""
    rng = np.random.default_rng(3)
    OnDevice(Case(rng.integers(0, 12, 2500), 2, 2, 16, BF16, seed=1, buckets=9, reach=7, p=0.3), device).check()


def test_positions_at_the_ends_of_int32(device):
    case = Case([40], 2, 2, 32, BF16, buckets=16, reach=30)
    ends = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, 5, -2 ** 31 + 3, 2 ** 31 - 20], dtype=torch.int64)
    case.pos = ends[torch.arange(case.T) % 6].int()
    OnDevice(case, device).check()


def test_buckets_outside_the_table_count_as_its_ends(device):
    case = Case([50, 5], 2, 2, 32, F16, buckets=8, reach=10)
    case.buckets = torch.arange(-7, 14, dtype=torch.int32)
    OnDevice(case, device).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("counts", [[20, 0, 47], [200, 30]])
def test_masked_rows_hold_anything(device, dtype, bad, counts):
    """What edges at the cutoff and dead rows hold reaches no result, nor does a NaN cutoff factor's edge."""
    case = Case(counts, 4, 2, 32, dtype, zeros=0.3, dead=6, buckets=8, reach=9, p=0.1)
    d = OnDevice(case, device)
    cf = case.cf
    for n in range(case.N):
        for s, row in enumerate(case.rows(n)):
            if s and cf[n, s] == 0.0:
                d.qkv[row], d.dmerged[row] = bad, bad
                if s % 2:
                    d.cf[n, s] = math.nan
    d.qkv[case.T - 6:], d.dmerged[case.T - 6:] = bad, bad
    out, tol, ml, ml_tol = case.forward()
    d.forward()
    within(d.merged, out, tol, "merged")
    within(d.ml, ml, ml_tol, "ml")
    for n in range(case.N):
        for s, row in enumerate(case.rows(n)):
            if s and cf[n, s] == 0.0:
                d.merged[row] = bad
    d.backward()
    got = {"qkv_adj": d.adj, "cf_seq_adj": d.cf_adj, "bias_adj": d.table_adj}
    clean = torch.where(torch.isfinite(d.merged.cpu()), d.merged.cpu(), 0.0)
    for name, (ref, bound) in case.backward(clean).items():
        within(got[name], ref, bound, name)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_that_no_key_is_left_for(device, dtype):
    """An atom whose factors are all 0, and one whose own token's is: zeros, not NaN; (0, 0) in ml."""
    case = Case([20, 9, 0, 130], 2, 2, 32, dtype, buckets=4, reach=3, p=0.2)
    case.cf[0] = 0.0
    case.cf[1, 0] = 0.0
    case.cf[2] = 0.0
    d = OnDevice(case, device)
    d.check()
    assert (d.merged[case.rows(0)] == 0).all() and (d.adj[case.rows(0)] == 0).all()
    assert (d.ml.view(case.N, 2, case.S, 2)[0] == 0).all() and (d.ml.view(case.N, 2, case.S, 2)[2] == 0).all()


def test_a_bias_of_minus_infinity_leaves_keys_out(device):
    case = Case([20, 70], 2, 2, 32, BF16, buckets=8, reach=20)
    case.table[2] = -math.inf
    d = OnDevice(case, device)
    out, tol, ml, ml_tol = case.forward()
    d.forward()
    within(d.merged, out, tol, "merged")
    d.backward()
    assert torch.isfinite(d.adj).all() and torch.isfinite(d.table_adj).all() and (d.table_adj[2] == 0).all()


def test_a_table_that_leaves_a_query_nothing(device):
    case = Case([5], 2, 2, 32, BF16, buckets=2, reach=2)
    case.table[:] = -math.inf
    d = OnDevice(case, device)
    d.forward(), d.backward()
    assert (d.merged == 0).all() and (d.ml == 0).all() and (d.adj == 0).all() and (d.cf_adj == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_adjoints_of_any_size(device, dtype):
    """Adjoints far smaller and larger than their values: fp16's probabilities times small adjoints keep their bits."""
    for size in (2.0 ** -12, 1.0, 2.0 ** 9):
        case = Case([300, 20], 2, 1, 32, dtype, buckets=4, reach=6)
        case.dmerged = (case.dmerged.double() * size * 8).to(dtype)
        OnDevice(case, device).check(f"times {size}")


def test_large_logits(device):
    OnDevice(Case([90, 20], 2, 2, 64, BF16, size=4.0), device).check()


def test_beta_and_what_is_left_out(device):
    case = Case([20, 70, 3], 4, 2, 32, BF16, buckets=8, reach=5, p=0.1)
    d = OnDevice(case, device)
    d.forward(), d.backward()
    cf, tab = d.cf_adj.clone(), d.table_adj.clone()
    d.cf_adj.fill_(2.0), d.table_adj.fill_(2.0)
    d.backward(beta=0.5)
    torch.testing.assert_close(d.cf_adj, 1.0 + cf, rtol=0, atol=float(4 * U * (1 + cf.abs().max())))
    torch.testing.assert_close(d.table_adj, 1.0 + tab, rtol=0, atol=float(4 * U * (1 + tab.abs().max())))
    adj = d.adj.clone()
    A.attn_bwd_typed(d.qkv, d.off, d.dmerged, d.merged, d.ml, d.cf, 4, 32, kv_heads=2, bias=d.bias, dropout=d.drop, qkv_adj=d.adj)
    assert torch.equal(adj, d.adj)
    merged, none = A.attn_fwd_typed(d.qkv, d.off, d.cf, 4, 32, kv_heads=2, bias=d.bias, dropout=d.drop, save=False)
    assert none is None and torch.equal(merged, d.merged)


def test_no_atoms_and_no_rows(device):
    off, cf = torch.zeros(1, dtype=torch.int32, device=device), torch.zeros((0, 3), device=device)
    table = torch.zeros((4, 2), device=device)
    for T in (0, 5):
        x = torch.ones((T, 96), dtype=BF16, device=device)
        bias = A.RelativeBias(table, A.relative_buckets(4, 2, device=device), torch.zeros(T, dtype=torch.int32, device=device))
        merged, ml = A.attn_fwd_typed(x, off, cf, 2, 16, dead=True, bias=bias)
        adj, _, tab = A.attn_bwd_typed(x, off, x[:, :32].contiguous(), merged, ml, cf, 2, 16, dead=True, bias=bias,
                                       bias_adj=torch.full((4, 2), 3.0, device=device))
        assert merged.shape == (T, 32) and (merged == 0).all() and (adj == 0).all() and (tab == 0).all()


def test_rows_behind_the_last_edge_are_left_alone_without_dead(device):
    case = Case([9, 20], 2, 2, 32, BF16, dead=4)
    d = OnDevice(case, device)
    A.attn_fwd_typed(d.qkv, d.off, d.cf, 2, 32, merged=d.merged, ml=d.ml)
    A.attn_bwd_typed(d.qkv, d.off, d.dmerged, d.merged, d.ml, d.cf, 2, 32, qkv_adj=d.adj)
    assert (d.merged[-4:] == 3).all() and (d.adj[-4:] == 3).all()


def test_counts_past_the_slots_or_the_rows_are_cut(device):
    """Offsets that promise more than S or T hold touch no other row (the library has no look at them)."""
    case = Case([9, 11, 5], 2, 2, 32, BF16, slots=12)
    case.cf = torch.ones((3, 12))
    d = OnDevice(case, device)
    d.off = torch.tensor([0, 9, 24, 4000], dtype=torch.int32, device=device)
    d.forward(), d.backward()
    d.off = torch.tensor([-4, 2 ** 30, 7, 7], dtype=torch.int32, device=device)
    d.forward(), d.backward()
    torch.cuda.synchronize()


def test_leading_dimensions_past_32_bits(device):
    """Element offsets past 2^31 in every matrix."""
    ld = (1 << 24) + 8
    case = Case([70, 71], 2, 2, 16, BF16, p=0.1)

    def wide(x):
        buf = torch.empty((case.T - 1) * ld + x.shape[1], dtype=x.dtype, device=device)
        v = buf.as_strided(x.shape, (ld, 1))
        v.copy_(x)
        return v
    assert (case.T - 1) * ld > 1 << 31
    d = OnDevice(case, device)
    d.qkv, d.dmerged, d.merged, d.adj = (wide(x.cpu()) for x in (d.qkv, d.dmerged, d.merged, d.adj))
    d.check()


@pytest.mark.parametrize("counts", [[40, 70, 3], [300, 140]])
def test_runs_repeat_bit_for_bit(device, counts):
    case = Case(counts, 4, 2, 32, BF16, buckets=16, reach=20, p=0.1)
    d = OnDevice(case, device)
    d.forward(), d.backward()
    first = [x.clone() for x in (d.merged, d.ml, d.adj, d.cf_adj, d.table_adj)]
    for _ in range(3):
        d.forward(), d.backward()
        for x, y in zip(first, (d.merged, d.ml, d.adj, d.cf_adj, d.table_adj)):
            assert torch.equal(x, y)


def test_captured_and_replayed_with_a_rising_step(device):
    """A graph of forward, dropout and backward, whose step the graph raises: each replay is the eager step's, bit for bit."""
    case = Case([40, 70, 3, 150], 4, 2, 32, BF16, buckets=16, reach=20, p=0.1, dead=3)
    eager, graphed = OnDevice(case, device), OnDevice(case, device)
    width = case.H * case.hd
    residual = torch.randn(case.T, width, device=device).to(BF16)
    nbytes = _lib.load().pet_attn_bwd_typed_workspace(1, A.shape(case.N, case.T, case.S, 4, 32), 2, 16)

    def step(d, out, scratch):
        d.drop.state[1:] += 1
        d.forward()
        L.dropout_rows(out, d.merged, A.Dropout(0.25, d.drop.state, 9), residual)
        L.dropout_rows(d.dmerged, residual, A.Dropout(0.25, d.drop.state, 9))
        d.backward(scratch=scratch)
        return out
    outs = [torch.empty_like(residual) for _ in range(2)]
    scratch = [torch.empty(nbytes, dtype=torch.uint8, device=device) for _ in range(2)]
    step(graphed, outs[1], scratch[1])
    graphed.drop.state.copy_(eager.drop.state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed, outs[1], scratch[1])
    seen = []
    for _ in range(4):
        graph.replay()
        step(eager, outs[0], scratch[0])
        torch.cuda.synchronize()
        for x, y in zip((eager.merged, eager.ml, eager.adj, eager.cf_adj, eager.table_adj, outs[0]),
                        (graphed.merged, graphed.ml, graphed.adj, graphed.cf_adj, graphed.table_adj, outs[1])):
            assert torch.equal(x, y)
        seen.append(outs[1].clone())
    assert not torch.equal(seen[0], seen[1])


def test_on_another_stream(device):
    case = Case([40, 70, 300], 4, 2, 32, F16, buckets=16, reach=20, p=0.1)
    d = OnDevice(case, device)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(device)
    with torch.cuda.stream(stream):
        d.check()
    stream.synchronize()


def test_two_streams_at_once(device):
    cases = [Case([40, 70, 300], 4, 2, 32, F16, seed=s, buckets=16, reach=20, p=0.1) for s in range(2)]
    ds = [OnDevice(c, device) for c in cases]
    for d in ds:
        d.forward(), d.backward()
    want = [[x.clone() for x in (d.merged, d.adj, d.cf_adj, d.table_adj)] for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in ds]
    for _ in range(5):
        for d, s in zip(ds, streams):
            with torch.cuda.stream(s):
                d.forward(), d.backward()
    torch.cuda.synchronize()
    for d, w in zip(ds, want):
        for x, y in zip((d.merged, d.adj, d.cf_adj, d.table_adj), w):
            assert torch.equal(x, y)


def test_gradients_against_differences(device):
    """The forward's own change along a direction, fp16 rows: the loss w.merged at +- a step of the cutoff factors and
    of the table, whose adjoints are in fp32. merged is off by up to its bound at each end, so the quotient is by their
    sum over the step; the loss' third derivative along the direction is at most 8 sum |w| |v| times the logits'
    change cubed."""
    case = Case([12, 30], 2, 2, 32, F16, buckets=8, reach=6, seed=5)
    d = OnDevice(case, device)
    d.forward(), d.backward()
    rng = np.random.default_rng(1)
    w = case.dmerged.double()
    for name, step in (("cf", 2.0 ** -3), ("table", 2.0 ** -3)):
        x = case.cf if name == "cf" else case.table
        keep = x.clone()
        delta = torch.from_numpy(rng.choice([-1.0, 1.0], x.shape)).float() * step
        if name == "cf":
            delta = delta * keep * (keep < 1)
        ends, slack = [], 0.0
        for sign in (1, -1):
            x.copy_(keep + sign * delta)
            e = OnDevice(case, device)
            e.forward()
            ends.append(float((w * e.merged.double().cpu()).sum()))
            slack += float((w.abs() * case.forward()[1]).sum())
        x.copy_(keep)
        got = d.cf_adj if name == "cf" else d.table_adj
        along = float((got.double().cpu() * delta.double()).sum())
        vmax = case.qkv.double()[:, 128:].abs().max()
        third = 8 * float(w.abs().sum()) * float(vmax) * (step if name == "table" else step / (1 - step)) ** 3
        assert abs((ends[0] - ends[1]) / 2 - along) <= slack / 2 + third, name


# ---- dropout of rows ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 3), (75, 128), (40, 333), (7, 4099), (2, 40000), (1, 270001), (3000, 8)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_rows(device, dtype, rows, width, residual):
    gen = torch.Generator().manual_seed(rows)
    x, r = (torch.randn(rows, width, generator=gen).to(dtype) for _ in range(2))
    pad = width % 3
    state = (1234567 << 30 | 99, (1 << 35) + 17)

    def put(t):
        buf = torch.empty(rows, width + pad, dtype=dtype, device=device)[:, :width]
        buf.copy_(t)
        return buf
    xd, rd, out = put(x), put(r) if residual else None, put(torch.zeros_like(x))
    drop = A.Dropout(0.3, torch.tensor(state, dtype=torch.int64, device=device), 2 ** 32 - 1)
    L.dropout_rows(out, xd, drop, rd)
    mask = rows_mask(*state, 2 ** 32 - 1, 0.3, rows, width)
    ref = x.double() * mask + (r.double() if residual else 0.0)
    # the scale is rounded, the product or the sum rounded once in fp32, and to the type
    tol = 3 * U * (x.double().abs() * mask + ref.abs()) + (0.0 if dtype == F32 else half(dtype) * ref.abs() * (1 + 4 * U)
                                                            + torch.finfo(dtype).smallest_normal * half(dtype))
    within(out, ref, tol, "out")
    if not residual:
        assert torch.equal(out.cpu() == 0, (mask == 0) | (x == 0))
    # in place, onto either
    y = put(x)
    L.dropout_rows(y, y, drop, rd)
    assert torch.equal(y, out)
    if residual:
        L.dropout_rows(rd, xd, drop, rd)
        assert torch.equal(rd, out)


def test_dropout_of_nan_and_infinity(device):
    state = torch.tensor([5, 6], dtype=torch.int64, device=device)
    x = torch.full((64, 64), math.nan, device=device, dtype=F16)
    out = torch.empty_like(x)
    L.dropout_rows(out, x, A.Dropout(0.5, state))
    mask = rows_mask(5, 6, 0, 0.5, 64, 64)
    assert torch.equal(torch.isnan(out).cpu(), mask != 0) and (out.cpu()[mask == 0] == 0).all()


@pytest.mark.parametrize("live", [-3, 0, 1, 17, 40, 1000])
def test_dropout_rows_live(device, live):
    state = torch.tensor([5, 6], dtype=torch.int64, device=device)
    x = torch.randn(40, 50, device=device)
    x[max(0, live):] = math.nan
    out = torch.full_like(x, 7.0)
    L.dropout_rows(out, x, A.Dropout(0.25, state, 3), live=torch.tensor([live], dtype=torch.int32, device=device))
    n = min(max(live, 0), 40)
    assert (out[n:] == 7).all() and torch.isfinite(out).all()
    full = torch.empty_like(x[:n])
    if n:
        L.dropout_rows(full, x[:n], A.Dropout(0.25, state, 3))
        assert torch.equal(full, out[:n])


def test_dropout_p(device):
    """The ends of p, its steps of 2^-16, and how many stay (within 6 standard deviations)."""
    state = torch.tensor([11, 0], dtype=torch.int64, device=device)
    x = torch.ones(1024, 1024, device=device)
    for p in (0.0, 2.0 ** -18, 0.1, 0.5, 0.9, 65534 / 65536):
        out = torch.empty_like(x)
        L.dropout_rows(out, x, A.Dropout(p, state))
        q = round(p * 65536) / 65536
        kept = int((out != 0).sum())
        assert abs(kept - (1 - q) * 2 ** 20) <= 6 * math.sqrt(2 ** 20 * q * (1 - q)) + 1e-9
        assert torch.unique(out[out != 0]).tolist() == [float(np.float32(1 / (1 - q)))]


def test_masks_differ_by_seed_step_and_call(device):
    x = torch.ones(64, 64, device=device)
    seen = []
    for seed, step, call in ((1, 1, 0), (2, 1, 0), (1, 2, 0), (1, 1, 1), (1 + (1 << 40), 1, 0)):
        out = torch.empty_like(x)
        L.dropout_rows(out, x, A.Dropout(0.5, torch.tensor([seed, step], dtype=torch.int64, device=device), call))
        agree = [float(((out == 0) == (o == 0)).float().mean()) for o in seen]
        assert all(abs(a - 0.5) < 6 * 0.5 / 64 for a in agree)
        seen.append(out)


def test_dropout_rows_past_32_bits(device):
    ld = (1 << 30) + 16
    buf = torch.empty(2 * ld + 64, dtype=BF16, device=device)
    x = buf.as_strided((3, 64), (ld, 1))
    x.copy_(torch.randn(3, 64))
    state = torch.tensor([5, 6], dtype=torch.int64, device=device)
    want = torch.empty(3, 64, dtype=BF16, device=device)
    L.dropout_rows(want, x.contiguous(), A.Dropout(0.25, state, 3))
    L.dropout_rows(x, x, A.Dropout(0.25, state, 3))
    assert torch.equal(x, want)
