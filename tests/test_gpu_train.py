"""A training step's operators on the GPU, each against its formula in 64 bits:
the typed norms and their backward with the parameters' gradients, a dense
layer's gradients, the gradients' norm and clipping, and an attention layer's
backward with all of them.

Tolerances. U = 2^-24 is half an fp32 step, `half(t)` half a step of the output
type t (U for float32, whose one rounding the counts below hold already, as they
hold a few for each sum). A sum of n terms in fp32, however it is cut, is within n U of
the sum of their magnitudes. The counts of roundings:

- norms: a lane adds up to 32 values of a row (64 at float32 past 4096
  columns), a butterfly and the waves' sums at most 6 + 8 more, then a division, a
  square root and three products: ROW = 96 roundings cover a row's mean and its
  1/sd, the latter to half of them relative. xhat is then within ROW U of X =
  |xhat| + max|x| / sd (the mean's error times 1/sd is part of it).
- parameters' gradients: a lane sums at most rows / groups + 1 terms, 16 groups
  meet in LDS, the rest is in double: (rows + 17 + ROW) U of sum |g| X.
- linear_grads: see `linear_bound`.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from pet_kokkos_amd import attention as A
from pet_kokkos_amd import grads as G
from pet_kokkos_amd import layer as L
from pet_kokkos_amd import linear as D
from pet_kokkos_amd import systems

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROW = 96
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def least(t):
    """Half the smallest step of the type: what a subnormal result is off by."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, ref, tol, what):
    got, ref, tol = got.double().cpu(), ref.cpu(), tol.cpu()
    assert torch.isfinite(got).all(), what
    excess = (got - ref).abs() - tol
    i = int(excess.argmax())
    assert excess.flatten()[i] <= 0, f"{what}: {got.flatten()[i]} against {ref.flatten()[i]}, allowed {tol.flatten()[i]}"


def rows_of(gen, rows, width, dtype, device, pad=0, off=0, size=1.0):
    """[rows, width] with columns of differing size in a buffer `pad` wider, `off` elements past its start."""
    buf = torch.full((rows * (width + pad) + off + 8,), math.nan, dtype=dtype, device=device)
    x = buf[off:off + rows * (width + pad)].view(rows, width + pad)[:, :width]
    col = torch.exp(0.5 * torch.randn(width, generator=gen))
    x.copy_((size * torch.randn((rows, width), generator=gen) * col + 0.1 * size).to(dtype))
    return x


def norm_ref(x, g, w, b, ln):
    """The norm of x (and its gradients for g) in 64 bits, and the magnitudes its error goes by."""
    x, w = x.double().cpu(), w.double().cpu()
    n = x.shape[1]
    mu = x.mean(1, keepdim=True) if ln else torch.zeros(len(x), 1, dtype=torch.float64)
    inv = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + (1e-5 if ln else 2.0 ** -23))
    xhat = (x - mu) * inv
    big = xhat.abs() + x.abs().amax(1, keepdim=True) * inv
    out = xhat * w + (b.double().cpu() if ln else 0.0)
    r = {"out": out, "out_tol": ROW * U * (big * w.abs() + out.abs())}
    if g is None:
        return r
    g = g.double().cpu()
    gw = g * w
    mg, mgx = (gw.mean(1, keepdim=True) if ln else 0.0), (gw * xhat).mean(1, keepdim=True)
    r["in_adj"] = inv * (gw - mg - xhat * mgx)
    size = inv * (gw.abs() + (gw.abs().mean(1, keepdim=True) if ln else 0.0) + big * (gw.abs() * big).mean(1, keepdim=True))
    r["in_tol"] = 3 * ROW * U * size  # three factors, each within ROW roundings
    r["w_adj"], r["b_adj"] = (g * xhat).sum(0), g.sum(0)
    r["w_tol"], r["b_tol"] = (len(x) + 17 + ROW) * U * (g.abs() * big).sum(0), (len(x) + 17) * U * g.abs().sum(0)
    return r


WIDTHS = [1, 3, 16, 64, 65, 128, 200, 256, 257, 512, 777, 1024, 1500, 2048, 2049, 4096, 5000, 8192, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("ln", [False, True])
def test_norm_rows(device, dtype, width, ln):
    gen = torch.Generator().manual_seed(width)
    w = (1 + 0.1 * torch.randn(width, generator=gen)).to(device)
    b = (0.1 * torch.randn(width, generator=gen)).to(device) if ln else None
    for rows, pad, off in ((1, 0, 0), (19, 0, 0), (33, 5, 1)):
        x = rows_of(gen, rows, width, dtype, device, pad, off)
        out = rows_of(gen, rows, width, dtype, device, pad + 2, off)
        L.norm_rows(out, x, w, b)
        r = norm_ref(x, None, w, b, ln)
        within(out, r["out"], r["out_tol"] + half(dtype) * (r["out"].abs() + r["out_tol"]) + least(dtype), "out")
        assert torch.isnan(out.as_strided((rows - 1, 2), (width + pad + 2, 1), out.storage_offset() + width)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("ln", [False, True])
def test_norm_rows_grads(device, dtype, width, ln):
    gen = torch.Generator().manual_seed(width + 1)
    w = (1 + 0.1 * torch.randn(width, generator=gen)).to(device)
    for rows, pad, off, beta, beta_w in ((1, 0, 0, 0.0, 0.0), (70, 0, 0, 0.0, 1.0), (37, 3, 1, 0.5, -0.5)):
        x, g = (rows_of(gen, rows, width, dtype, device, pad, off, s) for s in (1.0, 1e-2))
        adj = rows_of(gen, rows, width, dtype, device, pad + 1, off, 1e-2)
        before = adj.double().cpu()
        wa, ba = (torch.randn(width, generator=gen).to(device) for _ in range(2))
        wa0, ba0 = wa.double().cpu(), ba.double().cpu()
        L.norm_rows_grads(adj, wa, ba if ln else None, g, x, w, ln, beta, beta_w)
        r = norm_ref(x, g, w, None if not ln else w, ln)
        ref = r["in_adj"] + beta * before
        tol = r["in_tol"] + 2 * U * (beta * before).abs()
        within(adj, ref, tol + half(dtype) * (ref.abs() + tol) + least(dtype), "in_adj")
        within(wa, r["w_adj"] + beta_w * wa0, r["w_tol"] + 2 * U * (r["w_adj"].abs() + (beta_w * wa0).abs()), "w_adj")
        if ln:
            within(ba, r["b_adj"] + beta_w * ba0, r["b_tol"] + 2 * U * (r["b_adj"].abs() + (beta_w * ba0).abs()), "b_adj")
        else:
            assert torch.equal(ba.double().cpu(), ba0)


def test_norm_rows_grads_parts(device):
    """Each output on its own is the bits it is beside the others; in_adj in place of
    out_adj and of the input; the same bits twice; many rows."""
    gen = torch.Generator().manual_seed(5)
    for dtype, rows, width, ln in ((torch.float32, 9001, 128, True), (torch.bfloat16, 5003, 512, False),
                                   (torch.float16, 300, 9000, True), (torch.bfloat16, 700, 8000, True),
                                   (torch.float32, 2000, 3001, False), (torch.float32, 600, 16384, True)):
        x, g = rows_of(gen, rows, width, dtype, device), rows_of(gen, rows, width, dtype, device, size=1e-2)
        w = (1 + 0.1 * torch.randn(width, generator=gen)).to(device)

        def run(a, wa, ba, g=g, x=x):
            L.norm_rows_grads(a, wa, ba, g, x, w, ln)
            return a, wa, ba
        new = lambda n=None: torch.full((rows, width) if n is None else (n,), 7.0, dtype=dtype if n is None else torch.float32, device=device)
        a, wa, ba = run(new(), new(width), new(width) if ln else None)
        a2, wa2, _ = run(new(), new(width), new(width) if ln else None)
        assert torch.equal(a, a2) and torch.equal(wa, wa2)
        assert torch.equal(run(new(), None, None)[0], a)
        assert torch.equal(run(None, new(width), None)[1], wa)
        if ln:
            assert torch.equal(run(None, None, new(width))[2], ba)
        gc, xc = g.clone(), x.clone()
        assert torch.equal(run(gc, None, None, g=gc)[0], a)
        assert torch.equal(run(xc, new(width), None, x=xc)[0], a)
        r = norm_ref(x, g, w, w, ln)
        within(wa, r["w_adj"], r["w_tol"] + U * r["w_adj"].abs(), "w_adj")


def test_norm_rows_grads_against_differences(device):
    """The gradients are the derivatives of the forward: central differences of
    sum(out * g) in 64 bits."""
    gen = torch.Generator().manual_seed(6)
    for ln in (False, True):
        x, g = rows_of(gen, 5, 24, torch.float32, device), rows_of(gen, 5, 24, torch.float32, device)
        w = (1 + 0.1 * torch.randn(24, generator=gen)).to(device)
        b = torch.zeros(24, device=device)
        adj, wa, ba = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        L.norm_rows_grads(adj, wa, ba if ln else None, g, x, w, ln)

        def loss(x, w, b):
            return float((norm_ref(x, None, w, b, ln)["out"] * g.double().cpu()).sum())
        h = 1e-4  # the difference's own error: h^2 / 6 of a third derivative of order 10
        for t, adj_t, at in ((0, adj, (2, 7)), (0, adj, (4, 23)), (1, wa, (3,)), (2, ba if ln else None, (11,))):
            if adj_t is None:
                continue
            args = [x.double().cpu(), w.double().cpu(), b.double().cpu()]
            up, down = [a.clone() for a in args], [a.clone() for a in args]
            up[t][at] += h
            down[t][at] -= h
            assert abs((loss(*up) - loss(*down)) / (2 * h) - float(adj_t[at])) < 1e-5 * (1 + abs(float(adj_t[at])))


@pytest.mark.parametrize("live", [0, 1, 50, 77, 1000, -3])
def test_norm_rows_grads_live(device, live):
    """Rows from *live on: poisoned, neither read nor written."""
    gen = torch.Generator().manual_seed(8)
    rows, width = 77, 96
    n = min(max(live, 0), rows)
    x, g = rows_of(gen, rows, width, torch.float32, device), rows_of(gen, rows, width, torch.float32, device)
    w = torch.ones(width, device=device)
    x[n:], g[n:] = math.nan, math.inf
    adj, wa, ba = torch.full_like(x, 3.0), torch.ones(width, device=device), torch.ones(width, device=device)
    L.norm_rows_grads(adj, wa, ba, g, x, w, True, live=torch.tensor([live], dtype=torch.int32, device=device))
    assert (adj[n:] == 3.0).all()
    ref_a, ref_w, ref_b = torch.empty_like(x[:n]), torch.empty_like(w), torch.empty_like(w)
    L.norm_rows_grads(ref_a, ref_w, ref_b, g[:n].contiguous(), x[:n].contiguous(), w, True)
    assert torch.equal(adj[:n], ref_a)
    tol = (n + 17 + ROW) * 2 * U * (g[:n].abs() * 20).sum(0).double()  # the rows' split among lanes differs; |xhat| < sqrt(96)
    within(wa, ref_w.double(), tol, "w_adj")
    within(ba, ref_b.double(), tol, "b_adj")


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(device, dtype):
    """No rows: nothing is written but the parameters' gradients, beta times what they were."""
    x, w = torch.zeros((0, 40), dtype=dtype, device=device), torch.ones(40, device=device)
    if dtype != torch.float32:
        L.norm_rows(x, x, w, None)
    L.norm_rows_grads(x, None, None, x, x, w, False)
    wa, ba = torch.full_like(w, 4.0), torch.full_like(w, math.nan)
    L.norm_rows_grads(x, wa, None, x, x, w, True, beta_w=0.5)
    L.norm_rows_grads(None, None, ba, x, x, w, True)
    assert (wa == 2).all() and (ba == 0).all()


def test_norm_rows_not_finite(device):
    """A NaN or an infinity spoils its own row's adjoint and no other, and the columns it reaches."""
    gen = torch.Generator().manual_seed(9)
    x, g = rows_of(gen, 20, 64, torch.bfloat16, device), rows_of(gen, 20, 64, torch.bfloat16, device)
    w = torch.ones(64, device=device)
    clean = torch.empty_like(x)
    L.norm_rows_grads(clean, None, None, g, x, w, True)
    g[3, 5] = math.nan
    x[7, 1] = math.inf
    adj, wa, ba = torch.empty_like(x), torch.empty(64, device=device), torch.empty(64, device=device)
    L.norm_rows_grads(adj, wa, ba, g, x, w, True)
    rest = [i for i in range(20) if i not in (3, 7)]
    assert torch.equal(adj[rest], clean[rest]) and torch.isnan(adj[[3, 7]]).all()
    assert torch.isnan(wa).all()  # row 7's xhat is NaN in every column
    assert torch.isnan(ba[5]) and torch.isfinite(ba[[i for i in range(64) if i != 5]]).all()


def test_norm_rows_squares_past_fp32(device):
    """Rows whose squares pass fp32 come out as zeros, as fp32 arithmetic makes them, and no NaN."""
    x = torch.full((3, 4096), 1e25, device=device)
    w, out = torch.ones(4096, device=device), torch.full((3, 4096), 7.0, device=device)
    L.norm_rows(out, x, w, None)
    assert (out == 0).all()
    small = torch.full((3, 64), 1e25, device=device, dtype=torch.bfloat16)
    L.norm_rows(small, small, w[:64], None)
    assert (small == 0).all()


def test_offsets_past_32_bits(device):
    """Rows whose offsets, and a tensor whose elements, pass 2^31: the last ones count."""
    M, ld = (1 << 21) + 70000, 1024  # 2.2e9 elements
    base = torch.zeros((M, ld), dtype=torch.bfloat16, device=device)
    g, x = base[:, :4], base[:, 8:14]
    gen = torch.Generator().manual_seed(51)
    at = torch.tensor([0, 1, 1 << 20, (1 << 21) + 5, M - 2, M - 1])
    g[at] = torch.randn((6, 4), generator=gen).to(device).bfloat16()
    x[at] = torch.randn((6, 6), generator=gen).to(device).bfloat16()
    wa, ba = torch.empty((4, 6), device=device), torch.empty(4, device=device)
    D.linear_grads(g, x, wa, ba)
    gd, xd = g[at].double().cpu(), x[at].double().cpu()
    within(wa, gd.t() @ xd, 16 * U * (gd.abs().t() @ xd.abs()), "w_adj")
    within(ba, gd.sum(0), 16 * U * gd.abs().sum(0), "b_adj")
    w, wn, bn = torch.ones(4, device=device), torch.empty(4, device=device), torch.empty(4, device=device)
    adj = base[:, 20:24]
    L.norm_rows_grads(adj, wn, bn, g, base[:, 8:12], w, True)
    r = norm_ref(base[at, 8:12], g[at], w, w, True)  # (the other rows are zeros, and so are their adjoints)
    tol = r["in_tol"] + half(torch.bfloat16) * (r["in_adj"].abs() + r["in_tol"]) + least(torch.bfloat16)
    within(adj[at], r["in_adj"], tol, "in_adj")
    within(wn, r["w_adj"], 8 * r["w_tol"], "w_adj")  # (8 rows' lanes and parts, with zeros between)
    within(bn, r["b_adj"], 8 * r["b_tol"], "b_adj")
    out = base[:, 30:34]
    L.norm_rows(out, base[:, 8:12], w, w)
    ref = norm_ref(base[at, 8:12], None, w, w, True)
    within(out[at], ref["out"], ref["out_tol"] + half(torch.bfloat16) * (ref["out"].abs() + ref["out_tol"]), "out")
    base.zero_()
    flat = base.view(-1)[5:]
    flat[-1], flat[0] = 3.0, 4.0
    assert float(G.clip_grads([flat], 1.0, eps=0.0)) == 5.0
    assert flat[-1].item() == torch.tensor(0.6).bfloat16().item() and flat[0].item() == torch.tensor(0.8).bfloat16().item()


# ---- linear_grads -------------------------------------------------------------------


def linear_bound(g, x, dtype):
    """How far w_adj may be from sum g x, from the roundings of the sum: rows in
    steps of 32 (or one by one) over pieces, (M / 32 + 300) of them at most a sum
    of the kernel's step by step ones, each U of what is summed; a step's own 32
    products 8 more. For fp32 rows each product is of two values held to 2^-23
    and without the product of their low parts (2^-22): 8 U of its magnitude, and a value
    more than 2^-14 below its column's largest is held to 2^-35 of that."""
    g, x = g.double().cpu(), x.double().cpu()
    M = len(g)
    tol = (M / 32 + 308) * U * (g.abs().t() @ x.abs())
    if dtype == torch.float32 and M:
        ga, xa = g.abs(), x.abs()
        tol += 8 * U * (ga.t() @ xa)
        tol += 2.0 ** -35 * (ga.amax(0)[:, None] * xa.sum(0)[None] + ga.sum(0)[:, None] * xa.amax(0)[None])
    return tol


LINEAR = [(0, 8, 8), (1, 1, 1), (1, 64, 64), (3, 5, 7), (31, 33, 130), (32, 128, 128), (33, 16, 256), (64, 257, 31),
          (129, 200, 300), (500, 96, 64), (648, 1024, 256), (1000, 1, 513), (2049, 130, 4), (5003, 77, 129),
          (20000, 256, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", LINEAR)
def test_linear_grads(device, dtype, size):
    M, N, K = size
    gen = torch.Generator().manual_seed(M)
    for pad, off, beta in ((0, 0, 0.0), (3, 1, 0.5)):
        g, x = rows_of(gen, M, N, dtype, device, pad, off, 1e-2), rows_of(gen, M, K, dtype, device, pad, off)
        wa = torch.randn((N, K + pad), generator=gen).to(device)[:, :K]
        ba = torch.randn(N, generator=gen).to(device)
        wa0, ba0 = wa.double().cpu(), ba.double().cpu()
        edge = wa.as_strided((N, pad), (K + pad, 1), K).clone() if pad else None
        D.linear_grads(g, x, wa, ba, beta)
        ref, bref = g.double().cpu().t() @ x.double().cpu(), g.double().cpu().sum(0)
        tol = linear_bound(g, x, dtype)
        within(wa, ref + beta * wa0, tol + 2 * U * (ref.abs() + (beta * wa0).abs()), "w_adj")
        btol = (M / 32 + 308 + 32) * U * g.double().cpu().abs().sum(0) + 2 * U * (bref.abs() + (beta * ba0).abs())
        within(ba, bref + beta * ba0, btol, "b_adj")
        if pad:
            assert torch.equal(wa.as_strided((N, pad), (K + pad, 1), K), edge)
        again, bagain = wa0.float().to(device), ba0.float().to(device)
        D.linear_grads(g, x, again, bagain, beta)
        assert torch.equal(again, wa) and torch.equal(bagain, ba)  # bit for bit
        D.linear_grads(g, x, again, None)
        one = torch.empty_like(again)
        D.linear_grads(g, x, one, bagain)
        assert torch.equal(again, one)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("live", [0, 1, 31, 333, 700, 9999, -1])
def test_linear_grads_live(device, dtype, live):
    gen = torch.Generator().manual_seed(12)
    M, N, K = 700, 72, 100
    n = min(max(live, 0), M)
    g, x = rows_of(gen, M, N, dtype, device), rows_of(gen, M, K, dtype, device)
    g[n:], x[n:] = math.nan, math.inf
    wa, ba = torch.full((N, K), math.nan, device=device), torch.full((N,), math.nan, device=device)
    D.linear_grads(g, x, wa, ba, live=torch.tensor([live], dtype=torch.int32, device=device))
    gd = g[:n].double().cpu()
    within(wa, gd.t() @ x[:n].double().cpu(), linear_bound(g[:n], x[:n], dtype) + least(torch.float32), "w_adj")
    within(ba, gd.sum(0), (M / 32 + 340) * U * gd.abs().sum(0) + least(torch.float32), "b_adj")


def test_linear_grads_scales(device):
    """fp32 rows whose columns, and whose rows, differ by many orders of magnitude:
    growing and shrinking along the sum, zeros first, the ends of the range."""
    gen = torch.Generator().manual_seed(13)
    M, N, K = 4100, 70, 66
    base_g, base_x = torch.randn((M, N), generator=gen), torch.randn((M, K), generator=gen)
    ramp = torch.linspace(-18, 18, M)[:, None]
    cols_n, cols_k = torch.linspace(-15, 15, N)[None], torch.linspace(15, -15, K)[None]
    late = (torch.arange(M) >= 3000).float()[:, None]
    cases = {"columns": (base_g * 10 ** cols_n, base_x * 10 ** cols_k), "grow": (base_g * 10 ** ramp, base_x),
             "shrink": (base_g, base_x * 10 ** -ramp), "late": (base_g * late, base_x * late * 1e20),
             "huge": (base_g * 1e30, base_x * 1e-30), "tiny": (base_g * 1e-25, base_x * 1e-12),
             "zero": (base_g * 0, base_x)}
    for name, (g, x) in cases.items():
        g, x = g.to(device), x.to(device)
        wa, ba = torch.empty((N, K), device=device), torch.empty(N, device=device)
        D.linear_grads(g, x, wa, ba)
        gd = g.double().cpu()
        within(wa, gd.t() @ x.double().cpu(), linear_bound(g, x, torch.float32) + 400 * least(torch.float32), name)
        within(ba, gd.sum(0), (M / 32 + 340) * U * gd.abs().sum(0) + least(torch.float32), name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 3000])
def test_linear_grads_not_finite(device, dtype, rows):
    """Infinities and NaN reach the elements that the formula takes them to, as
    fp32 products and sums do, and no others."""
    gen = torch.Generator().manual_seed(14)
    g, x = rows_of(gen, rows, 150, dtype, device), rows_of(gen, rows, 140, dtype, device)
    g[7, 3], g[rows - 2, 80], x[9, 11], x[20, 139] = math.inf, math.nan, -math.inf, math.nan
    x[7, 100] = 0.0  # inf * 0
    wa, ba = torch.empty((150, 140), device=device), torch.empty(150, device=device)
    D.linear_grads(g, x, wa, ba)
    gd, xd = g.double().cpu(), x.double().cpu()
    ref = (gd[:, :, None] * xd[:, None, :]).sum(0) if rows < 100 else gd.t() @ xd
    got = wa.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], ref[inf])
    ok = torch.isfinite(ref)
    tol = linear_bound(g.nan_to_num(0, 0, 0), x.nan_to_num(0, 0, 0), dtype)
    assert ((got - ref).abs()[ok] <= tol[ok]).all()
    assert torch.isinf(ba[3]) and torch.isnan(ba[80]) and torch.isfinite(ba).sum() == 148


# ---- the gradients' norm and clipping -----------------------------------------------


def gradient_set(device, kind, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, t=torch.float32: (torch.randn(s, generator=gen)).to(device=device, dtype=t)
    if kind == "one":
        return [r(1)]
    if kind == "model":
        return [r(*s) for _ in range(30) for s in ((96, 64), (96,), (64, 96), (64,), (64,))]  # more than one launch holds
    if kind == "mixed":
        flat = r(5001, t=torch.bfloat16)
        wide = r(33, 50)
        return [r(3, 7, t=torch.float16), flat[1:4098], flat[4099:], r(40, 30).t(), wide[:, :20], wide[:, 21:50],
                r(0), r(257, 3, t=torch.float16)[1:], r(5, 8)[:, 3], r(2, 3, 4).permute(2, 0, 1), r(70001, t=torch.bfloat16)]
    return [r(4095), r(4096), r(4097), r(3000000, t=torch.bfloat16), r(1234567), r(1000003, t=torch.float16)]


def norm_of(tensors, p, scale=1.0):
    flat = torch.cat([t.double().flatten().cpu() for t in tensors])
    return abs(scale) * float(flat.abs().max() if p == math.inf else (flat.abs() ** p).sum() ** (1 / p))


@pytest.mark.parametrize("kind", ["one", "model", "mixed", "large"])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_grad_norm_and_clip(device, kind, p):
    """The norm is a double's, rounded once; a clipped gradient is off by its
    factor's rounding, its product's and its type's."""
    for scale, part in ((1.0, 0.5), (1.0, 2.0), (-0.37, 0.1), (0.25, 3.0)):
        t = gradient_set(device, kind)
        before = [x.double().cpu() for x in t]
        ref = norm_of(t, p, scale)
        got = G.grad_norm(t, p, scale)
        assert got.dim() == 0 and got.dtype == torch.float32
        assert abs(float(got) - ref) <= 1.01 * U * ref
        bound = part * ref
        out = G.clip_grads(t, bound, p, scale)
        assert torch.equal(out, got)
        factor = scale * min(1.0, bound / (ref + 1e-6))
        for x, b in zip(t, before):
            want = factor * b
            if x.numel():
                within(x, want, (2.01 * U + half(x.dtype)) * want.abs() + least(x.dtype), "clipped")
            if factor == 1.0:
                assert torch.equal(x.double().cpu(), b)


def test_clip_leaves_the_rest(device):
    """Columns beside a view, and elements around a slice, stay as they were."""
    base, flat = torch.ones(40, 64, device=device), torch.ones(9000, dtype=torch.float16, device=device)
    G.clip_grads([base[:, 3:50], flat[7:8190]], 0.0)
    want = torch.ones(40, 64)
    want[:, 3:50] = 0
    assert torch.equal(base.cpu(), want)
    assert flat.sum().item() == 9000 - 8183 and (flat[7:8190] == 0).all()


def test_clip_range(device):
    """Gradients whose squares leave fp32's range, nothing at all, zeros, a NaN, an infinity."""
    for size in (1e30, 1e-30):
        t = [torch.full((5000,), size, device=device), torch.full((3,), -size, device=device)]
        ref = norm_of(t, 2.0)
        assert abs(float(G.clip_grads(t, size, eps=0.0)) - ref) <= 1.01 * U * ref
        within(t[0], torch.full((5000,), float(torch.tensor(size)) * size / ref, dtype=torch.float64), torch.full((5000,), 3 * U * size / 70), "clipped")
    assert float(G.grad_norm([])) == 0.0 == float(G.clip_grads([], 1.0))
    empty = torch.zeros(0, device=device)
    assert float(G.clip_grads([empty], 1.0)) == 0.0
    zero = torch.zeros(10, device=device)
    assert float(G.clip_grads([zero], 0.0, eps=0.0)) == 0.0 and (zero == 0).all()
    for p in (1.0, 2.0, math.inf):
        t = [torch.ones(5000, device=device), torch.ones(7, device=device)]
        t[0][4321] = math.nan
        assert math.isnan(float(G.clip_grads(t, 1.0, p))) and torch.isnan(t[1]).all()
        t = [torch.ones(5000, device=device), torch.ones(7, device=device)]
        t[0][4321] = -math.inf
        assert float(G.clip_grads(t, 1.0, p)) == math.inf
        assert (t[1] == 0).all() and torch.isnan(t[0][4321]) and (t[0][:4321] == 0).all()
    t = [torch.full((9,), 2.0, device=device)]
    assert float(G.clip_grads(t, math.inf)) == 6.0 and (t[0] == 2).all()


def test_gradient_lists_refuse(device):
    a = torch.zeros(100, device=device)
    for bad in ([a, a], [a[:60], a[59:]], [a.view(10, 10)[:, :6], a.view(10, 10)[:, 5:]], [a.view(10, 10)[::2, ::2]],
                [a.double()], [a, a.cpu()],
                # a third view beside the second and over the first
                [a.view(10, 10)[:, :5], a.view(10, 10)[:, 5:], a.view(10, 10)[5:, :2]]):
        with pytest.raises(ValueError):
            G.clip_grads(bad, 1.0)
    G.clip_grads([a.view(10, 10)[:, :6], a.view(10, 10)[:, 6:]], 1.0)
    b = torch.ones(50, device=device)
    lst = G.GradList([b])
    b.data = torch.zeros(50, device=device)  # the list keeps the memory it was made of
    assert abs(float(G.grad_norm(lst)) - math.sqrt(50)) < 1e-6
    for kw in (dict(norm_type=3.0), dict(scale=math.nan), dict(eps=-1.0), dict(out=torch.zeros(2, device=device))):
        with pytest.raises(ValueError):
            G.clip_grads([a], 1.0, **kw)
    with pytest.raises(ValueError):
        G.clip_grads([a], math.nan)


def test_refusals_on_the_device(device):
    x, w = torch.zeros(4, 8, device=device), torch.zeros(8, device=device)
    live = torch.zeros(1, dtype=torch.int64, device=device)
    bad = [lambda: L.norm_rows_grads(x[:3], w, None, x, x, w, False), lambda: L.norm_rows_grads(x, w[:7], None, x, x, w, False),
           lambda: L.norm_rows_grads(x, w, w, x, x, w, False), lambda: L.norm_rows_grads(None, None, None, x, x, w, False),
           lambda: L.norm_rows_grads(x.half(), w, None, x, x, w, False), lambda: L.norm_rows_grads(x, w, None, x.t(), x.t(), w, False),
           lambda: L.norm_rows_grads(x, w, None, x, x, w, False, live=live), lambda: L.norm_rows(x.half(), x.half(), w.half(), None),
           lambda: L.norm_rows(x.double(), x.double(), w, None), lambda: L.norm_rows_grads(x, w.cpu(), None, x, x, w, False),
           lambda: L.norm_rows_grads(x, w, None, x[:1].expand(4, 8), x, w, False),
           lambda: D.linear_grads(x, x[:3], torch.zeros(8, 8, device=device)), lambda: D.linear_grads(x, x, torch.zeros(8, 7, device=device)),
           lambda: D.linear_grads(x, x.half(), torch.zeros(8, 8, device=device)), lambda: D.linear_grads(x, x, torch.zeros(8, 8, device=device).half()),
           lambda: D.linear_grads(x, x, torch.zeros(8, 8, device=device).t()[:, ::2]), lambda: D.linear_grads(x, x, torch.zeros(8, 8, device=device), w[:3]),
           lambda: D.linear_grads(x, x, torch.zeros(8, 8, device=device), live=live)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: D.linear_grads(x, x, torch.zeros(8, 8, device=device), scratch=torch.zeros(1, device=device)),
              lambda: L.norm_rows_grads(x, w, None, x, x, w, False, scratch=torch.zeros(1, device=device)),
              lambda: G.grad_norm([x], scratch=torch.zeros(1, device=device))):
        with pytest.raises(RuntimeError):
            f()


# ---- together -----------------------------------------------------------------------


def attention_f64(tokens, nw, nb, w_in, b_in, w_out, b_out, tk, cf, H, hd, temp):
    """The attention block in float64 on torch's CPU, differentiable."""
    N = tk.n_atoms
    if nb is None:
        xhat = tokens / torch.sqrt((tokens ** 2).mean(1, keepdim=True) + 2.0 ** -23)
        normed = xhat * nw
    else:
        c = tokens - tokens.mean(1, keepdim=True)
        normed = c / torch.sqrt((c ** 2).mean(1, keepdim=True) + 1e-5) * nw + nb
    q, k, v = (normed @ w_in.t() + b_in).split(H * hd, 1)
    merged = torch.zeros_like(tokens)
    for n in range(N):
        rows = [n] + list(range(N + int(tk.off[n]), N + int(tk.off[n + 1])))
        c = cf[n, :len(rows)]
        heads = lambda t: t[rows].view(len(rows), H, hd).transpose(0, 1)
        s = heads(q) @ heads(k).transpose(1, 2) / (math.sqrt(hd) * temp) + torch.log(c.clamp_min(1e-300))
        s = s.masked_fill((c <= 0)[None, None], -math.inf)
        o = torch.softmax(s, -1) @ heads(v)
        o = torch.where((c > 0)[None, :, None], o, 0.0)
        merged[rows] = o.transpose(0, 1).reshape(len(rows), H * hd)
    return merged @ w_out.t() + b_out


def layer_case(device, ln, dead, seed=21):
    rng = np.random.default_rng(seed)
    H, hd = 2, 32
    Dm = H * hd
    tk = systems.tokens_from_counts([5, 1, 20, 9, 33], seed=seed)
    T = tk.n_rows + (6 if dead else 0)
    a = {"tokens": rng.standard_normal((T, Dm)), "nw": 1 + 0.1 * rng.standard_normal(Dm), "nb": 0.1 * rng.standard_normal(Dm),
         "w_in": rng.standard_normal((3 * Dm, Dm)) / 8, "b_in": 0.1 * rng.standard_normal(3 * Dm),
         "w_out": rng.standard_normal((Dm, Dm)) / 8, "b_out": 0.1 * rng.standard_normal(Dm), "g": rng.standard_normal((T, Dm))}
    a = {k: torch.from_numpy(v.astype(np.float32)).to(device) for k, v in a.items()}
    if dead:
        a["g"][tk.n_rows:] = math.nan if dead == "nan" else 1e6  # a capacity's rows count for nothing
    if not ln:
        a["nb"] = None
    return a, tk, T, H, hd


NAMES = {"norm_w": "nw", "norm_b": "nb", "w_in": "w_in", "b_in": "b_in", "w_out": "w_out", "b_out": "b_out"}


@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("dead", [False, True])
def test_attention_layer_grads(device, ln, dead):
    """Every parameter's gradient of an attention block against float64 autograd:
    the parity bar of the library's attention (1e-5 of a tensor's largest value, sums
    over 73 rows of terms of either sign), tokens_adj the plain backward's."""
    a, tk, T, H, hd = layer_case(device, ln, dead)
    Dm, S, temp = H * hd, tk.slots, 1.1
    off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
    t, ws = A.Tokens(off, tk.n_atoms, bool(dead)), A.Workspace(device)
    out = torch.empty((T, Dm), device=device)
    L.attention_layer(ws, "l", out, a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"], a["b_out"], t, S, H, hd, temp)
    grads = {n: torch.full_like(a[k], 2.0) for n, k in NAMES.items() if a[k] is not None}
    results = []
    for with_grads in (True, False):
        tadj, csa = torch.full((T, Dm), 0.5, device=device), torch.zeros((tk.n_atoms, S), device=device)
        args = (tadj, csa, a["g"], a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"], t, S, H, hd, temp)
        if with_grads:
            L.attention_layer_grads(ws, "l", grads, *args, beta=0.5)
        else:
            L.attention_layer_bwd(ws, "l", *args)
        results.append((tadj, csa))
    for x, y in zip(*results):
        assert float((x - y).abs().max()) <= 1e-5 * float(y.abs().max())
    leaves = {n: a[k].double().cpu().requires_grad_() for n, k in NAMES.items() if a[k] is not None}
    live = tk.n_rows
    ref = attention_f64(a["tokens"][:live].double().cpu(), leaves["norm_w"], leaves.get("norm_b"), leaves["w_in"], leaves["b_in"],
                        leaves["w_out"], leaves["b_out"], tk, torch.from_numpy(tk.cf_seq).double(), H, hd, temp)
    (ref * a["g"][:live].double().cpu()).sum().backward()
    for n, g in grads.items():
        want = leaves[n].grad + 0.5 * 2.0
        assert float((g.double().cpu() - want).abs().max()) <= 1e-5 * float(leaves[n].grad.abs().max()) + 2 * U, n
    some = {"w_out": torch.empty_like(a["w_out"])}  # a part of them
    L.attention_layer_grads(ws, "l", some, tadj, csa, a["g"], a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf,
                            a["w_out"], t, S, H, hd, temp)
    assert float((some["w_out"] - (grads["w_out"] - 1.0)).abs().max()) <= 1e-5 * float(some["w_out"].abs().max()) + 4 * U
    with pytest.raises(ValueError):
        L.attention_layer_grads(ws, "l", {"w": some["w_out"]}, *args)
    with pytest.raises(ValueError):
        L.attention_layer_grads(ws, "l", {"b_out": a["b_out"]}, *args)
    for i, bad in ((2, a["g"][:-1]), (3, a["tokens"][:, 1:]), (6, a["w_out"]), (8, cf[:, 1:]), (0, tadj.half())):
        with pytest.raises(ValueError):
            L.attention_layer_grads(ws, "l", some, *args[:i], bad, *args[i + 1:])


@pytest.mark.parametrize("ln", [False, True])
def test_training_step_captured(device, ln):
    """A whole step of one attention block (forward, backward with every gradient,
    clipping, the update) recorded as a HIP graph on a stream of its own and replayed
    between eager work, bit for bit the eager step; the block's output moves
    toward its target by what the gradients say."""
    a, tk, T, H, hd = layer_case(device, ln, False)
    Dm, S = H * hd, tk.slots
    off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
    t = A.Tokens(off, tk.n_atoms, False)
    target = a["g"].clone()

    def fresh():
        p = {n: a[k].clone() for n, k in NAMES.items() if a[k] is not None}
        return p, {n: torch.zeros_like(v) for n, v in p.items()}, A.Workspace(device)

    def step(p, grads, lst, ws, buf):
        L.attention_layer(ws, "l", buf["out"], a["tokens"], p["norm_w"], p.get("norm_b"), p["w_in"], p["b_in"], cf, p["w_out"],
                          p["b_out"], t, S, H, hd, 1.0)
        torch.sub(buf["out"], target, out=buf["g"])
        buf["csa"].zero_()
        buf["tadj"].zero_()
        L.attention_layer_grads(ws, "l", grads, buf["tadj"], buf["csa"], buf["g"], a["tokens"], p["norm_w"], p.get("norm_b"),
                                p["w_in"], p["b_in"], cf, p["w_out"], t, S, H, hd, 1.0)
        G.clip_grads(lst, 1.0, out=buf["norm"])
        for n in p:
            p[n].add_(grads[n], alpha=-0.01)

    def buffers():
        return {"out": torch.empty((T, Dm), device=device), "g": torch.empty((T, Dm), device=device),
                "tadj": torch.empty((T, Dm), device=device), "csa": torch.empty((tk.n_atoms, S), device=device),
                "norm": torch.empty((), device=device)}
    runs = []
    for captured in (False, True):
        p, grads, ws = fresh()
        lst, buf, norms = G.GradList(grads.values()), buffers(), []
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            keep = {n: v.clone() for n, v in p.items()}
            with torch.cuda.stream(side):
                step(p, grads, lst, ws, buf)  # warm: handles, LDS limits, the workspace
            side.synchronize()
            for n in p:
                p[n].copy_(keep[n])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(p, grads, lst, ws, buf)
        for i in range(5):
            if captured:
                graph.replay()
                torch.cuda.synchronize()
                G.grad_norm([torch.ones(1000 + i, device=device)])  # eager work between
            else:
                step(p, grads, lst, ws, buf)
            norms.append(buf["norm"].clone())
        torch.cuda.synchronize()
        runs.append((p, norms, (buf["g"] ** 2).sum().item()))
    for n in runs[0][0]:
        assert torch.equal(runs[0][0][n], runs[1][0][n]), n
    assert torch.equal(torch.stack(runs[0][1]), torch.stack(runs[1][1]))
    assert all(float(v) > 1.0 for v in runs[0][1])  # every step clipped


def test_streams_and_two_graphs(device):
    """Each operator on another stream than its tensors' own, and two graphs of the
    same operator replayed in turn: each with its own scratch, each the eager bits."""
    gen = torch.Generator().manual_seed(31)
    x, g = rows_of(gen, 3000, 200, torch.float32, device), rows_of(gen, 3000, 200, torch.float32, device)
    x2 = rows_of(gen, 3000, 200, torch.float32, device)
    w = torch.ones(200, device=device)

    def work(x, o):
        L.norm_rows_grads(o["adj"], o["wa"], o["ba"], g, x, w, True)
        D.linear_grads(g, x, o["w"], o["b"])
        G.clip_grads([o["w"], o["b"], o["wa"]], 1.0, out=o["norm"])

    def outs():
        return {"adj": torch.empty_like(x), "wa": torch.empty_like(w), "ba": torch.empty_like(w),
                "w": torch.empty((200, 200), device=device), "b": torch.empty_like(w), "norm": torch.empty((), device=device)}
    eager = [outs(), outs()]
    work(x, eager[0])
    work(x2, eager[1])
    side, o = torch.cuda.Stream(), outs()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x, o)
    side.synchronize()
    assert all(torch.equal(o[k], eager[0][k]) for k in o)
    graphs, got = [], [outs(), outs()]
    for data, o in zip((x, x2), got):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            work(data, o)
        graphs.append(graph)
    for _ in range(3):
        for graph, o in zip(graphs, got):
            for v in o.values():
                v.fill_(math.nan)
            graph.replay()
        torch.cuda.synchronize()
        for o, e in zip(got, eager):
            assert all(torch.equal(o[k], e[k]) for k in o)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(257, 260), (384, 131), (260, 321), (129, 388), (300, 140)])
def test_linear_grads_past_a_tile(device, dtype, n, k):
    """Results that end a few columns into a tile, with enough rows that the widest
    tiles take them: the waves past the edge leave their products out."""
    gen = torch.Generator().manual_seed(n * k)
    M = int(4.1e9 / (n * k)) + 1
    g = torch.randn((M, n), generator=gen).to(device).to(dtype)
    x = torch.randn((M, k), generator=gen).to(device).to(dtype)
    wa, ba = torch.full((n, k), math.nan, device=device), torch.full((n,), math.nan, device=device)
    D.linear_grads(g, x, wa, ba)
    ref = torch.zeros((n, k), dtype=torch.float64)
    size = torch.zeros((n, k), dtype=torch.float64)
    for r in range(0, M, 65536):
        gd, xd = g[r:r + 65536].double().cpu(), x[r:r + 65536].double().cpu()
        ref += gd.t() @ xd
        size += gd.abs().t() @ xd.abs()
    # as linear_bound: normals, so no value is far below its column's largest that matters
    within(wa, ref, (M / 32 + 320) * U * size, "w_adj")
    within(ba, g.double().sum(0).cpu(), (M / 32 + 340) * U * g.double().abs().sum(0).cpu(), "b_adj")


@pytest.mark.parametrize("dtype", TYPES)
def test_workspaces_are_enough(device, dtype):
    """Nothing is written past the bytes that the workspace functions name."""
    lib, guard = A._lib.load(), 1 << 20
    for rows, width in ((1, 300), (5, 16384), (9, 4096), (70, 64), (700, 8192), (3000, 513), (40000, 200), (40000, 7)):
        need = lib.pet_norm_rows_grads_workspace(rows, width)
        room = torch.full((need + guard,), 171, dtype=torch.uint8, device=device)
        x, w = torch.ones((rows, width), dtype=dtype, device=device), torch.ones(width, device=device)
        L.norm_rows_grads(None, torch.empty_like(w), torch.empty_like(w), x, x, w, True, scratch=room[:need])
        assert (room[need:] == 171).all(), (rows, width)
    for M, N, K in ((3, 40, 50), (3000, 130, 70), (50000, 300, 300), (2000, 65, 65)):
        need = lib.pet_linear_grads_workspace(A.DTYPES[dtype], M, N, K)
        room = torch.full((need + guard,), 171, dtype=torch.uint8, device=device)
        g, x = torch.ones((M, N), dtype=dtype, device=device), torch.ones((M, K), dtype=dtype, device=device)
        w, b = torch.empty((N, K), device=device), torch.empty(N, device=device)
        D.linear_grads(g, x, w, b, scratch=room[:need])
        assert (room[need:] == 171).all() and (w == M).all() and (b == M).all(), (M, N, K)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_linear_grads_subnormal(device, dtype):
    """16-bit values below the type's smallest normal one count like any other."""
    gen = torch.Generator().manual_seed(31)
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    top = int(1 / torch.finfo(dtype).eps) - 1
    for M, N, K in ((3000, 300, 260), (648, 64, 64)):
        g = (torch.randint(-top, top + 1, (M, N), generator=gen).double() * step).to(dtype)
        x = (torch.randn((M, K), generator=gen) * (2.0 ** 20 if dtype == torch.bfloat16 else 1.0)).to(dtype)
        gd, xd, ref = g.to(device), x.to(device), g.double().t() @ x.double()
        wa, ba, turned = (torch.empty(s, device=device) for s in ((N, K), (N,), (K, N)))
        D.linear_grads(gd, xd, wa, ba)
        D.linear_grads(xd, gd, turned)
        tol = linear_bound(g, x, dtype) + 400 * least(torch.float32)
        within(wa, ref, tol, "w_adj")
        within(turned.t(), ref, tol, "the other way round")
        within(ba, g.double().sum(0), (M / 32 + 340) * U * g.double().abs().sum(0) + least(torch.float32), "b_adj")


def test_many_tensors_of_every_layout(device):
    """More tensors than a launch takes, consecutive and with rows apart by turns,
    then only the one and only the other, with chunks' edges among their sizes."""
    gen = torch.Generator().manual_seed(37)
    sizes = [1, 8191, 8192, 8193, 77, 16384, 5, 300]
    flat = [torch.randn(sizes[i % 8], generator=gen).to(TYPES[i % 3]).to(device) for i in range(500)]
    base = [torch.randn((sizes[i % 8] // 60 + 1, 70), generator=gen).to(TYPES[i % 3]).to(device) for i in range(260)]
    apart = [b[:, 2:66] for b in base]
    for t in (flat, apart, [x for pair in zip(flat, apart) for x in pair]):
        before, edges = [x.double().cpu() for x in t], [b[:, [0, 1, 66, 67, 68, 69]].clone() for b in base]
        ref = math.sqrt(sum(float((b ** 2).sum()) for b in before))
        assert abs(float(G.grad_norm(t)) - ref) <= 1.01 * U * ref
        assert abs(float(G.clip_grads(t, 0.75 * ref, eps=0.0)) - ref) <= 1.01 * U * ref
        for x, b in zip(t, before):
            within(x, 0.75 * b, (2.01 * U + half(x.dtype)) * 0.75 * b.abs() + least(x.dtype), "clipped")
        assert all(torch.equal(b[:, [0, 1, 66, 67, 68, 69]], e) for b, e in zip(base, edges))


def test_gradients_between_each_other(device):
    """Columns of one matrix as gradients of their own, transposed views among them."""
    m = torch.arange(1.0, 2401.0, device=device).view(40, 60)
    before = m.double().cpu()
    for views in ([m[:, 0], m[:, 1], m[:, 2]], [m.t()[:7], m.t()[7:50]], [m[::2, :9], m[1::2, :9], m[:, 9]]):
        took = torch.zeros(40, 60, dtype=torch.bool, device=device)
        for v in views:
            torch.as_strided(took, v.shape, v.stride(), v.storage_offset()).fill_(True)
        took, m0 = took.cpu(), m.double().cpu()
        ref = float(m0[took].pow(2).sum().sqrt())
        assert abs(float(G.clip_grads(views, 0.5 * ref, eps=0.0)) - ref) <= 1.01 * U * ref
        within(m, torch.where(took, 0.5 * m0, m0), torch.where(took, 2.01 * U * m0, 0.0), "clipped")
        m.copy_(before)
    with pytest.raises(ValueError):
        G.GradList([m[:, :2], m[:, 1]])


def test_norm_rows_past_a_launch(device):
    """More rows than one launch's threads: 2^28 of them at 16 lanes a row."""
    rows = (1 << 28) + 21
    x = torch.empty((rows, 1), dtype=torch.bfloat16, device=device)
    for r in range(0, rows, 1 << 26):
        n = min(1 << 26, rows - r)
        x[r:r + n, 0] = (torch.arange(r, r + n, device=device) % 7 - 3).bfloat16()
    out, w = torch.full_like(x, 9.0), torch.full((1,), 2.0, device=device)
    L.norm_rows(out, x, w, None)
    for r in range(0, rows, 1 << 26):  # x / |x|: exact in bf16
        assert torch.equal(out[r:r + (1 << 26)], 2 * torch.sign(x[r:r + (1 << 26)]))
    x32, out32 = x[:1000].float(), torch.empty((1000, 1), device=device)
    A._lib.check(A._lib.load().pet_norm_rows_typed(0, 1000, 1, out32.data_ptr(), 1, x32.data_ptr(), 1, w.data_ptr(), None,
                                                   A._stream()), "fp32")
    assert torch.equal(out32.bfloat16(), out[:1000])


def test_fp32_rows_past_a_launch(device):
    """The same of the fp32 norms to 2048 columns, at 64 lanes a row: forward, the
    typed entry that calls it, backward."""
    rows = (1 << 26) + 300
    x = (torch.arange(rows, device=device) % 5 - 2).float()[:, None]
    w, lib = torch.full((1,), 2.0, device=device), A._lib.load()
    for call in (lambda o: L.norm_rows(o, x, w, None),
                 lambda o: A._lib.check(lib.pet_norm_rows_typed(0, rows, 1, o.data_ptr(), 1, x.data_ptr(), 1, w.data_ptr(), None,
                                                                A._stream()), "typed")):
        out = torch.full_like(x, 9.0)
        call(out)
        for r in range(0, 5):  # a value's rows are of the same bits, 2 sign(x) to eps and four roundings
            part = out[r::5]
            assert (part == part[0]).all() and abs(float(part[0]) - 2 * ((r > 2) - (r < 2))) <= 10 * U
    adj = torch.full_like(x, 9.0)
    L.norm_rows_bwd(adj, torch.ones_like(x), x, w, False)
    for r in range(0, 5):  # 2 eps / (x^2 + eps)^1.5: of x = 0 2 / sqrt(eps), else eps and the roundings of 2 - 2 xhat^2
        part = adj[r::5]
        ref, tol = (2 * 2 ** 11.5, 8 * U * 2 ** 12.5) if r == 2 else (0.0, 32 * U)
        assert (part == part[0]).all() and abs(float(part[0]) - ref) <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ln", [False, True])
def test_norms_in_place(device, dtype, ln):
    """The forward over its input, the adjoint over out_adj and over the input (beta
    0 and not): the bits of the calls that write elsewhere."""
    gen = torch.Generator().manual_seed(41)
    for width, pad in ((5, 0), (63, 3), (200, 0), (777, 1), (1024, 0), (3001, 1), (5000, 0), (9001, 1)):
        x, g = rows_of(gen, 41, width, dtype, device, pad), rows_of(gen, 41, width, dtype, device, pad, size=1e-2)
        w = (1 + 0.1 * torch.randn(width, generator=gen)).to(device)
        b = (0.1 * torch.randn(width, generator=gen)).to(device) if ln else None

        def copy(t):
            return torch.empty_strided(t.shape, t.stride(), dtype=dtype, device=device).copy_(t)
        out, into = copy(x), copy(x)
        L.norm_rows(out, x, w, b)
        L.norm_rows(into, into, w, b)
        assert torch.equal(out, into), width
        for beta in (0.0, 0.5):
            for at in (0, 1):
                args = [copy(g), copy(x)]
                adj = copy(args[at])
                L.norm_rows_grads(adj, None, None, *args, w, ln, beta)
                L.norm_rows_grads(args[at], None, None, *args, w, ln, beta)
                assert torch.equal(adj, args[at]), (width, beta, at)


def fp32_rows_bound(g, x, roundings=None):
    """What include/pet_model.h states of fp32 rows: a factor is held to 2^-23 of itself or
    2^-36 of its column's largest, a product to a further 2^-22; then the sum's roundings
    (linear_bound's where none are given)."""
    g, x = g.double().cpu().abs(), x.double().cpu().abs()
    off_g = torch.maximum(2.0 ** -23 * g, 2.0 ** -36 * g.amax(0, keepdim=True))
    off_x = torch.maximum(2.0 ** -23 * x, 2.0 ** -36 * x.amax(0, keepdim=True))
    products = off_g.t() @ (x + off_x) + g.t() @ off_x + 2.0 ** -22 * (g.t() @ x)
    return products + (roundings or len(g) / 32 + 308) * U * (g.t() @ x + products)


@pytest.mark.parametrize("times", [1e4, 1e6, 1e8, 1e12])
def test_linear_grads_outliers(device, times):
    """One value `times` the rest of its column, where the other factor is zero: the
    column's other products are held to 2^-36 of it, and no other column is touched."""
    gen = torch.Generator().manual_seed(61)
    for M, N, K in ((1024, 80, 70), (40000, 300, 400)):
        g, x = torch.randn((M, N), generator=gen), torch.randn((M, K), generator=gen)
        g[M // 3, 7], x[M // 3] = times, 0.0
        x[M // 2, 11], g[M // 2] = -times, 0.0
        wa, ba = torch.empty((N, K), device=device), torch.empty(N, device=device)
        D.linear_grads(g.to(device), x.to(device), wa, ba)
        ref, size = g.double().t() @ x.double(), g.double().abs().t() @ x.double().abs()
        within(wa, ref, fp32_rows_bound(g, x), "w_adj")
        rest = torch.ones((N, K), dtype=torch.bool)
        rest[7], rest[:, 11] = False, False
        off = (wa.double().cpu() - ref).abs() / size
        print(f"{M} x {N} x {K}, {times:g}: {float(off[rest].max()):.1e} of the sum's magnitude, with outliers {float(off[~rest].max()):.1e}")
        assert float(off[rest].max()) <= (M / 32 + 308 + 8) * U
        within(ba, g.double().sum(0), (M / 32 + 340) * U * g.double().abs().sum(0), "b_adj")


# ---- every tile of the weight gradients: 256, 128 and 64 columns wide, many pieces and one ----


def tile_of(dtype, M, N, K):
    """The tile that a size takes, told from its workspace (the pieces' sums and their
    biases'), or None of one piece, which needs none."""
    step = 32 if dtype == torch.float32 else 64
    need = A._lib.load().pet_linear_grads_workspace(A.DTYPES[dtype], M, N, K)
    if need <= 16:
        return None
    found = []
    for tile, (edge, resident) in enumerate(((256, 256), (128, 512), (64, 1024))):
        tn, tk, steps = -(-N // edge), -(-K // edge), -(-M // step)
        pieces = max(1, min(resident // (tn * tk), (steps + 3) // 4))
        pieces = pieces & ~7 if pieces > 8 else pieces
        pieces = -(-M // (-(-steps // pieces) * step))
        pieces = (pieces + 7) & ~7 if pieces > 8 else pieces
        if need == (pieces * tk * N * 8 + 15) // 16 * 16 + pieces * N * K * 4:
            found.append(tile)
    assert len(found) == 1, (dtype, M, N, K, need)
    return found[0]


TILES = [(0, 30011, 401, 355), (0, 8001, 257, 2000), (1, 5003, 390, 517), (1, 18001, 330, 200), (2, 26671, 128, 130),
         (2, 5003, 77, 129), (None, 400, 4097, 4099), (None, 70, 4097, 4099), (None, 5, 2050, 2049)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile,M,N,K", TILES)
def test_tiles_of_integers(device, dtype, tile, M, N, K):
    """Small integers, whose sums fp32 holds: every tile's result is exact, onto beta times
    what was there, from rows at any address, and of the live rows alone."""
    assert tile_of(dtype, M, N, K) == tile
    gen = torch.Generator(device=device).manual_seed(M)
    ints = lambda *s: torch.randint(-8, 9, s, generator=gen, device=device)
    for pad, off, beta, live in ((0, 0, 0.0, None), (3, 1, 0.5, None), (8, 0, 1.0, M - M // 3), (1, 2, 0.0, 1), (0, 0, 0.5, 0)):
        n = M if live is None else live
        g, x = (torch.full((off + M * (c + pad),), math.nan, dtype=dtype, device=device)[off:].view(M, c + pad)[:, :c]
                for c in (N, K))
        g[:n], x[:n] = ints(n, N).to(dtype), ints(n, K).to(dtype)
        w0, b0 = 2.0 * ints(N, K), 2.0 * ints(N)
        wa = torch.full((N, K + pad), 77.0, device=device)
        wa[:, :K] = w0
        ba = b0.clone()
        D.linear_grads(g, x, wa[:, :K], ba, beta, live=None if live is None else torch.tensor([live], dtype=torch.int32, device=device))
        gd = g[:n].double()
        ref = gd.t().contiguous() @ x[:n].double()
        assert float(ref.abs().max()) < 2 ** 22 and torch.equal(wa[:, :K].double(), ref + beta * w0)
        assert torch.equal(ba.double(), gd.sum(0) + beta * b0) and (wa[:, K:] == 77).all()


@pytest.mark.parametrize("tile,M,N,K", TILES)
@pytest.mark.parametrize("way", ["even", "grow", "shrink", "columns"])
def test_tiles_of_few_rows(device, tile, M, N, K, way):
    """fp32 rows that are zero but for a few, so that a bound of a few roundings holds:
    the pairs' low parts count, and scales that change from row to row are handed on
    to every wave. One factor grows or shrinks by 10^20 along the rows."""
    gen = torch.Generator(device=device).manual_seed(N)
    at = torch.unique(torch.tensor([0, 1, 31, 32, 33, 64, 95, 127, M // 3, M // 2, M - 40, M - 2, M - 1], device=device).clamp(0, M - 1))
    g, x = torch.zeros((M, N), device=device), torch.zeros((M, K), device=device)
    ramp = torch.linspace(-10, 10, len(at), device=device)[:, None]
    size_g, size_x = {"even": (0 * ramp, 0 * ramp), "grow": (ramp, 0 * ramp), "shrink": (0 * ramp, -ramp),
                      "columns": (torch.linspace(-15, 15, N, device=device)[None], torch.linspace(15, -15, K, device=device)[None])}[way]
    g[at] = torch.randn((len(at), N), generator=gen, device=device) * 10 ** size_g
    x[at] = torch.randn((len(at), K), generator=gen, device=device) * 10 ** size_x
    wa, ba = torch.full((N, K), math.nan, device=device), torch.full((N,), math.nan, device=device)
    D.linear_grads(g, x, wa, ba)
    gd, xd = g[at].double().cpu(), x[at].double().cpu()
    ref = gd.t() @ xd
    # a step's own products 8 roundings (linear_bound), its sum's addition one more, and the joining of the pieces
    within(wa, ref, fp32_rows_bound(gd, xd, 9 * len(at) + 4), "w_adj")
    within(ba, gd.sum(0), (len(at) + 4) * U * gd.abs().sum(0), "b_adj")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile,M,N,K", [t for t in TILES if t[0] in (0, 1)] + [(None, 400, 4097, 4099)])
def test_tiles_not_finite(device, dtype, tile, M, N, K):
    """Infinities and NaN in every tile: where the formula takes them and nowhere else."""
    gen = torch.Generator(device=device).manual_seed(K)
    g, x = (torch.randint(-8, 9, (M, c), generator=gen, device=device).to(dtype) for c in (N, K))
    g[g == 0], x[x == 0] = 1.0, 1.0
    g[7, 3], g[M - 2, 80], x[9, 11], x[M // 2, K - 1] = math.inf, math.nan, -math.inf, math.nan
    x[7, 100] = 0.0  # inf * 0
    wa, ba = torch.empty((N, K), device=device), torch.empty(N, device=device)
    D.linear_grads(g, x, wa, ba)
    clean = g.double().nan_to_num(0, 0, 0).t().contiguous() @ x.double().nan_to_num(0, 0, 0)
    ref = clean.clone()
    ref[3] = torch.copysign(torch.full((K,), math.inf, dtype=torch.float64, device=device), x[7].double())
    up = torch.copysign(torch.full((N,), math.inf, dtype=torch.float64, device=device), -g[9].double())
    ref[:, 11] = torch.where(torch.isinf(ref[:, 11]) & (ref[:, 11] != up), math.nan, up)
    ref[3, 100], ref[80], ref[:, K - 1] = math.nan, math.nan, math.nan
    got = wa.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    ok = ~torch.isnan(ref)
    assert torch.equal(got[ok], ref[ok])  # the rest are integers that fp32 holds
    assert torch.isinf(ba[3]) and torch.isnan(ba[80]) and int(torch.isfinite(ba).sum()) == N - 2


# ---- the attention layer's gradients at the sizes of its other products --------------------


def large_layer(device, H, hd, atoms, ln, extra, seed=71):
    rng = np.random.default_rng(seed)
    Dm = H * hd
    tk = systems.tokens_from_counts(list(rng.integers(1, 150, atoms)), seed=seed)
    T = tk.n_rows + extra
    a = {"tokens": rng.standard_normal((T, Dm)), "nw": 1 + 0.1 * rng.standard_normal(Dm), "nb": 0.1 * rng.standard_normal(Dm),
         "w_in": rng.standard_normal((3 * Dm, Dm)) / Dm ** 0.5, "b_in": 0.1 * rng.standard_normal(3 * Dm),
         "w_out": rng.standard_normal((Dm, Dm)) / Dm ** 0.5, "b_out": 0.1 * rng.standard_normal(Dm),
         "g": rng.standard_normal((T, Dm))}
    a = {k: torch.from_numpy(v.astype(np.float32)).to(device) for k, v in a.items()}
    if not ln:
        a["nb"] = None
    return a, tk, T


@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("H,hd,atoms", [(4, 32, 120), (8, 32, 300), (4, 64, 300), (2, 32, 8)])
def test_attention_layer_grads_large(device, H, hd, atoms, ln):
    """Every parameter's gradient where the layer's products take the three-part kernels
    (2^27 products and more) and the split ones (2^32, where the plain backward keeps
    no fp32 adjoint of qkv), against float64 and the plain backward. The rows of a
    capacity hold NaN, in out_adj, the tokens and the saved rows: none is read."""
    Dm, temp = H * hd, 1.1
    a, tk, T = large_layer(device, H, hd, atoms, ln, 77)
    live, S = tk.n_rows, tk.slots
    for k in ("g", "tokens"):
        a[k][live:] = math.nan
    off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
    t, ws = A.Tokens(off, tk.n_atoms, True), A.Workspace(device)
    out = torch.empty((T, Dm), device=device)
    L.attention_layer(ws, "l", out, a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"], a["b_out"], t, S, H, hd, temp)
    ws.peek2("l:merged")[live:] = math.nan
    grads = {n: torch.full_like(a[k], math.nan) for n, k in NAMES.items() if a[k] is not None}
    got = []
    for with_grads in (True, False):
        tadj, csa = torch.full((T, Dm), 0.5, device=device), torch.zeros((tk.n_atoms, S), device=device)
        args = (tadj, csa, a["g"], a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"], t, S, H, hd, temp)
        if with_grads:
            L.attention_layer_grads(ws, "l", grads, *args)
        else:
            L.attention_layer_bwd(ws, "l", *args)
        assert (tadj[live:] == 0.5).all() and torch.isfinite(tadj).all() and torch.isfinite(csa).all(), with_grads
        got.append((tadj, csa))
    for x, y in zip(*got):
        assert float((x - y).abs().max()) <= 1e-5 * float(y.abs().max())
    leaves = {n: a[k].double().cpu().requires_grad_() for n, k in NAMES.items() if a[k] is not None}
    tokens = a["tokens"][:live].double().cpu().requires_grad_()
    ref = attention_f64(tokens, leaves["norm_w"], leaves.get("norm_b"), leaves["w_in"], leaves["b_in"],
                        leaves["w_out"], leaves["b_out"], tk, torch.from_numpy(tk.cf_seq).double(), H, hd, temp)
    (ref * a["g"][:live].double().cpu()).sum().backward()
    for n, g in grads.items():
        want = leaves[n].grad
        off_by = float((g.double().cpu() - want).abs().max()) / float(want.abs().max())
        print(f"{H} x {hd}, {live} rows, {n}: {off_by:.1e}", flush=True)
        assert off_by <= 1e-5, n
    sink = tokens.grad + 0.5 * (torch.arange(live) >= tk.n_atoms)[:, None]
    assert float((got[0][0][:live].double().cpu() - sink).abs().max()) <= 1e-5 * float(sink.abs().max())


def test_attention_layer_grads_views(device):
    """Rows in wider buffers: the results of contiguous ones, to the products' other
    kernels, and nothing beside the rows is touched. Offsets that are not consecutive
    are refused."""
    a, tk, T, H, hd = layer_case(device, True, False)
    Dm, S = H * hd, tk.slots
    off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
    t, ws = A.Tokens(off, tk.n_atoms, False), A.Workspace(device)
    out = torch.empty((T, Dm), device=device)
    L.attention_layer(ws, "l", out, a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"], a["b_out"], t, S, H, hd, 1.0)
    results = []
    for pad in (0, 4, 3):
        def wide(x):
            buf = torch.full((x.shape[0], x.shape[1] + pad), 9.0, device=device)
            buf[:, :x.shape[1]] = x
            return buf[:, :x.shape[1]], buf[:, x.shape[1]:]
        (tadj, e0), (csa, e1) = wide(torch.full((T, Dm), 0.5, device=device)), wide(torch.zeros((tk.n_atoms, S), device=device))
        (g, _), (tokens, _), (c, _) = wide(a["g"]), wide(a["tokens"]), wide(cf)
        grads = {n: torch.full_like(a[k], math.nan) for n, k in NAMES.items()}
        args = (grads, tadj, csa, g, tokens, a["nw"], a["nb"], a["w_in"], a["b_in"], c, a["w_out"])
        L.attention_layer_grads(ws, "l", *args, t, S, H, hd, 1.0)
        assert (e0 == 9).all() and (e1 == 9).all()
        results.append([tadj, csa, *grads.values()])
    for got in results[1:]:
        for x, y in zip(got, results[0]):
            assert float((x - y).abs().max()) <= 1e-6 * float(y.abs().max())
    apart = torch.zeros(2 * (tk.n_atoms + 1), dtype=torch.int32, device=device)[::2]
    apart.copy_(off)
    with pytest.raises(ValueError):
        L.attention_layer_grads(ws, "l", *args, A.Tokens(apart, tk.n_atoms, False), S, H, hd, 1.0)


def test_no_fp32_rows(device):
    x, w = torch.zeros((0, 40), device=device), torch.ones(40, device=device)
    L.norm_rows(x, x, w, None)
    L.norm_rows(x, x, w, w)
    L.norm_rows_bwd(x, x, x, w, True)


@pytest.mark.parametrize("ln", [False, True])
def test_attention_layer_grads_whatever_is_dead(device, ln):
    """What a capacity's rows of out_adj hold changes no bit of any result."""
    results = []
    for dead in ("nan", True):
        a, tk, T, H, hd = layer_case(device, ln, dead)
        Dm, S = H * hd, tk.slots
        off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
        t, ws = A.Tokens(off, tk.n_atoms, True), A.Workspace(device)
        out, tadj, csa = torch.empty((T, Dm), device=device), torch.zeros((T, Dm), device=device), torch.zeros((tk.n_atoms, S), device=device)
        args = (a["tokens"], a["nw"], a["nb"], a["w_in"], a["b_in"], cf, a["w_out"])
        L.attention_layer(ws, "l", out, *args, a["b_out"], t, S, H, hd, 1.0)
        grads = {n: torch.full_like(a[k], math.nan) for n, k in NAMES.items() if a[k] is not None}
        L.attention_layer_grads(ws, "l", grads, tadj, csa, a["g"], *args, t, S, H, hd, 1.0)
        results.append([tadj, csa, *grads.values()])
    assert all(torch.equal(x, y) and torch.isfinite(x).all() for x, y in zip(*results))


def attention_of_normed(normed, w_in, b_in, w_out, b_out, tk, cf, H, hd):
    """attention_f64 (temperature 1) from the normed tokens on."""
    q, k, v = ((normed @ w_in.t() + b_in)[:, i * H * hd:(i + 1) * H * hd] for i in range(3))
    merged = torch.zeros_like(normed)
    for n in range(tk.n_atoms):
        rows = [n] + list(range(tk.n_atoms + int(tk.off[n]), tk.n_atoms + int(tk.off[n + 1])))
        c = cf[n, :len(rows)]
        on = [r for r, x in zip(rows, c) if x > 0]
        cols = [slice(h * hd, (h + 1) * hd) for h in range(H)]
        o = [torch.softmax(q[on, s] @ k[on, s].t() / math.sqrt(hd) + torch.log(c[c > 0]), -1) @ v[on, s] for s in cols]
        merged[on] = torch.cat(o, 1)
    return merged @ w_out.t() + b_out


@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("H,hd,counts,kind", [(3, 5, [4, 0, 9], "random"), (1, 24, [1, 30], "zeros"), (2, 40, [0], "ones"),
                                              (4, 16, [300, 5, 0, 700], "zeros"), (1, 128, [17, 3], "zeros"), (2, 1, [6, 2], "random")])
def test_attention_layer_grads_of_any_shape(device, H, hd, counts, kind, ln):
    """Head widths of no vector's multiple, atoms without edges, edges at their cutoff
    (whose rows are masked), more slots than the LDS-staged kernels hold."""
    Dm = H * hd
    rng = np.random.default_rng(91)
    tk = systems.tokens_from_counts(counts, seed=5, cf_kind=kind)
    T, S, N = tk.n_rows, tk.slots, tk.n_atoms
    r = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(device)
    tokens, g, nw, nb = r(T, Dm), r(T, Dm), 1 + 0.1 * r(Dm), 0.1 * r(Dm) if ln else None
    w_in, b_in, w_out, b_out = r(3 * Dm, Dm) / Dm ** 0.5, 0.1 * r(3 * Dm), r(Dm, Dm) / Dm ** 0.5, r(Dm)
    off, cf = torch.from_numpy(tk.off).to(device), torch.from_numpy(tk.cf_seq).to(device)
    t, ws = A.Tokens(off, N), A.Workspace(device)
    out, tadj, csa = torch.empty((T, Dm), device=device), torch.zeros((T, Dm), device=device), torch.zeros((N, S), device=device)
    L.attention_layer(ws, "l", out, tokens, nw, nb, w_in, b_in, cf, w_out, b_out, t, S, H, hd, 1.0)
    given = {"norm_w": nw, "norm_b": nb, "w_in": w_in, "b_in": b_in, "w_out": w_out, "b_out": b_out}
    grads = {n: torch.full_like(v, math.nan) for n, v in given.items() if v is not None}
    L.attention_layer_grads(ws, "l", grads, tadj, csa, g, tokens, nw, nb, w_in, b_in, cf, w_out, t, S, H, hd, 1.0)
    leaves = {n: v.double().cpu().requires_grad_() for n, v in given.items() if v is not None}
    x, gd, w = tokens.double().cpu().requires_grad_(), g.double().cpu(), leaves["norm_w"]
    c = x - x.mean(1, keepdim=True) if ln else x
    inv = 1 / torch.sqrt((c ** 2).mean(1, keepdim=True) + (1e-5 if ln else 2.0 ** -23))
    normed = c * inv * w + leaves["norm_b"] if ln else c * inv * w
    normed.retain_grad()
    ref = attention_of_normed(normed, leaves["w_in"], leaves["b_in"], leaves["w_out"], leaves["b_out"], tk,
                              torch.from_numpy(tk.cf_seq).double(), H, hd)
    (ref * gd).sum().backward()
    for name, got, want in [("out", out, ref.detach())] + [(n, v, leaves[n].grad) for n, v in grads.items()]:
        # the attention's bar, of a tensor's largest value; where that is a cancellation of larger terms, of those
        scale = max(float(want.abs().max()), 1e-2)
        assert float((got.double().cpu() - want).abs().max()) <= 1e-5 * scale, name
    # The normed tokens' adjoint h is within that bar, and the norm's adjoint is linear in it:
    # inv (h w - [mean(h w)] - xhat mean(h w xhat)) is within 1e-5 of the largest sum of its
    # terms' magnitudes. (Of two columns LayerNorm's terms cancel to 1e-5 of themselves: xhat is
    # +-1 to eps, and what is left of terms of 15 is 0.2.)
    with torch.no_grad():
        hw, xhat = (normed.grad * w).abs(), (c * inv).abs()
        terms = inv * (hw + (hw.mean(1, keepdim=True) if ln else 0.0) + xhat * (hw * xhat).mean(1, keepdim=True))
        print(f"{H} x {hd}, ln {ln}: terms to {float(terms.max()):.2g}, adjoint to {float(x.grad.abs().max()):.2g}")
        assert float((tadj.double().cpu() - x.grad).abs().max()) <= 1e-5 * float(terms.max())
