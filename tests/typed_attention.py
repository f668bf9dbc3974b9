"""The typed attention and the dropout from their formulas in 64 bits: what the
tests of both sides of the C ABI compare with, and how far off a result may be.

Bounds, with U = 2^-24 (half an fp32 step) and h half a step of the row type:

- a logit is an fp32 sum of head_dim products and a few terms: off by at most
  e_s = U (scale (head_dim + 4) |q|.|k| + 6 (|s| + |log cf| + |b| + |max|)), and a
  probability, with its maximum's, its sum's (S terms), the exponential's (2 U, and the
  exponent's rounding in base 2, in e_s) and the reciprocal's roundings, by the
  share e_p = 2 max_j e_s + (S + 16) U;
- the forward rounds the probabilities (h of each; fp16 under 2^-14 by 2^-25 of the
  row's largest) and its result: h |O| + (h + e_p + S U) sum_j P M |v_j|;
- dO.v_j and dO.O are fp32 sums: dS_ij is off by e_ds = e_p P (|dP| + |D|) +
  (head_dim + 8) U P (M |dO|.|v_j| + |dO|.|O|); dQ and dK round it (h) and their results,
  over sums of n terms (n U of the terms' magnitudes); dV as the forward; the cutoff
  factors' and the table's adjoints are fp32 sums of e_ds each and n roundings.
"""
from __future__ import annotations

import math

import numpy as np
import torch

U = 2.0 ** -24
TURNS = (13, 15, 26, 6, 17, 29, 16, 24)


def threefry(key, counter, rounds=13):
    """Threefry-2x32 of arrays of uint32 (numpy)."""
    k = [np.uint32(key[0]), np.uint32(key[1])]
    k.append(k[0] ^ k[1] ^ np.uint32(0x1BD11BDA))
    with np.errstate(over="ignore"):
        x = np.asarray(counter[0], dtype=np.uint32) + k[0]
        y = np.asarray(counter[1], dtype=np.uint32) + k[1]
        for i in range(rounds):
            x = x + y
            t = np.uint32(TURNS[i % 8])
            y = ((y << t) | (y >> (np.uint32(32) - t))) ^ x
            if i % 4 == 3:
                j = (i + 1) // 4
                x, y = x + k[j % 3], y + k[(j + 1) % 3] + np.uint32(j)
    return x, y


def numbers(seed, step, call, x, y):
    """The four 16-bit numbers of each block (x, y): [..., 4]."""
    seed, step = int(seed) & (1 << 64) - 1, int(step) & (1 << 64) - 1
    key = threefry((seed & 0xFFFFFFFF, seed >> 32), (np.uint32(step & 0xFFFFFFFF), np.uint32(call)))
    a, b = threefry((int(key[0]), int(key[1])), np.broadcast_arrays(np.uint32(x), np.uint32(y)))
    low = np.uint32(0xFFFF)
    return np.stack([a & low, a >> np.uint32(16), b & low, b >> np.uint32(16)], -1)


def rows_mask(seed, step, call, p, rows, width):
    """M of dropout_rows, with its scale, float64 [rows, width]."""
    least = round(65536 * p)
    n = numbers(seed, step, call, np.arange(rows)[:, None], np.arange((width + 3) // 4)[None, :])
    return torch.from_numpy((n.reshape(rows, -1)[:, :width] >= least) * (65536.0 / (65536 - least)))


def attention_mask(seed, step, call, p, rows, heads):
    """M of one atom's attention, [heads, count, count], for its tokens' rows."""
    least, count = round(65536 * p), len(rows)
    groups = (count + 3) // 4
    y = np.arange(groups)[None, None, :] * heads + np.arange(heads)[:, None, None]
    n = numbers(seed, step, call, np.asarray(rows)[None, :, None], y)
    return torch.from_numpy((n.reshape(heads, count, -1)[..., :count] >= least) * (65536.0 / (65536 - least)))


def half(t):
    return torch.finfo(t).eps / 2


class Case:
    """One layout with everything that its attention takes, in 64 bits on the host."""

    def __init__(self, counts, heads, kv_heads, head_dim, dtype, seed=0, buckets=0, reach=0, p=0.0, zeros=0.0, dead=0,
                 temperature=1.0, slots=None, size=0.7):
        rng = np.random.default_rng(seed)
        self.counts = [int(c) for c in counts]  # edges
        self.N, self.H, self.Hk, self.hd, self.dtype, self.p, self.temperature = (
            len(self.counts), heads, kv_heads, head_dim, dtype, p, temperature)
        self.off = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.T = self.N + int(self.off[-1]) + dead
        self.dead = dead
        self.S = (max(self.counts, default=0) + 1) if slots is None else slots
        W = (heads + 2 * kv_heads) * head_dim
        self.qkv = torch.from_numpy(rng.standard_normal((self.T, W)) * size).to(dtype)
        self.dmerged = torch.from_numpy(rng.standard_normal((self.T, heads * head_dim)) * 0.05).to(dtype)
        self.cf = torch.zeros((self.N, self.S), dtype=torch.float32)
        for n, c in enumerate(self.counts):
            v = rng.uniform(0.05, 1.0, c)
            v[rng.random(c) < zeros] = 0.0
            self.cf[n, 0] = 1.0
            self.cf[n, 1:c + 1] = torch.from_numpy(v)
        self.table = torch.from_numpy(rng.standard_normal((buckets, heads)) * 0.5).float() if buckets else None
        self.pos = torch.from_numpy(rng.integers(-3 * reach - 5, 3 * reach + 5, self.T)).int() if buckets else None
        self.reach = reach
        self.buckets = None
        self.state = (int(rng.integers(0, 1 << 62)), int(rng.integers(0, 1 << 40)))
        self.call = 7

    def rows(self, n):
        return [n] + list(range(self.N + int(self.off[n]), self.N + int(self.off[n + 1])))

    def parts(self, n):
        """(rows, q, k, v [heads, count, hd], cf, which keys, which queries, bias, mask) of an atom, masked rows zero."""
        rows, H, Hk, hd = self.rows(n), self.H, self.Hk, self.hd
        c = len(rows)
        x = self.qkv[rows].double()
        cf = self.cf[n, :c].double()
        keys = cf > 0
        queries = keys.clone()
        queries[0] = True
        x = torch.where((keys | queries)[:, None], x, 0.0)
        q = x[:, :H * hd].view(c, H, hd).transpose(0, 1) * queries[None, :, None]
        k = (x[:, H * hd:(H + Hk) * hd].view(c, Hk, hd).transpose(0, 1)).repeat_interleave(H // Hk, 0)
        v = (x[:, (H + Hk) * hd:].view(c, Hk, hd).transpose(0, 1)).repeat_interleave(H // Hk, 0)
        k, v = (torch.where(keys[None, :, None], t, 0.0) for t in (k, v))
        bias = index = None
        if self.table is not None:
            pos = self.pos[rows].long()
            index = self.buckets[(pos[None, :] - pos[:, None]).clamp(-self.reach, self.reach) + self.reach].long()
            index = index.clamp(0, self.table.shape[0] - 1)
            bias = self.table.double()[index].permute(2, 0, 1)
        mask = attention_mask(*self.state, self.call, self.p, rows, H) if self.p else None
        return rows, q, k, v, cf, keys, queries, bias, index, mask

    @property
    def scale(self):
        return float(np.float32(1.0 / (math.sqrt(self.hd) * self.temperature)))

    def attend(self, n):
        rows, q, k, v, cf, keys, queries, bias, index, mask = self.parts(n)
        s = self.scale * (q @ k.transpose(1, 2))
        if bias is not None:
            s = s + bias
        s = torch.where(keys[None, None, :], s + torch.log(torch.where(keys, cf, 1.0)), -math.inf)
        top = s.amax(-1, keepdim=True)
        some = queries[None, :, None] & (top > -math.inf)
        e = torch.where(some, torch.exp(s - torch.where(some, top, 0.0)), 0.0)
        total = e.sum(-1, keepdim=True)
        prob = torch.where(some, e / torch.where(some, total, 1.0), 0.0)
        # the logits' errors, and the probabilities'
        a = self.scale * (self.hd + 4) * (q.abs() @ k.abs().transpose(1, 2))
        extra = torch.log(torch.where(keys, cf, 1.0)).abs()[None, None, :] + (bias.abs() if bias is not None else 0.0)
        fin = torch.where(torch.isfinite(s), s.abs(), 0.0)
        e_s = U * (a + 6 * (fin + torch.where(torch.isfinite(extra), extra, 0.0) + torch.where(some, top.abs(), 0.0)))
        e_p = 2 * torch.where(keys[None, None, :], e_s, 0.0).amax(-1, keepdim=True) + (len(rows) + 16) * U
        return rows, q, k, v, cf, keys, queries, index, mask, prob, top, total, some, e_p

    def forward(self):
        """(merged, its bound, ml, its bound) in 64 bits."""
        H, hd, h = self.H, self.hd, half(self.dtype)
        out, tol = (torch.zeros((self.T, H * hd), dtype=torch.float64) for _ in range(2))
        ml, ml_tol = (torch.zeros((self.N, H, self.S, 2), dtype=torch.float64) for _ in range(2))
        for n in range(self.N):
            rows, q, k, v, cf, keys, queries, index, mask, prob, top, total, some, e_p = self.attend(n)
            c = len(rows)
            pm = prob if mask is None else prob * mask
            o, mag = pm @ v, pm @ v.abs()
            o[~some.expand_as(o)] = 0.0
            few = 0.0
            if self.dtype == torch.float16:
                few = 2.0 ** -25 * v.abs().sum(1, keepdim=True) / torch.where(some, total, 1.0) * (1 if mask is None else mask.max())
            t = h * o.abs() + (h + e_p + (c + 2) * U) * mag + few + torch.finfo(self.dtype).smallest_normal * h
            out[rows] = o.transpose(0, 1).reshape(c, -1)
            tol[rows] = (t * some).transpose(0, 1).reshape(c, -1)
            ml[n, :, :c, 0] = torch.where(some, top, 0.0)[..., 0]
            ml[n, :, :c, 1] = torch.where(some, 1.0 / torch.where(some, total, 1.0), 0.0)[..., 0]
            ml_tol[n, :, :c, 0] = (e_p * some)[..., 0]
            ml_tol[n, :, :c, 1] = (2 * e_p * ml[n, :, :c, 1:]) [..., 0]
        return out, tol, ml.view(-1, 2), ml_tol.view(-1, 2)

    def backward(self, merged):
        """{name: (value, bound)} of the adjoints for dO = dmerged and the forward's rounded merged."""
        H, Hk, hd, h = self.H, self.Hk, self.hd, half(self.dtype)
        G = H // Hk
        adj, tol = (torch.zeros_like(self.qkv, dtype=torch.float64) for _ in range(2))
        cf_adj, cf_tol = (torch.zeros((self.N, self.S), dtype=torch.float64) for _ in range(2))
        nb = 0 if self.table is None else self.table.shape[0]
        tab, tab_mag, tab_err = (torch.zeros((nb, H), dtype=torch.float64) for _ in range(3))
        least = torch.finfo(self.dtype).smallest_normal * h
        pairs = 0
        for n in range(self.N):
            rows, q, k, v, cf, keys, queries, index, mask, prob, top, total, some, e_p = self.attend(n)
            c = len(rows)
            pairs += ((c + 31) // 32 * 32) ** 2
            do, o = (torch.where(queries[:, None], x[rows].double(), 0.0).view(c, H, hd).transpose(0, 1)
                     for x in (self.dmerged, merged))
            m = 1.0 if mask is None else mask
            dp = m * (do @ v.transpose(1, 2))
            dp_mag = m * (do.abs() @ v.abs().transpose(1, 2))
            d, d_mag = (do * o).sum(-1, keepdim=True), (do * o).abs().sum(-1, keepdim=True)
            ds = prob * (dp - d)
            e_ds = e_p * prob * (dp.abs() + d.abs()) + (hd + 8) * U * prob * (dp_mag + d_mag)
            ads = ds.abs()
            tiny = 0.0
            if self.dtype == torch.float16:  # under the scaled adjoints' smallest normal
                bound = do.norm(dim=-1).max() * v.norm(dim=-1).max() * (m if mask is None else m.max()) + d.abs().max()
                tiny = float(bound) * 2.0 ** -38
            e16 = h * ads + e_ds + tiny
            dq, dq_t = ds @ k, (e16 + c * U * ads) @ k.abs()
            dk, dk_t = ds.transpose(1, 2) @ q, (e16 + G * c * U * ads).transpose(1, 2) @ q.abs()
            pm = prob * m
            few = 2.0 ** -25 * (1 if mask is None else float(m.max())) if self.dtype == torch.float16 else 0.0
            dv, dv_t = pm.transpose(1, 2) @ do, ((h + e_p + (G * c + 4) * U) * pm + few).transpose(1, 2) @ do.abs()
            def grouped(x):
                return (x * keys[None, :, None]).reshape(Hk, G, c, hd).sum(1).transpose(0, 1).reshape(c, -1)
            adj[rows] = torch.cat([self.scale * dq.transpose(0, 1).reshape(c, -1), self.scale * grouped(dk), grouped(dv)], 1)
            tol[rows] = torch.cat([self.scale * dq_t.transpose(0, 1).reshape(c, -1), self.scale * grouped(dk_t),
                                   grouped(dv_t)], 1)
            safe = torch.where(keys, cf, 1.0)
            cf_adj[n, :c] = torch.where(keys, ds.sum((0, 1)) / safe, 0.0)
            cf_tol[n, :c] = torch.where(keys, (e_ds + (H + c) * U * ads).sum((0, 1)) / safe, 0.0)
            if nb:
                for b in range(nb):
                    at = index == b
                    tab[b] += (ds * at).sum((1, 2))
                    tab_mag[b] += (ads * at).sum((1, 2))
                    tab_err[b] += (e_ds * at).sum((1, 2))
        tol = tol + h * adj.abs() + 4 * least
        got = {"qkv_adj": (adj, tol), "cf_seq_adj": (cf_adj, cf_tol + 4 * U * cf_adj.abs())}
        if nb:
            got["bias_adj"] = (tab, tab_err + (pairs / 64 + 260) * U * tab_mag)
        return got
